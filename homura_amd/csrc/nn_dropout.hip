// hmn_dropout: out = residual + (kept ? src / (1 - p) : 0), the mask computed where it is used.
//
// Element i is kept when word i % 4 of Philox block offset + i / 4 reaches the threshold, so a thread that owns four
// elements in a row needs one block and nothing is stored for the backward pass, which is this kernel again.
#include "nn.hpp"
#include "philox.hpp"

namespace hmr {
namespace nn {
namespace {

struct DropoutArgs {
    char *out;
    const char *src;
    const char *residual;  // or nullptr
    const uint64_t *base;  // or nullptr
    uint64_t seed, offset;
    int64_t n;
    double scale;        // 1 / (1 - p)
    uint32_t threshold;  // a word below it drops its element
    int ndim;            // merged dimensions, outermost first
    int64_t size[HMR_MAX_DIMS];
    int64_t stride[3][HMR_MAX_DIMS];  // of out, src, residual
};

// A thread owns a Philox block, four elements that follow each other in row-major order, wherever they lie.
template <class T>
__global__ void __launch_bounds__(kBlock) dropout_any_kernel(DropoutArgs a, bool none) {
    using C = typename Comp<T>::C;
    const uint64_t offset = a.offset + (a.base != nullptr ? *a.base : 0);
    const int64_t blocks = (a.n + 3) / 4;
    for (int64_t b = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; b < blocks;
         b += static_cast<int64_t>(gridDim.x) * kBlock) {
        const Word4 w = philox_block(offset + static_cast<uint64_t>(b), a.seed);
        for (int j = 0; j < 4; ++j) {
            int64_t i = 4 * b + j;
            if (i >= a.n) break;
            int64_t at[3] = {0, 0, 0};
            for (int k = a.ndim - 1; k >= 0; --k) {
                const int64_t q = i / a.size[k], r = i - q * a.size[k];
                for (int o = 0; o < 3; ++o) at[o] += r * a.stride[o][k];
                i = q;
            }
            const bool keep = !none && w.v[j] >= a.threshold;
            C y = keep ? Comp<T>::up(reinterpret_cast<const T *>(a.src)[at[1]]) * static_cast<C>(a.scale) : C(0);
            if (a.residual != nullptr) y = Comp<T>::up(reinterpret_cast<const T *>(a.residual)[at[2]]) + y;
            reinterpret_cast<T *>(a.out)[at[0]] = Comp<T>::down(y);
        }
    }
}

hmr_status dropout(hmr_context_t ctx, const hmr_tensor_desc *out, const hmr_tensor_desc *src, const hmr_tensor_desc *residual,
                   double p, uint64_t seed, uint64_t offset, const uint64_t *base) {
    constexpr const char *who = "hmn_dropout";
    if (out == nullptr) return refuse(who, "out is NULL");
    if (out->ndim < 0 || out->ndim > HMR_MAX_DIMS) return refuse(who, "invalid number of dimensions " + std::to_string(out->ndim));
    if (hmr_status s = check_operand(who, "out", out, out->ndim, out->sizes, true)) return s;
    if (hmr_status s = check_operand(who, "src", src, out->ndim, out->sizes, false)) return s;
    if (residual != nullptr) {
        if (hmr_status s = check_operand(who, "residual", residual, out->ndim, out->sizes, false)) return s;
    }
    if (!is_float(out->dtype)) return refuse(who, "dropout takes floating point tensors");
    if (src->dtype != out->dtype || (residual != nullptr && residual->dtype != out->dtype)) {
        return refuse(who, "operands have different dtypes");
    }
    if (!(p >= 0.0 && p <= 1.0)) return refuse(who, "the probability has to be in 0..1");
    if (ctx == nullptr) return refuse(who, "null context");
    // The dimensions merged with respect to every operand.
    const hmr_tensor_desc *descs[3] = {out, src, residual};
    MapCall call;
    if (hmr_status s = prepare_map(call, 3, descs, nullptr)) return s;
    if (call.n == 0) return HMR_OK;
    DropoutArgs a{};
    a.out = call.ptr[0], a.src = call.ptr[1], a.residual = call.ptr[2];
    a.base = base, a.seed = seed, a.offset = offset, a.n = call.n;
    a.ndim = call.ndim;
    for (int k = 0; k < call.ndim; ++k) {
        a.size[k] = call.size[k];
        for (int o = 0; o < 3; ++o) a.stride[o][k] = call.stride[o][k];
    }
    const double threshold = std::nearbyint(p * 4294967296.0);
    const bool none = threshold >= 4294967296.0;  // p so near one that no word reaches it
    a.threshold = none ? 0 : static_cast<uint32_t>(threshold);
    a.scale = none ? 0.0 : 1.0 / (1.0 - p);
    return queue_on(ctx, who, [&](hipStream_t stream) {
        return with_float_type(out->dtype, [&](auto tag) {
            using T = typename decltype(tag)::type;
            const int64_t groups = ((a.n + 3) / 4 + kBlock - 1) / kBlock, most = int64_t{32} * ctx->compute_units;
            dropout_any_kernel<T><<<static_cast<uint32_t>(groups < most ? groups : most), kBlock, 0, stream>>>(a, none);
        });
    });
}

}  // namespace
}  // namespace nn
}  // namespace hmr

extern "C" hmr_status hmn_dropout(hmr_context_t ctx, const hmr_tensor_desc *out, const hmr_tensor_desc *src,
                                  const hmr_tensor_desc *residual, double p, uint64_t seed, uint64_t offset,
                                  const uint64_t *base) {
    return hmr::fenced([&] { return hmr::nn::dropout(ctx, out, src, residual, p, seed, offset, base); });
}
