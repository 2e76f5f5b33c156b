// hmn_dropout: out = residual + (kept ? src / (1 - p) : 0), the mask computed where it is used.
//
// Element i is kept when word i % 4 of Philox block offset + i / 4 reaches the threshold, so a thread that owns four
// elements in a row needs one block and nothing is stored for the backward pass, which is this kernel again.
//
// A block is ten rounds of two 32 x 32 -> 64 multiplications (quarter rate): some 100 cycles of a SIMD an element and
// wave, 43 us for 67 million elements if nothing overlapped. The memory takes longer, so the work is to keep both busy.
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
__global__ void __launch_bounds__(kBlock) dropout_any_kernel(DropoutArgs a) {
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
            const bool keep = w.v[j] >= a.threshold;
            // A dropped element is not multiplied: nothing of an infinity or a NaN is left.
            C y = keep ? Comp<T>::up(reinterpret_cast<const T *>(a.src)[at[1]]) * static_cast<C>(a.scale) : C(0);
            if (a.residual != nullptr) y = Comp<T>::up(reinterpret_cast<const T *>(a.residual)[at[2]]) + y;
            reinterpret_cast<T *>(a.out)[at[0]] = Comp<T>::down(y);
        }
    }
}

// Nothing is kept: the residual, or zeros.
template <class T>
__global__ void __launch_bounds__(kBlock) dropout_none_kernel(DropoutArgs a) {
    using C = typename Comp<T>::C;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; i < a.n; i += static_cast<int64_t>(gridDim.x) * kBlock) {
        int64_t rest = i, at[2] = {0, 0};
        for (int k = a.ndim - 1; k >= 0; --k) {
            const int64_t q = rest / a.size[k], r = rest - q * a.size[k];
            at[0] += r * a.stride[0][k], at[1] += r * a.stride[2][k];
            rest = q;
        }
        C y = 0;
        if (a.residual != nullptr) y = Comp<T>::up(reinterpret_cast<const T *>(a.residual)[at[1]]) + y;
        reinterpret_cast<T *>(a.out)[at[0]] = Comp<T>::down(y);
    }
}

// Rows of elements that lie next to each other in every operand and hold whole vectors (a lone row may end inside one): a
// lane moves one vector of V elements (16 bytes) with its V / 4 blocks (half a block in f64, whose neighbour computes the
// same one). More vectors a lane were slower: 67 million bf16 elements with a residual 64 us with one, 65 with two, 69
// with four (6.3 TB/s with one, and the vector units busy for 60 % of it).
struct DropoutRows {
    DropoutArgs a;
    int64_t vectors;
    int outer;  // dimensions outside the rows
    FastDiv by_row, by[kFastDims];  // vectors of a row; the outer dimensions, innermost first
    int64_t step[3][kFastDims];
};

template <class T, bool RESIDUAL, bool PAST>
__global__ void __launch_bounds__(kBlock) dropout_rows_kernel(DropoutRows s) {
    using C = typename Comp<T>::C;
    constexpr int V = 16 / static_cast<int>(sizeof(T)), B = V >= 4 ? V / 4 : 1;
    const DropoutArgs &a = s.a;
    const uint64_t offset = a.offset + (a.base != nullptr ? *a.base : 0);
    const C scale = static_cast<C>(a.scale);
    const int64_t v = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x;
    if (v >= s.vectors) return;
    int64_t at[3] = {v * V, v * V, v * V};
    if (s.outer > 0) {  // the host has checked that the vectors' numbers fit 31 bits
        uint32_t row = divide(static_cast<uint32_t>(v), s.by_row);
        at[0] = at[1] = at[2] = static_cast<int64_t>(static_cast<uint32_t>(v) - row * s.by_row.div) * V;
        for (int k = 0; k < s.outer; ++k) {
            const uint32_t q = divide(row, s.by[k]), in = row - q * s.by[k].div;
            for (int o = 0; o < 3; ++o) at[o] += in * s.step[o][k];
            row = q;
        }
    }
    const T *src = reinterpret_cast<const T *>(a.src) + at[1], *residual = reinterpret_cast<const T *>(a.residual) + at[2];
    T *out = reinterpret_cast<T *>(a.out) + at[0];
    const bool whole = (v + 1) * V <= a.n;
    Vec<T, V> x, r;
    if (whole) {
        x.template load<PAST>(src);
        if constexpr (RESIDUAL) r.template load<PAST>(residual);
    }
    uint32_t words[V >= 4 ? V : 4];
#pragma unroll
    for (int b = 0; b < B; ++b) {
        const Word4 w = philox_block(offset + static_cast<uint64_t>(V >= 4 ? v * B + b : v / 2), a.seed);
#pragma unroll
        for (int j = 0; j < 4; ++j) words[b * 4 + j] = w.v[j];
    }
    if (V < 4 && v % 2 != 0) words[0] = words[2], words[1] = words[3];
    // A dropped element is not multiplied: nothing of an infinity or a NaN is left.
    if (whole) {
        C y[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            y[i] = words[i] >= a.threshold ? x.get(i) * scale : C(0);
            if constexpr (RESIDUAL) y[i] = r.get(i) + y[i];
        }
        x.round(y);
        x.template store<PAST>(out);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (v * V + i >= a.n) break;
            C y = words[i] >= a.threshold ? Comp<T>::up(src[i]) * scale : C(0);
            if constexpr (RESIDUAL) y = Comp<T>::up(residual[i]) + y;
            out[i] = Comp<T>::down(y);
        }
    }
}

// Queues the rows kernel if the operands are such rows.
template <class T>
bool queue_rows(hipStream_t stream, const DropoutArgs &a) {
    constexpr int V = 16 / static_cast<int>(sizeof(T));
    DropoutRows s{};
    s.a = a;
    const bool residual = a.residual != nullptr;
    const int last = a.ndim - 1, operands = residual ? 3 : 2;
    for (int o = 0; o < operands; ++o) {
        if (a.ndim > 0 && a.stride[o][last] != 1) return false;
    }
    if (a.ndim <= 1) {
        s.vectors = (a.n + V - 1) / V;
    } else {
        if (a.size[last] % V != 0 || a.ndim - 1 > kFastDims || a.n / V >= int64_t{1} << 31) return false;
        s.vectors = a.n / V;
        s.outer = a.ndim - 1;
        s.by_row = make_fastdiv(static_cast<uint32_t>(a.size[last] / V));
        for (int k = 0; k < s.outer; ++k) {
            s.by[k] = make_fastdiv(static_cast<uint32_t>(a.size[last - 1 - k]));
            for (int o = 0; o < 3; ++o) s.step[o][k] = a.stride[o][last - 1 - k];
        }
    }
    const int64_t groups = (s.vectors + kBlock - 1) / kBlock;
    if (!fits_launch(groups, kBlock)) return false;
    const uint32_t grid = static_cast<uint32_t>(groups);
    const bool past = a.n * static_cast<int64_t>(sizeof(T)) * operands > kCacheResidentBytes;
    if (residual) {
        if (past) dropout_rows_kernel<T, true, true><<<grid, kBlock, 0, stream>>>(s);
        else dropout_rows_kernel<T, true, false><<<grid, kBlock, 0, stream>>>(s);
    } else {
        if (past) dropout_rows_kernel<T, false, true><<<grid, kBlock, 0, stream>>>(s);
        else dropout_rows_kernel<T, false, false><<<grid, kBlock, 0, stream>>>(s);
    }
    return true;
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
            if (!none && queue_rows<T>(stream, a)) return;
            const int64_t groups = ((a.n + 3) / 4 + kBlock - 1) / kBlock, most = int64_t{32} * ctx->compute_units;
            const uint32_t grid = static_cast<uint32_t>(groups < most ? groups : most);
            if (none) dropout_none_kernel<T><<<grid, kBlock, 0, stream>>>(a);
            else dropout_any_kernel<T><<<grid, kBlock, 0, stream>>>(a);
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
