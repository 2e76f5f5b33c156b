// hmn_group_norm and hmn_group_norm_backward over [N, S, C], the channels last and in `groups` equal runs.
#include "nn_norm.hpp"

namespace hmr {
namespace nn {
namespace {

// The sum of every lane's value, in every lane of the workgroup, added in a fixed order.
__device__ __forceinline__ double workgroup_sum(double v) {
    __shared__ double sums[kBlock / 64];
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = v;
    __syncthreads();
    double all = 0;
#pragma unroll
    for (int k = 0; k < kBlock / 64; ++k) all += sums[k];
    return all;
}

// ---- one workgroup per group ---------------------------------------------------------------------------------
//
// Channels that do not lie next to each other, and short maps of huge groups: three passes over a group, element by
// element.

template <class T, int ACT>
__global__ void __launch_bounds__(kBlock) norm_kernel(NormArgs a) {
    using C = typename Comp<T>::C;
    const int64_t m = a.S * a.W;
    for (int64_t k = blockIdx.x; k < a.N * a.G; k += gridDim.x) {
        const int64_t n = k / a.G, g = k - n * a.G, c0 = g * a.W;
        double sum = 0;
        for (int64_t i = threadIdx.x; i < m; i += kBlock) sum += Comp<T>::up(a.src.get<T>(n, i / a.W, c0 + i % a.W));
        const double mean = workgroup_sum(sum) / static_cast<double>(m);
        sum = 0;
        for (int64_t i = threadIdx.x; i < m; i += kBlock) {
            const double d = Comp<T>::up(a.src.get<T>(n, i / a.W, c0 + i % a.W)) - mean;
            sum += d * d;
        }
        const double rstd = 1.0 / sqrt(workgroup_sum(sum) / static_cast<double>(m) + a.eps);
        if (threadIdx.x == 0) {
            if (a.mean.p != nullptr) reinterpret_cast<C *>(a.mean.p)[a.mean.at(n, g)] = static_cast<C>(mean);
            if (a.rstd.p != nullptr) reinterpret_cast<C *>(a.rstd.p)[a.rstd.at(n, g)] = static_cast<C>(rstd);
        }
        for (int64_t i = threadIdx.x; i < m; i += kBlock) {
            const int64_t s = i / a.W, c = c0 + i % a.W;
            const C hat = static_cast<C>((Comp<T>::up(a.src.get<T>(n, s, c)) - mean) * rstd);
            a.out.put<T>(n, s, c, Comp<T>::down(activate<T, ACT>(hat * weight_of<T>(a.weight, c) + bias_of<T>(a.bias, c))));
        }
    }
}

template <class T, int ACT>
__global__ void __launch_bounds__(kBlock) norm_back_kernel(NormArgs a) {
    using C = typename Comp<T>::C;
    const int64_t m = a.S * a.W;
    for (int64_t k = blockIdx.x; k < a.N * a.G; k += gridDim.x) {
        const int64_t n = k / a.G, g = k - n * a.G, c0 = g * a.W;
        const C mean = reinterpret_cast<const C *>(a.mean.p)[a.mean.at(n, g)], rstd = reinterpret_cast<const C *>(a.rstd.p)[a.rstd.at(n, g)];
        auto parts = [&](int64_t i, C &hat, C &d) {
            const int64_t s = i / a.W, c = c0 + i % a.W;
            const C w = weight_of<T>(a.weight, c);
            hat = (Comp<T>::up(a.src.get<T>(n, s, c)) - mean) * rstd;
            d = w * Comp<T>::up(a.grad.get<T>(n, s, c)) * slope<T, ACT>(hat * w + bias_of<T>(a.bias, c));
        };
        double d_sum = 0, dh_sum = 0;
        for (int64_t i = threadIdx.x; i < m; i += kBlock) {
            C hat, d;
            parts(i, hat, d);
            d_sum += d, dh_sum += static_cast<double>(d) * hat;
        }
        const C d_mean = static_cast<C>(workgroup_sum(d_sum) / static_cast<double>(m)), dh_mean = static_cast<C>(workgroup_sum(dh_sum) / static_cast<double>(m));
        for (int64_t i = threadIdx.x; i < m; i += kBlock) {
            C hat, d;
            parts(i, hat, d);
            a.out.put<T>(n, i / a.W, c0 + i % a.W, Comp<T>::down(rstd * (d - d_mean - hat * dh_mean)));
        }
    }
}

// One workgroup per channel.
template <class T, int ACT>
__global__ void __launch_bounds__(kBlock) norm_weights_kernel(NormArgs a) {
    using C = typename Comp<T>::C;
    for (int64_t c = blockIdx.x; c < a.C; c += gridDim.x) {
        const C w = weight_of<T>(a.weight, c), b = bias_of<T>(a.bias, c);
        double d_sum = 0, dh_sum = 0;
        for (int64_t i = threadIdx.x; i < a.N * a.S; i += kBlock) {
            const int64_t n = i / a.S, s = i - n * a.S, g = c / a.W;
            const C mean = reinterpret_cast<const C *>(a.mean.p)[a.mean.at(n, g)], rstd = reinterpret_cast<const C *>(a.rstd.p)[a.rstd.at(n, g)];
            const C hat = (Comp<T>::up(a.src.get<T>(n, s, c)) - mean) * rstd;
            const C d = Comp<T>::up(a.grad.get<T>(n, s, c)) * slope<T, ACT>(hat * w + b);
            d_sum += d, dh_sum += static_cast<double>(d) * hat;
        }
        d_sum = workgroup_sum(d_sum), dh_sum = workgroup_sum(dh_sum);
        if (threadIdx.x == 0) {
            if (a.d_bias.p != nullptr) store_state<T>(a.d_bias.p, c * a.d_bias.sc, a.d_bias.wide, static_cast<C>(d_sum));
            if (a.d_weight.p != nullptr) store_state<T>(a.d_weight.p, c * a.d_weight.sc, a.d_weight.wide, static_cast<C>(dh_sum));
        }
    }
}

// ---- checks ----------------------------------------------------------------------------------------------------

struct Named {
    const char *name;
    const hmr_tensor_desc *d;
    bool output;
};

hmr_status check_norm(const char *who, const hmr_tensor_desc *src, int64_t groups, int32_t activation,
                      std::initializer_list<Named> maps, std::initializer_list<Named> statistics,
                      std::initializer_list<Named> channels) {
    if (src == nullptr) return refuse(who, "src is NULL");
    if (hmr_status s = check_operand(who, "src", src, 3, src->sizes, false)) return s;
    if (!is_float(src->dtype)) return refuse(who, "group normalisation takes floating point tensors");
    if (groups < 1 || src->sizes[2] % groups != 0) {
        return refuse(who, std::to_string(src->sizes[2]) + " channels do not make " + std::to_string(groups) + " groups");
    }
    if (!with_activation(activation, [](auto) {})) return refuse(who, "unknown activation " + std::to_string(activation));
    for (const Named &x : maps) {
        if (hmr_status s = check_operand(who, x.name, x.d, 3, src->sizes, x.output)) return s;
        if (x.d->dtype != src->dtype) return refuse(who, std::string(x.name) + " has another dtype than src");
    }
    const int64_t per_group[2] = {src->sizes[0], groups};
    for (const Named &x : statistics) {
        if (x.d == nullptr && x.output) continue;
        if (hmr_status s = check_operand(who, x.name, x.d, 2, per_group, x.output)) return s;
        if (x.d->dtype != wide_type(src->dtype)) return refuse(who, std::string(x.name) + " has to be F32 (F64 beside F64)");
    }
    for (const Named &x : channels) {
        if (x.d == nullptr) continue;
        if (hmr_status s = check_operand(who, x.name, x.d, 1, src->sizes + 2, x.output)) return s;
        if (hmr_status s = check_type(who, x.name, x.d->dtype, src->dtype, wide_type(src->dtype))) return s;
    }
    return HMR_OK;
}

Maps maps_of(const hmr_tensor_desc *d) { return d ? Maps{first(*d), d->strides[0], d->strides[1], d->strides[2]} : Maps{}; }
PerGroup per_group(const hmr_tensor_desc *d) { return d ? PerGroup{first(*d), d->strides[0], d->strides[1]} : PerGroup{}; }
PerChannel per_channel(const hmr_tensor_desc *d) { return d ? PerChannel{first(*d), d->strides[0], d->dtype == HMR_F32} : PerChannel{}; }

NormArgs norm_args(const hmr_tensor_desc *src, int64_t groups) {
    NormArgs a{};
    a.N = src->sizes[0], a.S = src->sizes[1], a.C = src->sizes[2], a.G = groups, a.W = a.C / groups;
    a.src = maps_of(src);
    return a;
}

// Workspace for whichever kernels the operands' strides will call for.
int64_t norm_room(const hmr_tensor_desc *src, int64_t groups, bool backward) {
    const NormArgs a = norm_args(src, groups);
    if (a.C == 0) return 0;
    const int64_t rows = norm_rows_room(a, src->dtype, backward), maps = norm_maps_room(a, src->dtype, backward);
    return rows > maps ? rows : maps;
}

uint32_t grid_of(hmr_context_t ctx, int64_t groups) {
    const int64_t most = int64_t{64} * ctx->compute_units;
    return static_cast<uint32_t>(groups < most ? groups : most);
}

hmr_status forward(hmr_context_t ctx, const hmr_tensor_desc *out, const hmr_tensor_desc *mean, const hmr_tensor_desc *rstd,
                   const hmr_tensor_desc *src, const hmr_tensor_desc *weight, const hmr_tensor_desc *bias, int64_t groups, double eps,
                   int32_t activation, void *workspace, int64_t workspace_bytes) {
    constexpr const char *who = "hmn_group_norm";
    if (hmr_status s = check_norm(who, src, groups, activation, {{"out", out, true}}, {{"mean", mean, true}, {"rstd", rstd, true}},
                                  {{"weight", weight, false}, {"bias", bias, false}})) {
        return s;
    }
    if (!(eps >= 0.0) || std::isinf(eps)) return refuse(who, "eps has to be a number of at least zero");
    if (hmr_status s = check_room(who, workspace, workspace_bytes, norm_room(src, groups, false))) return s;
    if (ctx == nullptr) return refuse(who, "null context");
    NormArgs a = norm_args(src, groups);
    a.out = maps_of(out), a.mean = per_group(mean), a.rstd = per_group(rstd);
    a.weight = per_channel(weight), a.bias = per_channel(bias), a.eps = eps;
    // Without positions there are only the statistics to write.
    if (a.N == 0 || a.C == 0 || (a.S == 0 && a.mean.p == nullptr && a.rstd.p == nullptr)) return HMR_OK;
    return queue_on(ctx, who, [&](hipStream_t stream) {
        if (queue_norm_rows(stream, src->dtype, a, activation, workspace, false)) return true;
        if (queue_norm_maps(stream, src->dtype, a, activation, workspace, false)) return true;
        return with_float_type(src->dtype, [&](auto tag) {
            using T = typename decltype(tag)::type;
            with_activation(activation, [&](auto act) {
                norm_kernel<T, decltype(act)::value><<<grid_of(ctx, a.N * a.G), kBlock, 0, stream>>>(a);
            });
        });
    });
}

hmr_status backward(hmr_context_t ctx, const hmr_tensor_desc *d_src, const hmr_tensor_desc *d_weight, const hmr_tensor_desc *d_bias,
                    const hmr_tensor_desc *grad, const hmr_tensor_desc *src, const hmr_tensor_desc *mean, const hmr_tensor_desc *rstd,
                    const hmr_tensor_desc *weight, const hmr_tensor_desc *bias, int64_t groups, int32_t activation, void *workspace,
                    int64_t workspace_bytes) {
    constexpr const char *who = "hmn_group_norm_backward";
    if (hmr_status s = check_norm(who, src, groups, activation, {{"d_src", d_src, true}, {"grad", grad, false}},
                                  {{"mean", mean, false}, {"rstd", rstd, false}},
                                  {{"weight", weight, false}, {"bias", bias, false}, {"d_weight", d_weight, true}, {"d_bias", d_bias, true}})) {
        return s;
    }
    if (hmr_status s = check_room(who, workspace, workspace_bytes, norm_room(src, groups, true))) return s;
    if (ctx == nullptr) return refuse(who, "null context");
    NormArgs a = norm_args(src, groups);
    a.out = maps_of(d_src), a.grad = maps_of(grad), a.mean = per_group(mean), a.rstd = per_group(rstd);
    a.weight = per_channel(weight), a.bias = per_channel(bias), a.d_weight = per_channel(d_weight), a.d_bias = per_channel(d_bias);
    if (a.C == 0) return HMR_OK;
    return queue_on(ctx, who, [&](hipStream_t stream) {
        if (queue_norm_rows(stream, src->dtype, a, activation, workspace, true)) return true;
        if (queue_norm_maps(stream, src->dtype, a, activation, workspace, true)) return true;
        return with_float_type(src->dtype, [&](auto tag) {
            using T = typename decltype(tag)::type;
            with_activation(activation, [&](auto act) {
                constexpr int ACT = decltype(act)::value;
                if (a.N * a.S > 0) norm_back_kernel<T, ACT><<<grid_of(ctx, a.N * a.G), kBlock, 0, stream>>>(a);
                if (a.d_weight.p != nullptr || a.d_bias.p != nullptr) {
                    norm_weights_kernel<T, ACT><<<grid_of(ctx, a.C), kBlock, 0, stream>>>(a);
                }
            });
        });
    });
}

}  // namespace
}  // namespace nn
}  // namespace hmr

extern "C" {

hmr_status hmn_group_norm_workspace(const hmr_tensor_desc *src, int64_t groups, int32_t backward, int64_t *bytes) {
    return hmr::fenced([&] {
        constexpr const char *who = "hmn_group_norm_workspace";
        if (src == nullptr || bytes == nullptr) return hmr::nn::refuse(who, "an argument is NULL");
        int64_t n = 0;
        if (hmr_status s = hmr::check_desc(*src, n)) return s;
        if (src->ndim != 3) return hmr::nn::refuse(who, "src has " + std::to_string(src->ndim) + " dimensions, not 3");
        if (!hmr::nn::is_float(src->dtype)) return hmr::nn::refuse(who, "group normalisation takes floating point tensors");
        if (groups < 1 || src->sizes[2] % groups != 0) {
            return hmr::nn::refuse(who, std::to_string(src->sizes[2]) + " channels do not make " + std::to_string(groups) + " groups");
        }
        *bytes = hmr::nn::norm_room(src, groups, backward != 0);
        return HMR_OK;
    });
}

hmr_status hmn_group_norm(hmr_context_t ctx, const hmr_tensor_desc *out, const hmr_tensor_desc *mean, const hmr_tensor_desc *rstd,
                          const hmr_tensor_desc *src, const hmr_tensor_desc *weight, const hmr_tensor_desc *bias, int64_t groups,
                          double eps, int32_t activation, void *workspace, int64_t workspace_bytes) {
    return hmr::fenced([&] {
        return hmr::nn::forward(ctx, out, mean, rstd, src, weight, bias, groups, eps, activation, workspace, workspace_bytes);
    });
}

hmr_status hmn_group_norm_backward(hmr_context_t ctx, const hmr_tensor_desc *d_src, const hmr_tensor_desc *d_weight,
                                   const hmr_tensor_desc *d_bias, const hmr_tensor_desc *grad, const hmr_tensor_desc *src,
                                   const hmr_tensor_desc *mean, const hmr_tensor_desc *rstd, const hmr_tensor_desc *weight,
                                   const hmr_tensor_desc *bias, int64_t groups, int32_t activation, void *workspace,
                                   int64_t workspace_bytes) {
    return hmr::fenced([&] {
        return hmr::nn::backward(ctx, d_src, d_weight, d_bias, grad, src, mean, rstd, weight, bias, groups, activation, workspace,
                                 workspace_bytes);
    });
}

}  // extern "C"
