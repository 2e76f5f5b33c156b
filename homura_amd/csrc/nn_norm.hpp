// What the group normalisation's kernels share: their arguments, the activations and their slopes.
#pragma once

#include "nn.hpp"
#include "ops.hpp"

namespace hmr {
namespace nn {

// An [N, S, C] operand.
struct Maps {
    char *p;
    int64_t sn, ss, sc;
    __device__ __forceinline__ int64_t at(int64_t n, int64_t s, int64_t c) const { return n * sn + s * ss + c * sc; }
    template <class T>
    __device__ __forceinline__ T get(int64_t n, int64_t s, int64_t c) const {
        return reinterpret_cast<const T *>(p)[at(n, s, c)];
    }
    template <class T>
    __device__ __forceinline__ void put(int64_t n, int64_t s, int64_t c, T v) const {
        reinterpret_cast<T *>(p)[at(n, s, c)] = v;
    }
};

// An [N, groups] or [C] operand, or nothing (p null).
struct PerGroup {
    char *p;
    int64_t sn, sg;
    __device__ __forceinline__ int64_t at(int64_t n, int64_t g) const { return n * sn + g * sg; }
};
struct PerChannel {
    char *p;
    int64_t sc;
    bool wide;  // f32 beside 16-bit maps
};

struct NormArgs {
    int64_t N, S, C, G, W;  // W = C / G, the channels of a group
    Maps src, out;          // backwards, out is d_src
    Maps grad;
    PerGroup mean, rstd;
    PerChannel weight, bias, d_weight, d_bias;
    double eps;
};

// ---- activations in the computation type -------------------------------------------------------------------------

// 1 / (1 + exp(-z)) of an f32 from the hardware's exp2 and reciprocal, within three units of its last place.
__device__ __forceinline__ float logistic(float z) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504088896341f * z));
}
__device__ __forceinline__ double logistic(double z) { return 1.0 / (1.0 + exp(-z)); }

constexpr double kRootHalf = 0.70710678118654752440;       // sqrt(1/2)
constexpr double kRootTwoByPi = 0.79788456080286535588;    // sqrt(2/pi)
constexpr double kTanhInner = 0.044715;

// (1 + tanh(u)) / 2 is the logistic function of 2 u, which keeps its digits where tanh nears -1.
template <int ACT, class C>
__device__ __forceinline__ C activate(C z) {
    if constexpr (ACT == HMR_UNARY_RELU) return z < C(0) ? C(0) : z;
    else if constexpr (ACT == HMR_UNARY_SILU) return z * logistic(z);
    else if constexpr (ACT == HMR_UNARY_GELU) return C(0.5) * z * erfc(-z * C(kRootHalf));
    else if constexpr (ACT == HMR_UNARY_GELU_TANH) return z * logistic(C(2 * kRootTwoByPi) * (z + C(kTanhInner) * z * z * z));
    else return z;
}

template <int ACT, class C>
__device__ __forceinline__ C slope(C z) {
    if constexpr (ACT == HMR_UNARY_RELU) {
        return z > C(0) ? C(1) : (z != z ? z : C(0));
    } else if constexpr (ACT == HMR_UNARY_SILU) {
        const C q = logistic(z);
        return q * (C(1) + z * (C(1) - q));
    } else if constexpr (ACT == HMR_UNARY_GELU) {
        return C(0.5) * erfc(-z * C(kRootHalf)) + z * exp(C(-0.5) * z * z) * C(0.5 * kRootTwoByPi);
    } else if constexpr (ACT == HMR_UNARY_GELU_TANH) {
        const C q = logistic(C(2 * kRootTwoByPi) * (z + C(kTanhInner) * z * z * z));
        return q * (C(1) + z * (C(1) - q) * C(2 * kRootTwoByPi) * (C(1) + C(3 * kTanhInner) * z * z));
    } else {
        return C(1);
    }
}

// The weight and bias of a channel in the computation type.
template <class T>
__device__ __forceinline__ typename Comp<T>::C weight_of(const PerChannel &w, int64_t c) {
    using C = typename Comp<T>::C;
    return w.p != nullptr ? load_state<T>(w.p, c * w.sc, w.wide) : C(1);
}
template <class T>
__device__ __forceinline__ typename Comp<T>::C bias_of(const PerChannel &b, int64_t c) {
    using C = typename Comp<T>::C;
    return b.p != nullptr ? load_state<T>(b.p, c * b.sc, b.wide) : C(0);
}

// Calls f(IntTag<activation>) for a known activation.
template <class F>
bool with_activation(int32_t activation, F &&f) {
    return with_code(activation, std::integer_sequence<int, HMN_ACTIVATION_NONE, HMR_UNARY_RELU, HMR_UNARY_SILU, HMR_UNARY_GELU,
                                                       HMR_UNARY_GELU_TANH>{}, f);
}

}  // namespace nn
}  // namespace hmr
