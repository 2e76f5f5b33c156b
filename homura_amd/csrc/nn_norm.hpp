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

// 1 / (1 + exp(-z)) of an f32 from the hardware's exp2 and reciprocal, within seven half steps, beside 16-bit tensors |z| more
// where z is negative (exp_parts; below 2^-126 it is zero). Where exp(-z) is past f32, e is infinite and 1 + t is not zero.
template <class T>
__device__ __forceinline__ float logistic(float z) {
    float e, t;
    exp_parts<T>(-z, e, t);
    return __builtin_amdgcn_rcpf(sizeof(T) > 2 ? fma_(e, 1.0f + t, 1.0f) : 1.0f + e);
}
template <class T>
__device__ __forceinline__ double logistic(double z) { return 1.0 / (1.0 + exp(-z)); }

constexpr double kRootHalf = 0.70710678118654752440;       // sqrt(1/2)
constexpr double kRootTwoByPi = 0.79788456080286535588;    // sqrt(2/pi)
constexpr double kTanhInner = 0.044715;

// (1 + tanh(u)) / 2 is the logistic function of 2 u, which keeps its digits where tanh nears -1: gelu_tanh's 2 u.
template <class C>
__device__ __forceinline__ C tanh_argument(C z) {
    return z * fma_(C(2 * kRootTwoByPi * kTanhInner) * z, z, C(2 * kRootTwoByPi));
}

// The normal distribution below z, and exp(-z^2 / 2). With a = |z| the tail beyond a is exp(-a^2 / 2) E(a), and E, which
// falls slowly from 1/2 to 1 / (a sqrt(2 pi)), is t P(t) with t = 1 / (1 + 0.34 a): P is the polynomial of degree 8 of the
// least relative error on a in 0..15, found by weighted least squares on 4000 Chebyshev points (half a unit of 2^-24; seven
// as evaluated in f32, its 0.34 among the values that gave the least). The exponential's argument adds 1.5 z^2 units. With
// the library's error function in its place [16384, 4096] bf16 took 118 us and its gradient for half as many rows 90, with
// this 79 and 54.
__device__ __forceinline__ void normal(float z, float &below, float &bell) {
    constexpr float kP[9] = {0.135622576f, 0.13607347f, 0.115497872f, 0.114096098f, -0.041554004f, 0.197331294f, -0.26867196f, 0.137242302f, -0.0256376024f};
    const float t = __builtin_amdgcn_rcpf(fma_(0.34f, fabsf(z), 1.0f));
    bell = __builtin_amdgcn_exp2f(z * z * -0.72134752044448170f);
    float p = kP[8];
#pragma unroll
    for (int k = 7; k >= 0; --k) p = fma_(p, t, kP[k]);
    const float tail = bell * (t * p);
    below = z < 0.0f ? tail : 1.0f - tail;
}
__device__ __forceinline__ void normal(double z, double &below, double &bell) {
    below = 0.5 * erfc(-z * kRootHalf), bell = exp(-0.5 * z * z);
}

template <class T, int ACT, class C>
__device__ __forceinline__ C activate(C z) {
    if constexpr (ACT == HMR_UNARY_RELU) {
        return z < C(0) ? C(0) : z;
    } else if constexpr (ACT == HMR_UNARY_SILU) {
        return z * logistic<T>(z);
    } else if constexpr (ACT == HMR_UNARY_GELU) {
        C below, bell;
        normal(z, below, bell);
        return z * below;
    } else if constexpr (ACT == HMR_UNARY_GELU_TANH) {
        return z * logistic<T>(tanh_argument(z));
    } else {
        return z;
    }
}

template <class T, int ACT, class C>
__device__ __forceinline__ C slope(C z) {
    if constexpr (ACT == HMR_UNARY_RELU) {
        return z > C(0) ? C(1) : (z != z ? z : C(0));
    } else if constexpr (ACT == HMR_UNARY_SILU) {
        const C q = logistic<T>(z);
        return fma_(z * q, C(1) - q, q);
    } else if constexpr (ACT == HMR_UNARY_GELU) {
        C below, bell;
        normal(z, below, bell);
        return fma_(z * bell, C(0.5 * kRootTwoByPi), below);
    } else if constexpr (ACT == HMR_UNARY_GELU_TANH) {
        // The factor of q (1 - q) is five where that is a tenth: beside F32 and F64 tensors 1 - q is not a difference.
        C q, rest;
        if constexpr (sizeof(T) == 2) q = logistic<T>(tanh_argument(z)), rest = C(1) - q;
        else sigmoid_pair<T>(tanh_argument(z), q, rest);
        // Far out, where q (1 - q) is zero, z^2 is kept finite.
        return fma_(z * q * rest, fma_(C(6 * kRootTwoByPi * kTanhInner), fmin(z * z, C(1e30)), C(2 * kRootTwoByPi)), q);
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
__host__ __device__ __forceinline__ bool with_activation(int32_t activation, F &&f) {
    switch (activation) {
        case HMN_ACTIVATION_NONE: f(IntTag<HMN_ACTIVATION_NONE>{}); return true;
        case HMR_UNARY_RELU: f(IntTag<HMR_UNARY_RELU>{}); return true;
        case HMR_UNARY_SILU: f(IntTag<HMR_UNARY_SILU>{}); return true;
        case HMR_UNARY_GELU: f(IntTag<HMR_UNARY_GELU>{}); return true;
        case HMR_UNARY_GELU_TANH: f(IntTag<HMR_UNARY_GELU_TANH>{}); return true;
        default: return false;
    }
}
// The same choice on the device, once for V elements (the activation is the launch's, so that nothing diverges).
template <class T, int V, class C>
__device__ __forceinline__ void activate_all(int32_t activation, C (&z)[V]) {
    with_activation(activation, [&](auto act) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            z[i] = activate<T, decltype(act)::value>(z[i]);
            // The 64-bit error function's many intermediate values, of one element at a time.
            if constexpr (decltype(act)::value == HMR_UNARY_GELU && sizeof(C) == 8) __builtin_amdgcn_sched_barrier(0);
        }
    });
}
template <class T, int V, class C>
__device__ __forceinline__ void slope_all(int32_t activation, C (&z)[V]) {
    with_activation(activation, [&](auto act) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            z[i] = slope<T, decltype(act)::value>(z[i]);
            // The 64-bit error function's many intermediate values, of one element at a time.
            if constexpr (decltype(act)::value == HMR_UNARY_GELU && sizeof(C) == 8) __builtin_amdgcn_sched_barrier(0);
        }
    });
}

// ---- sums over lanes ------------------------------------------------------------------------------------------------

template <int CTRL>
__device__ __forceinline__ float dpp_move(float v) {
    return bits_as<float>(__builtin_amdgcn_update_dpp(0, bits_as<int>(v), CTRL, 0xF, 0xF, true));
}
template <int CTRL>
__device__ __forceinline__ double dpp_move(double v) {
    const uint64_t b = bits_as<uint64_t>(v);
    const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(static_cast<uint32_t>(b)), CTRL, 0xF, 0xF, true));
    const uint32_t hi = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(static_cast<uint32_t>(b >> 32)), CTRL, 0xF, 0xF, true));
    return bits_as<double>((static_cast<uint64_t>(hi) << 32) | lo);
}
// The sum over each aligned run of `lanes` lanes (a power of two up to 64, the same for the whole wave), in every one of
// them. Within 16 lanes neighbours meet through cross-lane moves of the vector unit: pairs, quads, then mirrored halves
// (whose lanes agree by then), so that the order does not depend on the lane.
template <class A>
__device__ __forceinline__ A lanes_sum(A v, int lanes) {
    if (lanes > 1) v += dpp_move<0xB1>(v);    // quad_perm [1, 0, 3, 2]
    if (lanes > 2) v += dpp_move<0x4E>(v);    // quad_perm [2, 3, 0, 1]
    if (lanes > 4) v += dpp_move<0x141>(v);   // row_half_mirror
    if (lanes > 8) v += dpp_move<0x140>(v);   // row_mirror
    if (lanes > 16) v += __shfl_xor(v, 16, 64);
    if (lanes > 32) v += __shfl_xor(v, 32, 64);
    return v;
}

// 1 / sqrt(v) of a f64 from the hardware's estimate and two Newton steps (an f64 square root and division take some
// thirty-five instructions, this a dozen); 0 and infinity, where the steps make NaN of them, keep the estimate.
__device__ __forceinline__ double reciprocal_root(double v) {
    const double seed = __builtin_amdgcn_rsq(v);
    double y = seed;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const double e = __builtin_fma(-v * y, y, 1.0);
        y = __builtin_fma(0.5 * y, e, y);
    }
    return y == y ? y : seed;
}

// (x - mean) * rstd. In f32 the mean is subtracted as the nearest value and what is left of it, so that the difference
// keeps its digits where x is near a mean that is far from zero.
template <class C>
struct Centre;
template <>
struct Centre<float> {
    float near, scale, rest;
    Centre() = default;
    __device__ __forceinline__ Centre(double mean, double rstd) : near(static_cast<float>(mean)), scale(static_cast<float>(rstd)) {
        rest = static_cast<float>(static_cast<double>(near) - mean) * scale;
    }
    __device__ __forceinline__ float hat(float x) const { return fma_(x - near, scale, rest); }
};
template <>
struct Centre<double> {
    double mean, scale;
    Centre() = default;
    __device__ __forceinline__ Centre(double m, double rstd) : mean(m), scale(rstd) {}
    __device__ __forceinline__ double hat(double x) const { return (x - mean) * scale; }
};

// The weights or biases of V channels, which lie next to each other; `otherwise` without a tensor.
template <class T, int V>
__device__ __forceinline__ void load_channels(const PerChannel &w, int64_t c, typename Comp<T>::C otherwise, typename Comp<T>::C (&x)[V]) {
    if (w.p == nullptr) {
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = otherwise;
    } else if (!w.wide) {
        Vec<T, V> r;
        r.load(reinterpret_cast<const T *>(w.p) + c);
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = r.get(i);
    } else {
        Vec<typename Comp<T>::C, V> r;
        r.load(reinterpret_cast<const typename Comp<T>::C *>(w.p) + c);
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = r.get(i);
    }
}

// Whether the fast kernels take the operands: everything that has channels has them next to each other.
inline bool channels_adjacent(const NormArgs &a, bool backward) {
    auto dense = [](const PerChannel &w) { return w.p == nullptr || w.sc == 1; };
    return a.src.sc == 1 && a.out.sc == 1 && (!backward || a.grad.sc == 1) && dense(a.weight) && dense(a.bias);
}

// ---- rows: a group in the registers of a wave or a workgroup ------------------------------------------------------------
//
// Where the elements of a group fit, one pass reads, reduces and writes them. A group's vectors (V channels each, so V
// divides a group's channels) are spread over `lanes` lanes, M to a lane; a wave holds as many groups as fit side by side,
// all of them in one row of channels where there are enough, else from several rows. Each lane keeps its channels from
// row to row, so that the weights stay in registers (while they are few) and, backwards, the sums for the weights'
// gradients do too: they leave the workgroup once, as a row of partial sums that a second launch adds up in order.
struct RowsPlan {
    int32_t v, m;         // vector width and vectors of a lane; m == 0: the groups do not fit
    bool wide;            // a workgroup per group rather than lanes of a wave
    int32_t lanes;        // of a group
    int32_t vectors;      // of a group
    int32_t per_position; // vectors of a group at one position
    int32_t rows;         // of channels side by side in a wave
    int64_t blocks;       // of groups, across a row
    int64_t walkers;      // workgroups that share a block's rows
};
RowsPlan rows_plan(const NormArgs &a, int32_t dtype, bool backward);

// ---- maps: groups spread over workgroups --------------------------------------------------------------------------------
//
// Larger groups take two passes over the maps, the second one out of the memory-side cache where they fit it. A
// workgroup takes every `chunks`-th run of positions of up to 256 vectors of channels, so that all of them together move
// through memory in its order; lane (r, l) takes every `slots`-th position of a run and V channels of it. The first pass
// leaves the workgroup's sums (per group forwards, per channel backwards), the second one adds up what concerns it, in
// order, and writes.
struct MapsPlan {
    int32_t v;
    int32_t lanes, slots;  // across channels and positions
    int64_t blocks;        // of channels
    int64_t chunks;        // workgroups that share a block of channels of one map
    int64_t run;           // positions that a workgroup takes at a time
};
MapsPlan maps_plan(const NormArgs &a, int32_t dtype);

// Queue the kernels (nn_norm_rows.hip, nn_norm_maps.hip); false: the shape is not theirs.
bool queue_norm_rows(hipStream_t stream, int32_t dtype, const NormArgs &a, int32_t activation, void *room, bool backward);
bool queue_norm_maps(hipStream_t stream, int32_t dtype, const NormArgs &a, int32_t activation, void *room, bool backward);
int64_t norm_rows_room(const NormArgs &a, int32_t dtype, bool backward);
int64_t norm_maps_room(const NormArgs &a, int32_t dtype, bool backward);

// The sums of d and d * hat for the weights' gradients: a lane adds up its rows or positions in the computation type, f32 ones
// in runs of kMostRun. k additions in a row are off by up to k half steps (in the mean square 2048 of them by 18, 32 by 2 and
// pairwise sums by 1); a run is added to the runs before it without losing anything, the next one begins with what that
// addition rounded away. [65536, 4096] bf16 takes 296 us with it as without; runs added in f64 took 338 where each was a
// workgroup's of its own.
constexpr int kMostRun = 32;
// all += run; run becomes what the sum's rounding left of it (nothing where the sum is not finite).
template <class C>
__device__ __forceinline__ void add_run(C &all, C &run) {
    const C sum = all + run, part = sum - all, left = (all - (sum - part)) + (run - part);
    all = sum, run = left - left == C(0) ? left : C(0);
}

// The weights' gradients from `parts` rows of partial sums ([2][parts][C]: the weights', then the biases'). A workgroup of
// kBlock lanes adds up 16 channels: sixteen threads a channel take every sixteenth part in order, eight of each sum in flight,
// then the sixteen are added.
constexpr int kSumChannels = 16, kSumSlices = kBlock / kSumChannels;

template <class T>
__device__ __forceinline__ void sum_channels(const NormArgs &a, const typename Comp<T>::C *partial, int64_t parts, int64_t block) {
    using C = typename Comp<T>::C;
    __shared__ double slices[2][kSumSlices][kSumChannels];
    const int in = threadIdx.x % kSumChannels, slice = threadIdx.x / kSumChannels;
    const int64_t c = block * kSumChannels + in;
    double total[2] = {0, 0};
    if (c < a.C) {
        constexpr int kAhead = 8;
        for (int64_t k = slice; k < parts; k += kAhead * kSumSlices) {
            C x[2][kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                const int64_t part = k + j * kSumSlices;
                x[0][j] = x[1][j] = 0;
                if (part < parts) x[0][j] = partial[part * a.C + c], x[1][j] = partial[(parts + part) * a.C + c];
            }
#pragma unroll
            for (int j = 0; j < kAhead; ++j) total[0] += x[0][j], total[1] += x[1][j];
        }
    }
    slices[0][slice][in] = total[0], slices[1][slice][in] = total[1];
    __syncthreads();
    if (slice < 2 && c < a.C) {
        double sum = 0;
#pragma unroll
        for (int k = 0; k < kSumSlices; ++k) sum += slices[slice][k][in];
        const PerChannel &to = slice == 0 ? a.d_weight : a.d_bias;
        if (to.p != nullptr) store_state<T>(to.p, c * to.sc, to.wide, static_cast<C>(sum));
    }
}

}  // namespace nn
}  // namespace hmr
