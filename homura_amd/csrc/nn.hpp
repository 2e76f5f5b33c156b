// What the translation units of libhomura_nn share: the checks of its operands and the access to rows of elements.
// The library is linked apart from libhomura_rocm (its failure texts are its own, nn_runtime.cpp), but from the same
// headers: a context is the same struct, and its stream and its mailbox are treated as every entry point there does.
#pragma once

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <string>

#include "common.hpp"
#include "dispatch.hpp"
#include "elem.hpp"
#include "homura_nn.h"
#include "map.hpp"

namespace hmr {
namespace nn {

// ---- checks ---------------------------------------------------------------------------------------------------

inline hmr_status refuse(const char *who, const std::string &why) { return fail(HMR_INVALID, std::string(who) + ": " + why); }

inline bool is_float(int32_t dtype) { return dtype >= HMR_F16 && dtype <= HMR_F64; }
// The type statistics and states may have beside tensors of `dtype`.
inline int32_t wide_type(int32_t dtype) { return dtype == HMR_F64 ? HMR_F64 : HMR_F32; }

inline char *first(const hmr_tensor_desc &d) { return static_cast<char *>(d.data) + d.offset * dtype_size(d.dtype); }
inline char *first(const hmr_tensor_desc *d) { return d != nullptr ? first(*d) : nullptr; }

// One operand: not NULL, well formed, with these sizes (and, as an output, elements in places of their own).
inline hmr_status check_operand(const char *who, const char *name, const hmr_tensor_desc *d, int ndim, const int64_t *sizes,
                                bool output) {
    if (d == nullptr) return refuse(who, std::string(name) + " is NULL");
    int64_t n = 0;
    if (hmr_status s = check_desc(*d, n)) return s;
    if (d->ndim != ndim) {
        return refuse(who, std::string(name) + " has " + std::to_string(d->ndim) + " dimensions, not " + std::to_string(ndim));
    }
    for (int k = 0; k < ndim; ++k) {
        if (d->sizes[k] != sizes[k]) return refuse(who, std::string(name) + " has different sizes");
        if (output && n > 0 && d->sizes[k] > 1 && d->strides[k] == 0) {
            return refuse(who, std::string(name) + " is written and has elements in one place");
        }
    }
    if (n > 0 && d->data == nullptr) return refuse(who, std::string(name) + " has no memory");
    return HMR_OK;
}

inline hmr_status check_type(const char *who, const char *name, int32_t have, int32_t want, int32_t or_this) {
    if (have == want || have == or_this) return HMR_OK;
    return refuse(who, std::string(name) + " has another dtype than the operands it goes with");
}

inline hmr_status check_room(const char *who, const void *workspace, int64_t have, int64_t need) {
    if (need > 0 && (workspace == nullptr || have < need)) {
        return refuse(who, "the workspace has " + std::to_string(workspace == nullptr ? 0 : have) + " bytes, " + std::to_string(need) +
                               " are needed");
    }
    if (need > 0 && reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return refuse(who, "the workspace is not aligned to 16 bytes");
    return HMR_OK;
}

// A launch has fewer than 2^32 threads; what would take more goes to kernels that loop.
inline bool fits_launch(int64_t groups, int block) { return groups < (int64_t{1} << 32) / block; }

// ---- device side --------------------------------------------------------------------------------------------------

__device__ __forceinline__ float fma_(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
__device__ __forceinline__ double fma_(double a, double b, double c) { return __builtin_fma(a, b, c); }

// exp(v) in two parts, e and t: exp(v) = e (1 + t). e is the hardware's exp2 of the nearest f32 to v log2(e), and t what that
// rounding left of v. With it the exponential is off by some three half steps, without it by up to |v| more. Beside 16-bit
// tensors t is zero: |v| is below 104 where the result is not zero, and so many half steps of f32 are less than a 70th of the
// half step that such a tensor rounds by; the corrected form takes longer: sigmoid over [8, 2048, 4096] bf16 120 us for 108,
// norm + silu over [16384, 4096] 71 for 64; in f32 [2, 16411, 1003] 99.5 for 97. Where the product is infinite, t (which is
// then NaN or infinite) is at most 1, and e zero or infinity. e is zero where it would be below 2^-126.
template <class T>
__device__ __forceinline__ void exp_parts(float v, float &e, float &t) {
    constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f, kLn2Rest = -1.90465429995776804e-9f;
    const float p = v * kLog2e;
    e = __builtin_amdgcn_exp2f(p);
    t = 0;
    if constexpr (sizeof(T) > 2) t = fminf(fma_(p, -kLn2Rest, fma_(p, -kLn2, v)), 1.0f);
}

// sigmoid(z) and 1 - sigmoid(z), each to within seven half steps of its own, |z| more for the smaller one beside 16-bit
// sequences (exp_parts; below 2^-126 it is zero): the smaller of the two comes from exp(-|z|) itself, not from a subtraction.
template <class T>
__device__ __forceinline__ void sigmoid_pair(float z, float &a, float &rest) {
    float e, t;
    exp_parts<T>(-fabsf(z), e, t);
    if constexpr (sizeof(T) > 2) e = fma_(e, t, e);
    const float q = __builtin_amdgcn_rcpf(1.0f + e), r = e * q;
    a = z < 0.0f ? r : q;
    rest = z < 0.0f ? q : r;
}
template <class T>
__device__ __forceinline__ void sigmoid_pair(double z, double &a, double &rest) {
    const double e = exp(-fabs(z)), q = 1.0 / (1.0 + e), r = e * q;
    a = z < 0.0 ? r : q;
    rest = z < 0.0 ? q : r;
}

// V elements of type T as memory holds them, moved in accesses of up to 16 bytes. The vectors need no more alignment than
// an element has (global accesses of this target take any), so a row of odd length or an odd start costs a few split
// lines, not another kernel.
template <class T, int V>
struct Vec {
    using C = typename Comp<T>::C;
    static constexpr int kBytes = V * static_cast<int>(sizeof(T)), kWords = kBytes < 4 ? 1 : kBytes / 4;
    static constexpr int kWide = kWords % 4 == 0 ? 4 : (kWords % 2 == 0 ? 2 : 1);  // words of an access
    typedef uint32_t Access __attribute__((ext_vector_type(kWide), aligned(sizeof(T) < 4 ? sizeof(T) : 4)));
    static_assert(kBytes == 2 || kBytes % 4 == 0, "whole words, or one half");
    uint32_t w[kWords];

    // NT: past the caches, for data that is used once and larger than they are.
    template <bool NT = false>
    __device__ __forceinline__ void load(const T *p) {
        if constexpr (kBytes == 2) {
            w[0] = *reinterpret_cast<const uint16_t *>(p);
        } else {
#pragma unroll
            for (int i = 0; i < kWords / kWide; ++i) {
                const Access *q = reinterpret_cast<const Access *>(p) + i;
                const Access x = NT ? __builtin_nontemporal_load(q) : *q;
#pragma unroll
                for (int k = 0; k < kWide; ++k) w[i * kWide + k] = x[k];
            }
        }
    }
    template <bool NT = false>
    __device__ __forceinline__ void store(T *p) const {
        if constexpr (kBytes == 2) {
            *reinterpret_cast<uint16_t *>(p) = static_cast<uint16_t>(w[0]);
        } else {
#pragma unroll
            for (int i = 0; i < kWords / kWide; ++i) {
                Access x;
#pragma unroll
                for (int k = 0; k < kWide; ++k) x[k] = w[i * kWide + k];
                Access *q = reinterpret_cast<Access *>(p) + i;
                if constexpr (NT) __builtin_nontemporal_store(x, q);
                else *q = x;
            }
        }
    }
    // Element i in the computation type.
    __device__ __forceinline__ C get(int i) const {
        if constexpr (std::is_same_v<T, float>) {
            return bits_as<float>(w[i]);
        } else if constexpr (std::is_same_v<T, double>) {
            return bits_as<double>((static_cast<uint64_t>(w[2 * i + 1]) << 32) | w[2 * i]);
        } else if constexpr (std::is_same_v<T, bf16_t>) {
            return bits_as<float>(i % 2 == 0 ? w[i / 2] << 16 : w[i / 2] & 0xFFFF0000u);
        } else {
            return Comp<T>::up(T{static_cast<uint16_t>(i % 2 == 0 ? w[i / 2] : w[i / 2] >> 16)});
        }
    }
    // Computation-type values rounded into the vector.
    __device__ __forceinline__ void round(const C (&x)[V]) {
        if constexpr (std::is_same_v<T, float>) {
#pragma unroll
            for (int i = 0; i < V; ++i) w[i] = bits_as<uint32_t>(x[i]);
        } else if constexpr (std::is_same_v<T, double>) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const uint64_t b = bits_as<uint64_t>(x[i]);
                w[2 * i] = static_cast<uint32_t>(b), w[2 * i + 1] = static_cast<uint32_t>(b >> 32);
            }
        } else if constexpr (V == 1) {
            w[0] = Comp<T>::down(x[0]).bits;
        } else if constexpr (std::is_same_v<T, bf16_t>) {
#pragma unroll
            for (int i = 0; i < V; i += 2) w[i / 2] = bf16_round_pair(x[i], x[i + 1]);
        } else {
#pragma unroll
            for (int i = 0; i < V; i += 2) w[i / 2] = f16_round(x[i]).bits | (static_cast<uint32_t>(f16_round(x[i + 1]).bits) << 16);
        }
    }
    // Every element x (a value the type holds).
    __device__ __forceinline__ void fill(C x) {
        C all[V];
#pragma unroll
        for (int i = 0; i < V; ++i) all[i] = x;
        round(all);
    }
    // The vector as it is, or all zeros.
    __device__ __forceinline__ void only(bool as_it_is) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = as_it_is ? w[i] : 0;
    }
    // Makes the compiler forget what it knows of the words, so that what was computed from them is computed again where
    // it is used again instead of being kept in registers meanwhile.
    __device__ __forceinline__ void forget() {
#pragma unroll
        for (int i = 0; i < kWords; ++i) asm volatile("" : "+v"(w[i]));
    }
};

// How a kernel's large accesses treat the caches, fixed at compile time. A call that moves no more than the memory-side
// cache holds leaves everything to the caches (the next call finds its input there); a larger one loads and stores past
// them, but loads through them where rows begin inside cache lines, which neighbours then share.
enum Passing : int { kThroughCaches = 0, kPastCaches = 1, kStoresPastCaches = 2 };

inline Passing passing(int64_t bytes, bool whole_lines) {
    return bytes <= kCacheResidentBytes ? kThroughCaches : (whole_lines ? kPastCaches : kStoresPastCaches);
}

// Calls f(IntTag<Passing>).
template <class F>
void with_passing(Passing p, F &&f) {
    with_code(static_cast<int>(p), std::integer_sequence<int, kThroughCaches, kPastCaches, kStoresPastCaches>{}, f);
}

// One element of a tensor whose type is the computation type or, at run time, a narrower one.
template <class T>
__device__ __forceinline__ typename Comp<T>::C load_state(const char *p, int64_t at, bool wide) {
    using C = typename Comp<T>::C;
    if constexpr (std::is_same_v<T, C>) return reinterpret_cast<const T *>(p)[at];
    else return wide ? reinterpret_cast<const C *>(p)[at] : Comp<T>::up(reinterpret_cast<const T *>(p)[at]);
}
template <class T>
__device__ __forceinline__ void store_state(char *p, int64_t at, bool wide, typename Comp<T>::C v) {
    using C = typename Comp<T>::C;
    if constexpr (std::is_same_v<T, C>) reinterpret_cast<T *>(p)[at] = v;
    else if (wide) reinterpret_cast<C *>(p)[at] = v;
    else reinterpret_cast<T *>(p)[at] = Comp<T>::down(v);
}

}  // namespace nn
}  // namespace hmr
