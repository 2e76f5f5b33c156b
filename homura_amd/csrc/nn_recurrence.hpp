// What the recurrence's kernels share: their arguments and one step of the recurrence in either direction.
#pragma once

#include <initializer_list>

#include "nn.hpp"

namespace hmr {
namespace nn {

// A [B, T, C] operand.
struct Sequences {
    char *p;
    int64_t sb, st, sc;
    __device__ __forceinline__ int64_t at(int64_t b, int64_t t, int64_t c) const { return b * sb + t * st + c * sc; }
    template <class T>
    __device__ __forceinline__ T get(int64_t b, int64_t t, int64_t c) const {
        return reinterpret_cast<const T *>(p)[at(b, t, c)];
    }
    template <class T>
    __device__ __forceinline__ void put(int64_t b, int64_t t, int64_t c, T v) const {
        reinterpret_cast<T *>(p)[at(b, t, c)] = v;
    }
};

// A [B, C] operand, or nothing (p null); `wide`: f32 beside 16-bit sequences.
struct States {
    char *p;
    int64_t sb, sc;
    bool wide;
    __device__ __forceinline__ int64_t at(int64_t b, int64_t c) const { return b * sb + c * sc; }
};

struct RecurrenceArgs {
    int64_t B, T, C;
    Sequences gate, input, out;                // forwards
    Sequences grad, state, d_gate, d_input;    // backwards, with gate and input
    States entry, exit;                        // initial and last; grad_last and d_initial
    States initial;                            // backwards
    const char *lengths;                       // or nullptr
    int64_t lengths_stride;
    bool lengths64;

    // The steps of sequence b, whatever its length says inside 0..T.
    __device__ __forceinline__ int64_t steps(int64_t b) const {
        if (lengths == nullptr) return T;
        const int64_t n = lengths64 ? reinterpret_cast<const int64_t *>(lengths)[b * lengths_stride]
                                    : reinterpret_cast<const int32_t *>(lengths)[b * lengths_stride];
        return n < 0 ? 0 : (n > T ? T : n);
    }
};

__device__ __forceinline__ float fma_(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
__device__ __forceinline__ double fma_(double a, double b, double c) { return __builtin_fma(a, b, c); }

// sigmoid(z) and 1 - sigmoid(z), each to within a few units of its own last place: the smaller of the two comes from
// exp(-|z|) itself, not from a subtraction.
__device__ __forceinline__ void sigmoid_pair(float z, float &a, float &rest) {
    const float e = __builtin_amdgcn_exp2f(-1.44269504088896341f * fabsf(z)), q = __builtin_amdgcn_rcpf(1.0f + e), r = e * q;
    a = z < 0.0f ? r : q;
    rest = z < 0.0f ? q : r;
}
__device__ __forceinline__ void sigmoid_pair(double z, double &a, double &rest) {
    const double e = exp(-fabs(z)), q = 1.0 / (1.0 + e), r = e * q;
    a = z < 0.0 ? r : q;
    rest = z < 0.0 ? q : r;
}

// The factor and the addend of a step.
template <int FORM, class C>
__device__ __forceinline__ void factor_and_input(C gate, C input, C &factor, C &addend) {
    if constexpr (FORM == HMN_GATE_FACTOR) {
        factor = gate, addend = input;
    } else {
        C rest;
        sigmoid_pair(gate, factor, rest);
        addend = rest * input;
    }
}

// A step backwards: from the gradient g of the state it led to, the gradients of its gate and input and what is handed
// back to the state before it.
template <int FORM, class C>
__device__ __forceinline__ C step_back(C gate, C input, C g, C before, C &d_gate, C &d_input) {
    if constexpr (FORM == HMN_GATE_FACTOR) {
        d_gate = g * before, d_input = g;
        return gate * g;
    } else {
        C a, rest;
        sigmoid_pair(gate, a, rest);
        const C back = a * g;
        d_input = rest * g;
        d_gate = (before - input) * (back * rest);
        return back;
    }
}

// Bytes of workspace of either direction.
int64_t room_for(const hmr_tensor_desc *gate);

}  // namespace nn
}  // namespace hmr
