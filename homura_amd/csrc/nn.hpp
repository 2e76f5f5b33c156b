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

// ---- device side --------------------------------------------------------------------------------------------------

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
