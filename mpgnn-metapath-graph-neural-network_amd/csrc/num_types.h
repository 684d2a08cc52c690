// Element types of the operators that take fp32, bf16 and fp16 tensors (enum mpgnn_dtype): the
// device types, 16-byte vectors of them, and the argument checks their entry points share.
// Arithmetic is fp32 (or wider) everywhere: a 16-bit element is widened when it is read and
// rounded once, to nearest even, when the result is written.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "mpgnn_rgcn.h"

namespace mpgnn {

void set_last_error_cstr(const char* msg) noexcept;  // plan.cpp

template <typename T, int V>
struct VecOf {
    typedef T type __attribute__((ext_vector_type(V)));
};
template <typename T, int V>
__device__ __forceinline__ void load_vec(float (&dst)[V], const T* p) {
    const typename VecOf<T, V>::type v = *reinterpret_cast<const typename VecOf<T, V>::type*>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) dst[i] = (float)v[i];
}

template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const float (&src)[V]) {
    typename VecOf<T, V>::type v;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = (T)src[i];
    *reinterpret_cast<typename VecOf<T, V>::type*>(p) = v;
}

inline int dtype_bytes(int32_t dtype) {
    return dtype == MPGNN_F32 ? 4 : (dtype == MPGNN_BF16 || dtype == MPGNN_F16) ? 2 : 0;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

inline int32_t arg_error(const char* msg) noexcept {
    set_last_error_cstr(msg);
    return MPGNN_ERR_ARG;
}

inline int32_t unsupported(const char* msg) noexcept {
    set_last_error_cstr(msg);
    return MPGNN_ERR_UNSUPPORTED;
}

inline int32_t launch_status(const char* what) noexcept {
    if (hipGetLastError() == hipSuccess) return MPGNN_OK;
    set_last_error_cstr(what);
    return MPGNN_ERR_HIP;
}

}  // namespace mpgnn
