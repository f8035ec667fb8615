// Element types of the typed entry points (feq_dtype): vector loads and stores with
// float32 values in registers, and parameters of a type known at run time.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "flasheq.h"

namespace feq {
namespace {

template <class T, int V>
struct VecOf {
    typedef T type __attribute__((ext_vector_type(V)));
    typedef type any __attribute__((aligned(sizeof(T))));      // the same in memory, aligned as an element
};
template <class T>
struct VecOf<T, 1> {
    typedef T type;
    typedef T any;
};

// Rows whose width is no multiple of a vector, or that begin at an address that is none, are read and written in
// vectors all the same (gfx950 takes a vector at any element): the last one begins V before the row's end and
// shares its first elements with the one before.  Vector q of a row of `width` >= V elements:
template <int V>
__device__ __forceinline__ int vec_begin(int q, int width) { return q * V < width - V ? q * V : width - V; }
// and the number of its first elements that belong to the vector before it (V: the row has no vector q).
template <int V>
__device__ __forceinline__ int vec_shared(int q, int width) {
    const int s = q * V - (width - V);
    return s < 0 ? 0 : s < V ? s : V;
}

// V elements at p as float32 (exact).
template <class T, int V>
__device__ __forceinline__ void load_f(const T* __restrict__ p, float (&o)[V]) {
    if constexpr (V == 1) {
        o[0] = static_cast<float>(p[0]);
    } else {
        const typename VecOf<T, V>::type u = *reinterpret_cast<const typename VecOf<T, V>::any*>(p);
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = static_cast<float>(u[j]);
    }
}

// The float32 values rounded once to T (to nearest, ties to even).
template <class T, int V>
__device__ __forceinline__ void store_f(T* __restrict__ p, const float (&o)[V]) {
    if constexpr (V == 1) {
        p[0] = static_cast<T>(o[0]);
    } else {
        typename VecOf<T, V>::type u;
#pragma unroll
        for (int j = 0; j < V; ++j) u[j] = static_cast<T>(o[j]);
        *reinterpret_cast<typename VecOf<T, V>::any*>(p) = u;
    }
}

// Element i of an array of feq_dtype dt; dt is uniform over the launch.
__device__ __forceinline__ float load_any(const void* p, int dt, int64_t i) {
    if (dt == FEQ_F32) return static_cast<const float*>(p)[i];
    if (dt == FEQ_F16) return static_cast<float>(static_cast<const _Float16*>(p)[i]);
    return static_cast<float>(static_cast<const __bf16*>(p)[i]);
}
// V elements from i of an array of feq_dtype dt.
template <int V>
__device__ __forceinline__ void load_any_v(const void* p, int dt, int64_t i, float (&o)[V]) {
    if constexpr (V == 1) {
        o[0] = load_any(p, dt, i);
    } else if (dt == FEQ_F32) {
#pragma unroll
        for (int j = 0; j < V; j += 4) {
            float f[4];
            load_f<float, 4>(static_cast<const float*>(p) + i + j, f);
#pragma unroll
            for (int u = 0; u < 4; ++u) o[j + u] = f[u];
        }
    } else if (dt == FEQ_F16) {
        load_f<_Float16, V>(static_cast<const _Float16*>(p) + i, o);
    } else {
        load_f<__bf16, V>(static_cast<const __bf16*>(p) + i, o);
    }
}
__device__ __forceinline__ void store_any(void* p, int dt, int64_t i, float v) {
    if (dt == FEQ_F32) static_cast<float*>(p)[i] = v;
    else if (dt == FEQ_F16) static_cast<_Float16*>(p)[i] = static_cast<_Float16>(v);
    else static_cast<__bf16*>(p)[i] = static_cast<__bf16>(v);
}

}  // namespace

inline int elem_size(int dt) { return dt == FEQ_F32 ? 4 : 2; }
inline bool dtype_ok(int dt) { return dt == FEQ_F32 || dt == FEQ_F16 || dt == FEQ_BF16; }
inline bool aligned_to(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// f(T{}) for the element type dt.
template <class F>
inline int with_dtype(int dt, F&& f) {
    if (dt == FEQ_F32) return f(float{});
    if (dt == FEQ_F16) return f(_Float16{});
    return f(__bf16{});
}

}  // namespace feq
