// Element types of the learned layers' buffers (srx_dtype of include/srx.h) and their conversions.
#pragma once
#include "srx_common.h"

typedef _Float16 srx_f16;
typedef __bf16 srx_bf16;

static inline size_t srx_dtype_size(int dtype) { return dtype == SRX_F32 ? 4 : dtype == SRX_F16 || dtype == SRX_BF16 ? 2 : 0; }

// f32 -> T: one rounding to nearest even (the type's only rounding: everything before it is held in f32)
template <class T>
__device__ __forceinline__ T srx_from_f32(float v) { return (T)v; }
template <class T>
__device__ __forceinline__ float srx_to_f32(T v) { return (float)v; }

// V consecutive elements of one row as one load / store
template <class T, int V>
struct SrxVec { typedef T type __attribute__((ext_vector_type(V))); };
template <class T>
struct SrxVec<T, 1> { typedef T type; };
template <class T, int V>
__device__ __forceinline__ float srx_elem(const typename SrxVec<T, V>::type &v, int i) {
    if constexpr (V == 1) return srx_to_f32<T>(v); else return srx_to_f32<T>(v[i]);
}
template <class T, int V>
__device__ __forceinline__ typename SrxVec<T, V>::type srx_pack(const float (&f)[V]) {
    typename SrxVec<T, V>::type r;
    if constexpr (V == 1) r = srx_from_f32<T>(f[0]);
    else {
#pragma unroll
        for (int i = 0; i < V; i++) r[i] = srx_from_f32<T>(f[i]);
    }
    return r;
}

static inline bool srx_aligned(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

// A launch takes less than 2^32 threads along a dimension
static inline bool srx_grid_fits(int64_t blocks, int threads) { return blocks < (1ll << 32) / threads; }
