// 16- and 32-bit stream types of the conditioning operators (codes.hip, trunk.hip, linear8.hip): element types by number, vector loads and
// stores that widen to / round from fp32 once.  Rounding to 16 bits is round-to-nearest-even (the compiler's conversion of a float).
#pragma once
#include "nvp_common.h"

typedef _Float16 nvp_f16;
typedef __bf16 nvp_bf16;

template <typename T, int V> struct alignas(sizeof(T) * V) nvp_vec { T v[V]; };

// V consecutive elements, widened.  `p` must be aligned to V elements.
template <typename T, int V> __device__ __forceinline__ void nvp_load(const T* __restrict__ p, float (&f)[V]) {
    const nvp_vec<T, V> t = *reinterpret_cast<const nvp_vec<T, V>*>(p);
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = (float)t.v[e];
}
template <typename T, int V> __device__ __forceinline__ void nvp_store(T* __restrict__ p, const float (&f)[V]) {
    nvp_vec<T, V> t;
#pragma unroll
    for (int e = 0; e < V; ++e) t.v[e] = (T)f[e];
    *reinterpret_cast<nvp_vec<T, V>*>(p) = t;
}

__host__ inline int nvp_type_size(int32_t type) { return type == NVP_F32 ? 4 : type == NVP_BF16 || type == NVP_F16 ? 2 : 0; }

// widest vector (in elements, <= limit) that divides d and keeps every pointer of `ored` (OR of the base addresses) aligned
__host__ inline int nvp_vec_width(int64_t d, int size, uintptr_t ored, int limit) {
    int v = limit;
    while (v > 1 && (d % v || ored % ((uintptr_t)v * size))) v >>= 1;
    return v;
}
