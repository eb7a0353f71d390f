// 16- and 32-bit stream types of the conditioning operators (codes.hip, trunk.hip, linear8.hip): element types by number, vector loads and
// stores that widen to / round from fp32 once.  Rounding to 16 bits is round-to-nearest-even (the compiler's conversion of a float).
#pragma once
#include "nvp_common.h"

typedef _Float16 nvp_f16;
typedef __bf16 nvp_bf16;

template <typename T, int V> struct nvp_vec { T v[V]; };

// V consecutive elements at any element address.  Global memory takes 16-byte accesses at unaligned addresses (amdhsa runs in unaligned access mode, which the
// compiler assumes: one global_load_dwordx4 / global_store_dwordx4), so rows of odd widths need no path of their own.
template <typename T, int V> __device__ __forceinline__ nvp_vec<T, V> nvp_load_raw(const T* __restrict__ p) {
    nvp_vec<T, V> t;
    __builtin_memcpy(&t, p, sizeof(t));
    return t;
}
template <typename T, int V> __device__ __forceinline__ void nvp_load(const T* __restrict__ p, float (&f)[V]) {
    const nvp_vec<T, V> t = nvp_load_raw<T, V>(p);
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = (float)t.v[e];
}
template <typename T, int V> __device__ __forceinline__ void nvp_store(T* __restrict__ p, const float (&f)[V]) {
    nvp_vec<T, V> t;
#pragma unroll
    for (int e = 0; e < V; ++e) t.v[e] = (T)f[e];
    __builtin_memcpy(p, &t, sizeof(t));
}

__host__ inline int nvp_type_size(int32_t type) { return type == NVP_F32 ? 4 : type == NVP_BF16 || type == NVP_F16 ? 2 : 0; }
