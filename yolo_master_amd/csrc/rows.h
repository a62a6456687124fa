// Vector access to rows of any width and alignment, for the row-wise token kernels (csrc/rmsnorm.hip, tokens.hip).  A lane handles 16 bytes of a row at
// a time: EVEN rows (16-byte aligned, a whole number of vectors) with aligned accesses, others with 16-byte accesses at the element's alignment, which
// the hardware splits where they cross a line (a row of 1021 fp32 values at 16 bytes a lane instead of 4: RN_ODD).
#pragma once
#include "ymk_common.h"

typedef u32x4 u32x4_u __attribute__((aligned(1)));
typedef u32x2 u32x2_u __attribute__((aligned(1)));
typedef uint32_t u32_u __attribute__((aligned(1)));

__device__ __forceinline__ void row_widen(const u32x4& t, float (&v)[8]) {
    v[0] = h16lo(t.x); v[1] = h16hi(t.x); v[2] = h16lo(t.y); v[3] = h16hi(t.y);
    v[4] = h16lo(t.z); v[5] = h16hi(t.z); v[6] = h16lo(t.w); v[7] = h16hi(t.w);
}
__device__ __forceinline__ void row_widen(const u32x4& t, float (&v)[4]) {
    const uint32_t a = t.x, b = t.y, c = t.z, d = t.w;
    v[0] = __uint_as_float(a); v[1] = __uint_as_float(b); v[2] = __uint_as_float(c); v[3] = __uint_as_float(d);
}
__device__ __forceinline__ u32x4 row_narrow(const float (&v)[8]) {
    return u32x4{pack_h16x2(v[0], v[1]), pack_h16x2(v[2], v[3]), pack_h16x2(v[4], v[5]), pack_h16x2(v[6], v[7])};
}
__device__ __forceinline__ u32x4 row_narrow(const float (&v)[4]) {
    return u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
}

// the first n (1 .. V) of V elements at p; the others are left as they are
template <typename T, bool EVEN, int V>
__device__ __forceinline__ void row_load(const T* p, int n, float (&v)[V]) {
    static_assert(V * sizeof(T) == 16, "16 bytes a lane");
    if constexpr (EVEN) row_widen(*reinterpret_cast<const u32x4*>(p), v);
    else if (n >= V) {
        const u32x4 t = *reinterpret_cast<const u32x4_u*>(p);
        row_widen(t, v);
    }
    else {
#pragma unroll
        for (int e = 0; e < V - 1; ++e) {   // no branches: the last one again, not used
            const float t = to_f32(p[e < n ? e : n - 1]);
            v[e] = e < n ? t : v[e];
        }
    }
}
template <typename T, bool EVEN, int V>
__device__ __forceinline__ void row_store(T* p, int n, const float (&v)[V]) {
    static_assert(V * sizeof(T) == 16, "16 bytes a lane");
    if constexpr (EVEN) *reinterpret_cast<u32x4*>(p) = row_narrow(v);
    else if (n >= V) *reinterpret_cast<u32x4_u*>(p) = row_narrow(v);
    else {
#pragma unroll
        for (int e = 0; e < V - 1; ++e)
            if (e < n) from_f32(p[e], v[e]);
    }
}
