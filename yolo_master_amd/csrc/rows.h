// Vector access to rows of any width and alignment, for the row-wise token kernels (csrc/rmsnorm.hip, tokens.hip).  A lane handles 16 bytes of a row at
// a time, at the element's alignment (the hardware splits an access where it crosses a line).  The last vector of a row ends with the row: where the
// width is no whole number of vectors it overlaps the one before it, both lanes hold the shared elements and write the same bytes.  Nothing branches on
// the width, so all loads of a row are in flight together (with a branch for the row's end each vector was waited for by itself: 15760 x 774 fp32,
// norm and gradients, 185 us).  Rows narrower than a vector are loaded element by element.
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

// 16 bytes of a row of n elements (n < V: those, with zeros behind them)
template <typename T, bool TINY>
__device__ __forceinline__ u32x4 row_load(const T* p, int n) {
    if constexpr (!TINY) return *reinterpret_cast<const u32x4_u*>(p);
    else {
        constexpr int V = 16 / sizeof(T);
        float v[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float t = to_f32(p[e < n ? e : n - 1]);
            v[e] = e < n ? t : 0.f;
        }
        return row_narrow(v);
    }
}
template <typename T, bool TINY, int V>
__device__ __forceinline__ void row_store(T* p, int n, const float (&v)[V]) {
    static_assert(V * sizeof(T) == 16, "16 bytes a lane");
    if constexpr (!TINY) *reinterpret_cast<u32x4_u*>(p) = row_narrow(v);
    else {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (e < n) from_f32(p[e], v[e]);
    }
}
