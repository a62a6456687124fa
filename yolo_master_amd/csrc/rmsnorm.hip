// Root-mean-square norm with the residual's addition, its 8-bit output and its gradient (include/ymk_tokens.h).
//
// Memory-bound: a row is read once, kept in registers between the statistic and the output, and written once.  A row belongs to a group of
// 2^n lanes (8..64 of one wave, or a whole workgroup of 128..1024): a lane holds up to NV vectors of V elements, vector i of lane l at column
// (l + i * group) * V, so every load and store of a group is contiguous.  V is 16 bytes where rows are 16-byte aligned and single elements
// otherwise.  Groups of one wave need no LDS and no barrier, so they take every width that fits their registers once there are rows enough;
// wide rows, and few rows, are spread over a workgroup.
#include "ymk_common.h"
#include "../../include/ymk_tokens.h"

#ifndef YMK_MAX_BLOCKS
#define RN_MAX_WAVES (256 * 32)   // waves of the one-wave kernels that stay resident and walk the rows: 8 per SIMD
#define RN_MAX_GROUPS 2048        // ... and workgroups of the wide ones
#define RN_BWD_BLOCKS 1024        // workgroups of the gradient: each leaves one partial row of dweight
#else
#define RN_MAX_WAVES 8
#define RN_MAX_GROUPS YMK_MAX_BLOCKS
#define RN_BWD_BLOCKS YMK_MAX_BLOCKS
#endif

#define RN_TINY 0x1.cp-118f   // 448 * 2^-126: below it the scale would be subnormal and its reciprocal infinite

namespace {

template <typename T, int V>
__device__ __forceinline__ void rn_load(const T* p, float (&v)[V]) {
    if constexpr (V == 1) v[0] = to_f32(*p);
    else load_vec_f32(p, v);
}
template <typename T, int V>
__device__ __forceinline__ void rn_store(T* p, const float (&v)[V]) {
    if constexpr (V == 1) from_f32(*p, v[0]);
    else store_vec_f32(p, v);
}
// the value as it is stored
template <typename T>
__device__ __forceinline__ float rn_round(float v) {
    if constexpr (sizeof(T) == 4) return v;
    else return h16_to_f32(f32_to_h16(v));
}
__device__ __forceinline__ void rn_store_e4m3(uint8_t* p, const float (&v)[8]) {
    int lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false), hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4], v[5], 0, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], lo, true);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6], v[7], hi, true);
    *reinterpret_cast<u32x2*>(p) = u32x2{(uint32_t)lo, (uint32_t)hi};
}
__device__ __forceinline__ void rn_store_e4m3(uint8_t* p, const float (&v)[4]) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
    *reinterpret_cast<uint32_t*>(p) = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], w, true);
}
__device__ __forceinline__ void rn_store_e4m3(uint8_t* p, const float (&v)[1]) { *p = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[0], 0.f, 0, false); }

// Sum (and, below, largest bit pattern) over the group of a lane: lanes [l - l % group, + group) of a wave, or all `group` lanes of the workgroup
// through LDS (two slots used in turn: one barrier a reduction).  Every lane gets the result of the same tree: bit-identical within the group.
struct RnGroup {
    int group, slot;
    float (*part)[16];
    template <typename F>
    __device__ __forceinline__ float all(float v, F op) {
        for (int o = min(group, 64) >> 1; o > 0; o >>= 1) v = op(v, __shfl_xor(v, o));
        if (group > 64) {
            slot ^= 1;
            if ((threadIdx.x & 63) == 0) part[slot][threadIdx.x >> 6] = v;
            __syncthreads();
            v = part[slot][0];
            for (int w = 1; w < group >> 6; ++w) v = op(v, part[slot][w]);
        }
        return v;
    }
    __device__ __forceinline__ float sum(float v) { return all(v, [](float a, float b) { return a + b; }); }
    // largest |v| by its bits: finite < infinity < NaN, so that a NaN is not lost
    __device__ __forceinline__ float top(float v) {
        return all(v, [](float a, float b) { return __float_as_uint(a) > __float_as_uint(b) ? a : b; });
    }
};

struct RnArgs {
    const void* x;
    const void* res;
    void* h;
    void* y;
    float* stat;   // rstd, or the scale of the 8-bit output
    const float* weight;
    int64_t rows;
    int32_t ldx, ldr, ldh, ldy, C, group;
    float eps;
};

template <typename T, int V, int NV, bool QUANT>
__global__ __launch_bounds__(1024) void rms_norm_kernel(RnArgs a) {
    __shared__ float part[2][16];
    RnGroup g{a.group, 0, part};
    const int lane = threadIdx.x & (a.group - 1), per = blockDim.x / a.group;
    const T* x = static_cast<const T*>(a.x);
    const T* res = static_cast<const T*>(a.res);
    float w[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (lane + i * a.group) * V;
#pragma unroll
        for (int e = 0; e < V; ++e) w[i][e] = c < a.C ? a.weight[c + e] : 0.f;
    }
    const float inv_c = 1.0f / (float)a.C;
    for (int64_t r0 = (int64_t)blockIdx.x * per; r0 < a.rows; r0 += (int64_t)gridDim.x * per) {   // the same trips for the whole workgroup
        const int64_t r = r0 + threadIdx.x / a.group;
        const int cols = r < a.rows ? a.C : 0;
        float v[NV][V];
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (lane + i * a.group) * V;
#pragma unroll
            for (int e = 0; e < V; ++e) v[i][e] = 0.f;
            if (c < cols) rn_load<T, V>(x + r * a.ldx + c, v[i]);
        }
        if (res) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (lane + i * a.group) * V;
                if (c < cols) {
                    float b[V];
                    rn_load<T, V>(res + r * a.ldr + c, b);
#pragma unroll
                    for (int e = 0; e < V; ++e) v[i][e] = rn_round<T>(v[i][e] + b[e]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) ss = fmaf(v[i][e], v[i][e], ss);
        const float rstd = 1.0f / sqrtf(g.sum(ss) * inv_c + a.eps);
        if (res) {   // after the reduction: every lane of the group has read what h may alias
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (lane + i * a.group) * V;
                if (c < cols) rn_store<T, V>(static_cast<T*>(a.h) + r * a.ldh + c, v[i]);
            }
        }
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                v[i][e] = v[i][e] * rstd * w[i][e];
                if constexpr (QUANT) {
                    const float m = __uint_as_float(__float_as_uint(v[i][e]) & 0x7fffffffu);
                    top = __float_as_uint(m) > __float_as_uint(top) ? m : top;
                }
            }
        float stat = rstd;
        if constexpr (QUANT) {
            top = g.top(top);
            const float scale = top < RN_TINY ? 1.0f : top * (1.0f / 448.0f) < __uint_as_float(0x7f800000u) ? top / 448.0f : __uint_as_float(0x7fc00000u);
            stat = scale;
            // y * (1 / scale) is within 2^-23 of y / scale and never above 448 * (1 + 2^-22), which rounds to 448: no clamp, and NaN stays NaN
            const float inv = 1.0f / scale;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (lane + i * a.group) * V;
#pragma unroll
                for (int e = 0; e < V; ++e) v[i][e] = top < RN_TINY ? 0.f : v[i][e] * inv;
                if (c < cols) rn_store_e4m3(static_cast<uint8_t*>(a.y) + r * a.ldy + c, v[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (lane + i * a.group) * V;
                if (c < cols) rn_store<T, V>(static_cast<T*>(a.y) + r * a.ldy + c, v[i]);
            }
        }
        if (a.stat && lane == 0 && cols) a.stat[r] = stat;
    }
}

struct RnBwdArgs {
    const void* dy;
    const void* h;
    const float* rstd;
    const float* weight;
    const void* dres;
    void* dx;
    float* part;   // [gridDim.x][C] or NULL
    int64_t rows;
    int32_t lddy, ldh, lddr, lddx, C, group;
};

// dx of a row in one pass over it; dweight: a lane sums its columns over the rows it walks, the groups of a workgroup are added in a fixed
// order through LDS, and each workgroup leaves one partial row that rms_norm_dweight_kernel adds up — no atomics, the same bits every time.
template <typename T, int V, int NV>
__global__ __launch_bounds__(1024) void rms_norm_backward_kernel(RnBwdArgs a) {
    __shared__ float part[2][16];
    extern __shared__ float dw_lds[];   // [groups of the workgroup][columns of a group]
    RnGroup g{a.group, 0, part};
    const int lane = threadIdx.x & (a.group - 1), per = blockDim.x / a.group;
    const T* dyp = static_cast<const T*>(a.dy);
    const T* hp = static_cast<const T*>(a.h);
    const T* drp = static_cast<const T*>(a.dres);
    float w[NV][V], dw[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (lane + i * a.group) * V;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            w[i][e] = c < a.C ? a.weight[c + e] : 0.f;
            dw[i][e] = 0.f;
        }
    }
    const float inv_c = 1.0f / (float)a.C;
    for (int64_t r0 = (int64_t)blockIdx.x * per; r0 < a.rows; r0 += (int64_t)gridDim.x * per) {   // the same trips for the whole workgroup
        const int64_t r = r0 + threadIdx.x / a.group;
        const int cols = r < a.rows ? a.C : 0;
        float n[NV][V], d[NV][V], o[NV][V];
        const float rstd = cols ? a.rstd[r] : 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (lane + i * a.group) * V;
#pragma unroll
            for (int e = 0; e < V; ++e) n[i][e] = d[i][e] = o[i][e] = 0.f;
            if (c < cols) {
                rn_load<T, V>(hp + r * a.ldh + c, n[i]);
                rn_load<T, V>(dyp + r * a.lddy + c, d[i]);
                if (drp) rn_load<T, V>(drp + r * a.lddr + c, o[i]);
            }
        }
        float gn = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                n[i][e] *= rstd;
                dw[i][e] = fmaf(d[i][e], n[i][e], dw[i][e]);
                d[i][e] *= w[i][e];
                gn = fmaf(d[i][e], n[i][e], gn);
            }
        gn = g.sum(gn) * inv_c;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (lane + i * a.group) * V;
#pragma unroll
            for (int e = 0; e < V; ++e) o[i][e] = fmaf(rstd, fmaf(-n[i][e], gn, d[i][e]), o[i][e]);
            if (c < cols) rn_store<T, V>(static_cast<T*>(a.dx) + r * a.lddx + c, o[i]);
        }
    }
    if (!a.part) return;
    float* out = a.part + (size_t)blockIdx.x * a.C;
    if (per == 1) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (lane + i * a.group) * V;
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (c < a.C) out[c + e] = dw[i][e];
        }
        return;
    }
    const int width = a.group * V * NV;   // columns a group holds, C or more
    float* mine = dw_lds + (threadIdx.x / a.group) * width;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) mine[(lane + i * a.group) * V + e] = dw[i][e];
    __syncthreads();
    for (int c = threadIdx.x; c < a.C; c += blockDim.x) {
        float s = 0.f;
        for (int q = 0; q < per; ++q) s += dw_lds[q * width + c];
        out[c] = s;
    }
}

// dweight[c] = sum over the partial rows: 64 columns by 16 strands of rows a workgroup, added in strand order
__global__ __launch_bounds__(1024) void rms_norm_dweight_kernel(const float* part, int blocks, int C, float* dweight) {
    __shared__ float s[16][64];
    const int c = blockIdx.x * 64 + (threadIdx.x & 63), q = threadIdx.x >> 6;
    float v = 0.f;
    if (c < C)
        for (int b = q; b < blocks; b += 16) v += part[(size_t)b * C + c];
    s[q][threadIdx.x & 63] = v;
    __syncthreads();
    if (q == 0 && c < C) {
        for (int i = 1; i < 16; ++i) v += s[i][threadIdx.x];
        dweight[c] = v;
    }
}

inline bool rn_al(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) == 0; }
inline bool rn_bad(const void* p, int32_t ld, int32_t C, int es) { return !p || ld < C || !rn_al(p, es); }

// How a row of `vecs` vectors is spread: the group and the vectors a lane holds.  One wave holds up to 4 vectors a lane; with fewer rows than
// the chip has waves a row is spread wider instead, down to one vector a lane (up to 1024 lanes), which shortens a single row's time.
struct RnPlan {
    int group, nv, threads;
    unsigned grid;
};
inline RnPlan rn_plan(int64_t rows, int32_t vecs, int max_nv, int64_t max_waves, int64_t max_groups) {
    RnPlan p;
    const bool few = rows <= 512;
    p.group = 8;
    while (p.group < 64 && p.group * (few ? 1 : 2) < vecs) p.group *= 2;
    while (p.group < 1024 && p.group * (few ? 1 : max_nv > 4 ? max_nv : 4) < vecs) p.group *= 2;
    p.nv = 1;
    while (p.group * p.nv < vecs) p.nv *= 2;
    p.threads = p.group > 64 ? p.group : 256;   // a group wider than a wave is a workgroup of its own
    const int per = p.threads / p.group;
    const int64_t need = (rows + per - 1) / per;                                        // workgroups if none walked
    const int64_t most = p.group > 64 ? max_groups : max_waves / (p.threads / 64);
    const int64_t trips = (need + most - 1) / most;
    p.grid = (unsigned)((need + trips - 1) / trips);                                    // equal trips for all
    return p;
}

template <typename T, int V, bool QUANT, int NV = 1>
int rn_launch(const RnPlan& p, const RnArgs& a, void* stream) {
    if constexpr (NV > (V == 1 ? 16 : 4 * (int)sizeof(T) / 2)) return YMK_E_BADARG;
    else {
        if (p.nv > NV) return rn_launch<T, V, QUANT, NV * 2>(p, a, stream);
        hipLaunchKernelGGL((rms_norm_kernel<T, V, NV, QUANT>), dim3(p.grid), dim3(p.threads), 0, (hipStream_t)stream, a);
        return ymk_launch_status();
    }
}
template <typename T, int V, int NV = 1>
int rn_launch_backward(const RnPlan& p, const RnBwdArgs& a, void* stream) {
    if constexpr (NV > (V == 1 ? 16 : 4 * (int)sizeof(T) / 2)) return YMK_E_BADARG;
    else {
        if (p.nv > NV) return rn_launch_backward<T, V, NV * 2>(p, a, stream);
        const size_t lds = p.threads > p.group && a.part ? (size_t)p.threads * V * NV * sizeof(float) : 0;
        hipLaunchKernelGGL((rms_norm_backward_kernel<T, V, NV>), dim3(p.grid), dim3(p.threads), lds, (hipStream_t)stream, a);
        return ymk_launch_status();
    }
}
inline int rn_vec(int32_t dtype, int32_t C) { return C % (dtype == YMK_F32 ? 4 : 8) == 0 ? (dtype == YMK_F32 ? 4 : 8) : 1; }
inline int rn_max_nv(int32_t dtype, int V) { return V == 1 ? 16 : dtype == YMK_F32 ? 8 : 4; }

int rms_norm_any(bool quant, int32_t dtype, const void* x, int32_t ldx, const void* residual, int32_t ldr, void* h, int32_t ldh, void* y, int32_t ldy,
                 float* stat, int64_t rows, int32_t C, const float* weight, float eps, void* stream) {
    const int es = dtype == YMK_F32 ? 4 : 2;
    if ((dtype != YMK_F32 && dtype != YMK_H16) || C < 1 || C > YMK_NORM_MAX_C || rows < 0 || !(eps >= 0.f)) return YMK_E_BADARG;
    if (rows == 0) return YMK_OK;
    if (!weight || rn_bad(x, ldx, C, es) || (residual && (rn_bad(residual, ldr, C, es) || rn_bad(h, ldh, C, es))) || rn_bad(y, ldy, C, quant ? 1 : es) || (quant && !stat))
        return YMK_E_BADARG;
    int V = rn_vec(dtype, C);
    if (ldx % V || !rn_al(x, 16) || (residual && (ldr % V || ldh % V || !rn_al(residual, 16) || !rn_al(h, 16))) || ldy % V || !rn_al(y, quant ? V : 16)) V = 1;
    const RnArgs a{x, residual, h, y, stat, weight, rows, ldx, ldr, ldh, ldy, C, 0, eps};
    RnPlan p = rn_plan(rows, (C + V - 1) / V, rn_max_nv(dtype, V), RN_MAX_WAVES, RN_MAX_GROUPS);
    RnArgs b = a;
    b.group = p.group;
    if (dtype == YMK_F32) {
        if (quant) return V == 1 ? rn_launch<float, 1, true>(p, b, stream) : rn_launch<float, 4, true>(p, b, stream);
        return V == 1 ? rn_launch<float, 1, false>(p, b, stream) : rn_launch<float, 4, false>(p, b, stream);
    }
    if (quant) return V == 1 ? rn_launch<h16_t, 1, true>(p, b, stream) : rn_launch<h16_t, 8, true>(p, b, stream);
    return V == 1 ? rn_launch<h16_t, 1, false>(p, b, stream) : rn_launch<h16_t, 8, false>(p, b, stream);
}

}  // namespace

extern "C" int ymk_rms_norm(int32_t dtype, const void* x, int32_t ldx, const void* residual, int32_t ldr, void* h, int32_t ldh, void* y,
                            int32_t ldy, float* rstd, int64_t rows, int32_t C, const float* weight, float eps, void* stream) {
    return rms_norm_any(false, dtype, x, ldx, residual, ldr, h, ldh, y, ldy, rstd, rows, C, weight, eps, stream);
}

extern "C" int ymk_rms_norm_quant(int32_t dtype, const void* x, int32_t ldx, const void* residual, int32_t ldr, void* h, int32_t ldh, void* q,
                                  int32_t ldq, float* scale, int64_t rows, int32_t C, const float* weight, float eps, void* stream) {
    return rms_norm_any(true, dtype, x, ldx, residual, ldr, h, ldh, q, ldq, scale, rows, C, weight, eps, stream);
}

extern "C" size_t ymk_rms_norm_backward_workspace_bytes(int64_t rows, int32_t C) {
    return rows > 0 && C > 0 ? (size_t)(rows < RN_BWD_BLOCKS ? rows : RN_BWD_BLOCKS) * C * sizeof(float) : 0;   // a workgroup has a row at least
}

extern "C" int ymk_rms_norm_backward(int32_t dtype, const void* dy, int32_t lddy, const void* h, int32_t ldh, const float* rstd, const float* weight,
                                     const void* dres, int32_t lddr, void* dx, int32_t lddx, float* dweight, int64_t rows, int32_t C,
                                     void* workspace, size_t workspace_bytes, void* stream) {
    const int es = dtype == YMK_F32 ? 4 : 2;
    if ((dtype != YMK_F32 && dtype != YMK_H16) || C < 1 || C > YMK_NORM_MAX_C || rows < 0) return YMK_E_BADARG;
    if (rows > 0 && (!weight || !rstd || rn_bad(dy, lddy, C, es) || rn_bad(h, ldh, C, es) || (dres && rn_bad(dres, lddr, C, es)) || rn_bad(dx, lddx, C, es)))
        return YMK_E_BADARG;
    if (dweight && rows > 0 && (!workspace || workspace_bytes < ymk_rms_norm_backward_workspace_bytes(rows, C))) return YMK_E_WORKSPACE;
    if (rows > 0) {
        int V = rn_vec(dtype, C);
        if (lddy % V || ldh % V || lddx % V || !rn_al(dy, 16) || !rn_al(h, 16) || !rn_al(dx, 16) || (dres && (lddr % V || !rn_al(dres, 16)))) V = 1;
        const RnPlan p = rn_plan(rows, (C + V - 1) / V, rn_max_nv(dtype, V), (int64_t)RN_BWD_BLOCKS * 4, RN_BWD_BLOCKS);
        const RnBwdArgs a{dy, h, rstd, weight, dres, dx, dweight ? static_cast<float*>(workspace) : nullptr, rows, lddy, ldh, lddr, lddx, C, p.group};
        const int rc = dtype == YMK_F32 ? (V == 1 ? rn_launch_backward<float, 1>(p, a, stream) : rn_launch_backward<float, 4>(p, a, stream))
                                        : (V == 1 ? rn_launch_backward<h16_t, 1>(p, a, stream) : rn_launch_backward<h16_t, 8>(p, a, stream));
        if (rc != YMK_OK || !dweight) return rc;
        hipLaunchKernelGGL(rms_norm_dweight_kernel, dim3((unsigned)((C + 63) / 64)), dim3(1024), 0, (hipStream_t)stream, static_cast<const float*>(workspace), (int)p.grid,
                           (int)C, dweight);
    } else if (dweight) {   // no rows: the sum over none of them
        hipLaunchKernelGGL(rms_norm_dweight_kernel, dim3((unsigned)((C + 63) / 64)), dim3(1024), 0, (hipStream_t)stream, static_cast<const float*>(nullptr), 0, (int)C, dweight);
    }
    return ymk_launch_status();
}
