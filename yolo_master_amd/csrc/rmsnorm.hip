// Root-mean-square norm with the residual's addition, its 8-bit output and its gradient (include/ymk_tokens.h).
//
// Memory-bound: a row is read once, kept in registers between the statistic and the output, and written once.  A row belongs to a group of
// 2^n lanes (8..64 of one wave, or a whole workgroup of 128..1024): a lane holds up to NV vectors of V elements, vector i of lane l at column
// (l + i * group) * V, so every load and store of a group is contiguous; V is 16 bytes (csrc/rows.h).  Groups of one wave
// need no LDS and no barrier, so they take every width that fits their registers; wider rows are spread over a workgroup.
// Measured: residual sum, norm and e4m3 output of 25600 x 2048 bf16 70 us (5.3 TB/s); of 4 x 4096 4.4 us; 102400 x 256 bf16 forward 36 us (5.8 TB/s), gradients
// 37 + 5 us for dweight; 2041 x 1021 fp32 7.7 us (4.3 TB/s), gradients 10.3 + 3.8: one row a wave leaves 511 partial rows of dweight.
#include "ymk_common.h"
#include "rows.h"
#include "../../include/ymk_tokens.h"

#ifndef YMK_MAX_BLOCKS
#define RN_MAX_WAVES (256 * 32)   // waves of the one-wave kernels that stay resident and walk the rows: 8 per SIMD
#define RN_MAX_GROUPS 2048        // ... and workgroups of the wide ones
#define RN_BWD_BLOCKS 1280        // workgroups of the gradient: each leaves one partial row of dweight
#else
#define RN_MAX_WAVES 8
#define RN_MAX_GROUPS YMK_MAX_BLOCKS
#define RN_BWD_BLOCKS YMK_MAX_BLOCKS
#endif

#define RN_MAX_NV(T) (2 * (int)sizeof(T))    // vectors a lane holds at most: 32 values,
#define RN_MAX_NV_BWD(T) ((int)sizeof(T))    // 16 in the gradient, which keeps five of each (128 registers)
#define RN_SMALL 0x1.cp-118f   // 448 * 2^-126: below it the scale would be subnormal and its reciprocal infinite

namespace {

// the value as it is stored
template <typename T>
__device__ __forceinline__ float rn_round(float v) {
    if constexpr (sizeof(T) == 4) return v;
    else return h16_to_f32(f32_to_h16(v));
}
// V values in e4m3 (TINY: the first n)
__device__ __forceinline__ uint32_t rn_e4m3(float a, float b, float c, float d) {
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false), true);
}
template <bool TINY, int V>
__device__ __forceinline__ void rn_store_e4m3(uint8_t* p, int n, const float (&v)[V]) {
    if constexpr (!TINY) {
        if constexpr (V == 8) *reinterpret_cast<u32x2_u*>(p) = u32x2{rn_e4m3(v[0], v[1], v[2], v[3]), rn_e4m3(v[4], v[5], v[6], v[7])};
        else *reinterpret_cast<u32_u*>(p) = rn_e4m3(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (e < n) p[e] = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[e], 0.f, 0, false);
    }
}

// A lane's vectors of a row: vector i covers columns [at(i), at(i) + V), of which the first again(i) belong to an earlier vector (all V: the lane has none).
// EVEN widths have whole vectors only; TINY ones less than one.
enum { RN_EVEN, RN_RAGGED, RN_TINY };
template <int W, int V>
struct RnCols {
    int first, step, C;   // column of vector 0, and from one vector to the next
    __device__ __forceinline__ int at(int i) const { return W == RN_TINY ? 0 : min(first + i * step, C - V); }
    __device__ __forceinline__ bool mine(int i) const { return first + i * step < C; }
    __device__ __forceinline__ bool counts(int i, int e) const {   // element e of vector i is in the row and no other lane's
        if (W == RN_EVEN) return mine(i);
        if (W == RN_TINY) return mine(i) && e < C;
        return e >= first + i * step - at(i);
    }
};

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

template <typename T, int W, int NV, bool QUANT>
__global__ __launch_bounds__(NV == RN_MAX_NV(T) ? 256 : 1024) void rms_norm_kernel(RnArgs a) {
    constexpr int V = 16 / sizeof(T);
    constexpr bool TINY = W == RN_TINY;
    __shared__ float part[2][16];
    RnGroup g{a.group, 0, part};
    const int lane = threadIdx.x & (a.group - 1), per = blockDim.x / a.group;
    const RnCols<W, V> cols{lane * V, a.group * V, a.C};
    const T* x = static_cast<const T*>(a.x);
    const T* res = static_cast<const T*>(a.res);
    float w[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) w[i][e] = a.weight[TINY ? min(e, a.C - 1) : cols.at(i) + e];
    const float inv_c = 1.0f / (float)a.C;
    for (int64_t r0 = (int64_t)blockIdx.x * per; r0 < a.rows; r0 += (int64_t)gridDim.x * per) {   // the same trips for the whole workgroup
        const int64_t r = min(r0 + threadIdx.x / a.group, a.rows - 1);                            // a group behind the last row repeats it
        const bool live = r0 + threadIdx.x / a.group < a.rows;
        u32x4 raw[NV], add[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) raw[i] = row_load<T, TINY>(x + r * a.ldx + cols.at(i), a.C);
        if (res) {
#pragma unroll
            for (int i = 0; i < NV; ++i) add[i] = row_load<T, TINY>(res + r * a.ldr + cols.at(i), a.C);
        }
        float v[NV][V], ss = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            row_widen(raw[i], v[i]);
            if (res) {
                float b[V];
                row_widen(add[i], b);
#pragma unroll
                for (int e = 0; e < V; ++e) v[i][e] = rn_round<T>(v[i][e] + b[e]);
            }
#pragma unroll
            for (int e = 0; e < V; ++e) ss = cols.counts(i, e) ? fmaf(v[i][e], v[i][e], ss) : ss;
        }
        const float rstd = 1.0f / sqrtf(g.sum(ss) * inv_c + a.eps);
        if (res) {   // after the reduction: every lane of the group has read what h may alias
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (live && cols.mine(i)) row_store<T, TINY>(static_cast<T*>(a.h) + r * a.ldh + cols.at(i), a.C, v[i]);
        }
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                v[i][e] = v[i][e] * rstd * w[i][e];
                if constexpr (QUANT) {   // an element that two lanes hold does no harm; TINY zeros neither, unless the row's scale is not finite
                    const float m = __uint_as_float(__float_as_uint(v[i][e]) & 0x7fffffffu);
                    top = __float_as_uint(m) > __float_as_uint(top) ? m : top;
                }
            }
        float stat = rstd;
        if constexpr (QUANT) {
            top = g.top(top);
            const float scale = top < RN_SMALL ? 1.0f : top * (1.0f / 448.0f) < __uint_as_float(0x7f800000u) ? top / 448.0f : __uint_as_float(0x7fc00000u);
            stat = scale;
            // y * (1 / scale) is within 2^-23 of y / scale and never above 448 * (1 + 2^-22), which rounds to 448: no clamp, and NaN stays NaN
            const float inv = 1.0f / scale;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
#pragma unroll
                for (int e = 0; e < V; ++e) v[i][e] = top < RN_SMALL ? 0.f : v[i][e] * inv;
                if (live && cols.mine(i)) rn_store_e4m3<TINY>(static_cast<uint8_t*>(a.y) + r * a.ldy + cols.at(i), a.C, v[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (live && cols.mine(i)) row_store<T, TINY>(static_cast<T*>(a.y) + r * a.ldy + cols.at(i), a.C, v[i]);
        }
        if (a.stat && lane == 0 && live) a.stat[r] = stat;
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
template <typename T, int W, int NV>
__global__ __launch_bounds__(1024) void rms_norm_backward_kernel(RnBwdArgs a) {
    constexpr int V = 16 / sizeof(T);
    constexpr bool TINY = W == RN_TINY;
    __shared__ float part[2][16];
    extern __shared__ float dw_lds[];   // [groups of the workgroup][columns of a group]
    RnGroup g{a.group, 0, part};
    const int lane = threadIdx.x & (a.group - 1), per = blockDim.x / a.group;
    const RnCols<W, V> cols{lane * V, a.group * V, a.C};
    const T* dyp = static_cast<const T*>(a.dy);
    const T* hp = static_cast<const T*>(a.h);
    const T* drp = static_cast<const T*>(a.dres);
    float w[NV][V], dw[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) {
            w[i][e] = a.weight[TINY ? min(e, a.C - 1) : cols.at(i) + e];
            dw[i][e] = 0.f;
        }
    const float inv_c = 1.0f / (float)a.C;
    for (int64_t r0 = (int64_t)blockIdx.x * per; r0 < a.rows; r0 += (int64_t)gridDim.x * per) {   // the same trips for the whole workgroup
        const int64_t r = min(r0 + threadIdx.x / a.group, a.rows - 1);                            // a group behind the last row repeats it
        const bool live = r0 + threadIdx.x / a.group < a.rows;
        u32x4 hr[NV], dr[NV], orr[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            hr[i] = row_load<T, TINY>(hp + r * a.ldh + cols.at(i), a.C);
            dr[i] = row_load<T, TINY>(dyp + r * a.lddy + cols.at(i), a.C);
        }
        if (drp) {
#pragma unroll
            for (int i = 0; i < NV; ++i) orr[i] = row_load<T, TINY>(drp + r * a.lddr + cols.at(i), a.C);
        }
        const float rstd = a.rstd[r];
        float n[NV][V], d[NV][V], gn = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            row_widen(hr[i], n[i]);
            row_widen(dr[i], d[i]);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                n[i][e] *= rstd;
                dw[i][e] = live ? fmaf(d[i][e], n[i][e], dw[i][e]) : dw[i][e];
                d[i][e] *= w[i][e];
                gn = cols.counts(i, e) ? fmaf(d[i][e], n[i][e], gn) : gn;
            }
        }
        gn = g.sum(gn) * inv_c;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float o[V];
            if (drp) row_widen(orr[i], o);
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] = fmaf(rstd, fmaf(-n[i][e], gn, d[i][e]), drp ? o[e] : 0.f);
            if (live && cols.mine(i)) row_store<T, TINY>(static_cast<T*>(a.dx) + r * a.lddx + cols.at(i), a.C, o);
        }
    }
    if (!a.part) return;
    float* out = a.part + (size_t)blockIdx.x * a.C;
    if (per == 1) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (cols.counts(i, e)) out[cols.at(i) + e] = dw[i][e];
        return;
    }
    float* mine = dw_lds + (threadIdx.x / a.group) * a.C;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (cols.counts(i, e)) mine[cols.at(i) + e] = dw[i][e];
    __syncthreads();
    for (int c = threadIdx.x; c < a.C; c += blockDim.x) {
        float s = 0.f;
        for (int q = 0; q < per; ++q) s += dw_lds[q * a.C + c];
        out[c] = s;
    }
}

// dweight[c] = sum over the partial rows: 16 columns by 64 strands of rows a workgroup, four rows of a strand in flight at a time, added in strand order
// (64 columns by 16 strands of one row at a time: 18 us for 915 partial rows of 256, all of it waiting)
__global__ __launch_bounds__(1024) void rms_norm_dweight_kernel(const float* part, int blocks, int C, float* dweight) {
    __shared__ float s[64][17];
    const int c = blockIdx.x * 16 + (threadIdx.x & 15), q = threadIdx.x >> 4;
    float v = 0.f;
    if (c < C)
        for (int b = q; b < blocks; b += 256) {
            float p[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) p[i] = b + 64 * i < blocks ? part[(size_t)(b + 64 * i) * C + c] : 0.f;
            v += (p[0] + p[1]) + (p[2] + p[3]);
        }
    s[q][threadIdx.x & 15] = v;
    __syncthreads();
    if (q < 16) {   // thread (strand group q, column)
        v = (s[q][threadIdx.x & 15] + s[q + 16][threadIdx.x & 15]) + (s[q + 32][threadIdx.x & 15] + s[q + 48][threadIdx.x & 15]);
        __syncthreads();
        s[q][threadIdx.x & 15] = v;
    } else __syncthreads();
    __syncthreads();
    if (q == 0 && c < C) {
        for (int i = 1; i < 16; ++i) v += s[i][threadIdx.x];
        dweight[c] = v;
    }
}

inline bool rn_al(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) == 0; }
inline bool rn_bad(const void* p, int32_t ld, int32_t C, int es) { return !p || ld < C || !rn_al(p, es); }

// How a row of `vecs` vectors is spread: the group and the vectors a lane holds.  (Few rows spread wider, down to one vector a lane, measured the same: 4
// rows of 4096 7.3-7.6 us a call either way, 600 rows 7.2-7.3.)
struct RnPlan {
    int group, nv, threads;
    unsigned grid;
};
// max_nv / wide_nv: vectors a lane may hold in workgroups of up to 256 lanes and in wider ones.
inline RnPlan rn_plan(int64_t rows, int32_t vecs, int max_nv, int wide_nv, int64_t max_waves, int64_t max_groups) {
    RnPlan p;
    p.group = 8;
    while (p.group < 64 && p.group * 2 < vecs) p.group *= 2;
    while (p.group < 1024 && p.group * (p.group < 256 ? max_nv : wide_nv) < vecs) p.group *= 2;
    p.nv = 1;
    while (p.group * p.nv < vecs) p.nv *= 2;
    p.threads = p.group > 64 ? p.group : 256;   // a group wider than a wave is a workgroup of its own
    const int per = p.threads / p.group;
    const int64_t need = (rows + per - 1) / per;                                        // workgroups if none walked
    const int64_t most = p.group > 64 ? max_groups : max_waves / (p.threads / 64);
    // Equal trips for all workgroups and an equal number of workgroups for all 256 CUs: of the next few trip counts the one whose fullest CU walks least
    // (25600 rows of 2048, norm to 8 bits: 4 trips of 1600 workgroups, seven on some CUs, 97 us; 5 trips of 1280, five on each, 79 us)
    int64_t trips = (need + most - 1) / most, walked = INT64_MAX;
    for (int64_t t = trips, last = trips + 4; t < last; ++t) {
        const int64_t grid = (need + t - 1) / t, w = t * ((grid + 255) / 256);
        if (w < walked) {
            walked = w;
            trips = t;
        }
    }
    p.grid = (unsigned)((need + trips - 1) / trips);
    return p;
}

template <typename T, int W, bool QUANT, int NV = 1>
int rn_launch(const RnPlan& p, const RnArgs& a, void* stream) {
    if constexpr (NV > (W == RN_TINY ? 1 : RN_MAX_NV(T))) return YMK_E_BADARG;
    else {
        if (p.nv > NV) return rn_launch<T, W, QUANT, NV * 2>(p, a, stream);
        hipLaunchKernelGGL((rms_norm_kernel<T, W, NV, QUANT>), dim3(p.grid), dim3(p.threads), 0, (hipStream_t)stream, a);
        return ymk_launch_status();
    }
}
template <typename T, int W, int NV = 1>
int rn_launch_backward(const RnPlan& p, const RnBwdArgs& a, void* stream) {
    if constexpr (NV > (W == RN_TINY ? 1 : RN_MAX_NV_BWD(T))) return YMK_E_BADARG;
    else {
        if (p.nv > NV) return rn_launch_backward<T, W, NV * 2>(p, a, stream);
        const size_t lds = p.threads > p.group && a.part ? (size_t)(p.threads / p.group) * a.C * sizeof(float) : 0;
        hipLaunchKernelGGL((rms_norm_backward_kernel<T, W, NV>), dim3(p.grid), dim3(p.threads), lds, (hipStream_t)stream, a);
        return ymk_launch_status();
    }
}

template <typename T, bool QUANT>
int rn_width(const RnPlan& p, const RnArgs& a, void* stream) {
    constexpr int V = 16 / sizeof(T);
    return a.C < V ? rn_launch<T, RN_TINY, QUANT>(p, a, stream) : a.C % V ? rn_launch<T, RN_RAGGED, QUANT>(p, a, stream) : rn_launch<T, RN_EVEN, QUANT>(p, a, stream);
}
template <typename T>
int rn_width_backward(const RnPlan& p, const RnBwdArgs& a, void* stream) {
    constexpr int V = 16 / sizeof(T);
    return a.C < V ? rn_launch_backward<T, RN_TINY>(p, a, stream) : a.C % V ? rn_launch_backward<T, RN_RAGGED>(p, a, stream) : rn_launch_backward<T, RN_EVEN>(p, a, stream);
}

int rms_norm_any(bool quant, int32_t dtype, const void* x, int32_t ldx, const void* residual, int32_t ldr, void* h, int32_t ldh, void* y, int32_t ldy,
                 float* stat, int64_t rows, int32_t C, const float* weight, float eps, void* stream) {
    const int es = dtype == YMK_F32 ? 4 : 2;
    if ((dtype != YMK_F32 && dtype != YMK_H16) || C < 1 || C > YMK_NORM_MAX_C || rows < 0 || !(eps >= 0.f)) return YMK_E_BADARG;
    if (rows == 0) return YMK_OK;
    if (!weight || rn_bad(x, ldx, C, es) || (residual && (rn_bad(residual, ldr, C, es) || rn_bad(h, ldh, C, es))) || rn_bad(y, ldy, C, quant ? 1 : es) || (quant && !stat))
        return YMK_E_BADARG;
    const int V = 16 / es;
    const RnPlan p = rn_plan(rows, (C + V - 1) / V, dtype == YMK_F32 ? RN_MAX_NV(float) : RN_MAX_NV(h16_t), dtype == YMK_F32 ? RN_MAX_NV(float) / 2 : RN_MAX_NV(h16_t) / 2, RN_MAX_WAVES, RN_MAX_GROUPS);
    const RnArgs a{x, residual, h, y, stat, weight, rows, ldx, ldr, ldh, ldy, C, p.group, eps};
    if (dtype == YMK_F32) return quant ? rn_width<float, true>(p, a, stream) : rn_width<float, false>(p, a, stream);
    return quant ? rn_width<h16_t, true>(p, a, stream) : rn_width<h16_t, false>(p, a, stream);
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
        const int V = 16 / es;
        const RnPlan p = rn_plan(rows, (C + V - 1) / V, dtype == YMK_F32 ? RN_MAX_NV_BWD(float) : RN_MAX_NV_BWD(h16_t), dtype == YMK_F32 ? RN_MAX_NV_BWD(float) : RN_MAX_NV_BWD(h16_t), (int64_t)RN_BWD_BLOCKS * 4, RN_BWD_BLOCKS);
        const RnBwdArgs a{dy, h, rstd, weight, dres, dx, dweight ? static_cast<float*>(workspace) : nullptr, rows, lddy, ldh, lddr, lddx, C, p.group};
        const int rc = dtype == YMK_F32 ? rn_width_backward<float>(p, a, stream) : rn_width_backward<h16_t>(p, a, stream);
        if (rc != YMK_OK || !dweight) return rc;
        hipLaunchKernelGGL(rms_norm_dweight_kernel, dim3((unsigned)((C + 15) / 16)), dim3(1024), 0, (hipStream_t)stream, static_cast<const float*>(workspace), (int)p.grid,
                           (int)C, dweight);
    } else if (dweight) {   // no rows: the sum over none of them
        hipLaunchKernelGGL(rms_norm_dweight_kernel, dim3((unsigned)((C + 15) / 16)), dim3(1024), 0, (hipStream_t)stream, static_cast<const float*>(nullptr), 0, (int)C, dweight);
    }
    return ymk_launch_status();
}
