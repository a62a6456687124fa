// Tokens sorted by expert and back (include/ymk_tokens.h): the stable sort of the (token, choice) pairs, the move of rows into expert order and
// the weighted sum back, with their gradients.  Nothing here multiplies matrices: the sort is bound by latency (a launch, two dependent reads),
// the moves by memory — each row is read once and written once.
// Measured: sort of 16 pairs 2.7 us (one launch), of 98298 pairs over 64 experts 12 us (two); 25600 tokens of 512 bf16 channels, two of 16 experts:
// dispatch 15.7 us (4.6 TB/s), combine 16, its gradient 23 (5.2 TB/s); 16383 tokens of 2048 channels, six of 64: combine 97-116 us (4.0-4.8 TB/s).
#include "ymk_common.h"
#include "rows.h"
#include "../../include/ymk_tokens.h"

#ifndef YMK_MAX_BLOCKS
#define TK_MAX_BLOCKS (256 * 32)
#else
#define TK_MAX_BLOCKS YMK_MAX_BLOCKS
#endif
#define TK_MAX_C 0x7ffffff0   // widest row of the sums: the kernels count columns in 32 bits, a row rounded up to whole vectors included
#define TK_SORT_BLOCKS 256    // most workgroups of the two-launch sort: each sums the histograms of those before it
// Pairs that one workgroup sorts alone, in one launch: with one / two launches 7.6 / 10.5 us for 4096 pairs, 9.4 / 10.2 (16 experts) and 12.1 / 10.0 (128)
// for 8192, 16.1 / 10.2 for 16384
#define TK_SORT_ONE 4096

namespace {

// ------------------------------------------------------------------------------------------------------------ sort
// Counting sort by the key e = expert, E for a pair without one (those fill the tail).  A workgroup owns a contiguous range of pairs and a wave a
// contiguous part of it, so a pair's place is
//   (pairs of smaller keys) + (pairs of its key in earlier workgroups) + (... in earlier waves) + (... in earlier lanes of its wave's 64s),
// all of them integers: stable and the same every time.
struct SortArgs {
    const void* idx;
    int64_t pairs;
    int32_t wide;      // idx is int64
    int32_t E;
    int32_t per;       // pairs a workgroup owns
    int32_t* offsets;
    int32_t* src;
    int32_t* row;
    int32_t* hist;     // [workgroups][E + 1]
};

__device__ __forceinline__ int sort_key(const SortArgs& a, int64_t p) {
    if (a.wide) {
        const int64_t v = static_cast<const int64_t*>(a.idx)[p];
        return v >= 0 && v < a.E ? (int)v : a.E;
    }
    const int v = static_cast<const int32_t*>(a.idx)[p];
    return v >= 0 && v < a.E ? v : a.E;
}

// count[wave][key] of the workgroup's pairs; the caller zeroes nothing
template <int WAVES>
__device__ __forceinline__ void sort_count(const SortArgs& a, int64_t p0, int64_t p1, int32_t (*count)[YMK_TOKEN_MAX_E + 1]) {
    const int t = threadIdx.x, w = t >> 6, lane = t & 63;
    for (int i = t; i < WAVES * (YMK_TOKEN_MAX_E + 1); i += WAVES * 64) (&count[0][0])[i] = 0;
    __syncthreads();
    const int64_t part = (a.per + WAVES * 64 - 1) / (WAVES * 64) * 64, q0 = p0 + w * part, q1 = min(p1, q0 + part);
    for (int64_t p = q0 + lane; p < q1; p += 64) atomicAdd(&count[w][sort_key(a, p)], 1);   // integers in LDS: any order gives the same count
    __syncthreads();
}

// count[wave][key] -> first place of that wave's pairs of that key, from the workgroup's first place per key; then the pairs are placed
template <int WAVES>
__device__ __forceinline__ void sort_place(const SortArgs& a, int64_t p0, int64_t p1, int32_t (*count)[YMK_TOKEN_MAX_E + 1], const int32_t* first) {
    const int t = threadIdx.x, w = t >> 6, lane = t & 63;
    for (int e = t; e <= a.E; e += WAVES * 64) {
        int at = first[e];
        for (int i = 0; i < WAVES; ++i) {
            const int n = count[i][e];
            count[i][e] = at;
            at += n;
        }
    }
    __syncthreads();
    const int64_t part = (a.per + WAVES * 64 - 1) / (WAVES * 64) * 64, q0 = p0 + w * part, q1 = min(p1, q0 + part);
    int bits = 1;
    while ((1 << bits) <= a.E) ++bits;
    for (int64_t p = q0; p < q1; p += 64) {   // wave-uniform trips: every lane votes
        const bool live = p + lane < q1;
        const int e = live ? sort_key(a, p + lane) : a.E;
        unsigned long long same = __ballot(live);
        for (int b = 0; b < bits; ++b) {      // lanes of the same key
            const unsigned long long set = __ballot((e >> b) & 1);
            same &= (e >> b) & 1 ? set : ~set;
        }
        const unsigned long long before = same & ((1ull << lane) - 1ull);
        if (live) {
            const int at = count[w][e] + __popcll(before);
            const bool none = e == a.E;
            a.src[at] = none ? -1 : (int32_t)(p + lane);
            a.row[p + lane] = none ? -1 : at;
        }
        __builtin_amdgcn_wave_barrier();      // this wave alone touches count[w]: LDS operations of a wave stay in order
        if (live && before == 0) count[w][e] += __popcll(same);
        __builtin_amdgcn_wave_barrier();
    }
}

// exclusive sums over the keys of total[0..E] by the first wave; offsets are those of the experts
__device__ __forceinline__ void sort_starts(const int32_t* total, int E, int32_t* start, int32_t* offsets) {
    if (threadIdx.x < 64) {
        int base = 0;
        for (int e0 = 0; e0 <= E; e0 += 64) {
            const int e = e0 + (int)threadIdx.x;
            const int n = e <= E ? total[e] : 0;
            int sum = n;
            for (int o = 1; o < 64; o <<= 1) {
                const int v = __shfl_up(sum, o);
                if ((int)threadIdx.x >= o) sum += v;
            }
            if (e <= E) {
                start[e] = base + sum - n;
                if (offsets) offsets[e] = base + sum - n;
            }
            base += __shfl(sum, 63);
        }
    }
    __syncthreads();
}

__global__ __launch_bounds__(1024) void token_sort_one_kernel(SortArgs a) {
    __shared__ int32_t count[16][YMK_TOKEN_MAX_E + 1];
    __shared__ int32_t total[YMK_TOKEN_MAX_E + 1], start[YMK_TOKEN_MAX_E + 1];
    sort_count<16>(a, 0, a.pairs, count);
    for (int e = threadIdx.x; e <= a.E; e += 1024) {
        int n = 0;
        for (int i = 0; i < 16; ++i) n += count[i][e];
        total[e] = n;
    }
    __syncthreads();
    sort_starts(total, a.E, start, a.offsets);
    sort_place<16>(a, 0, a.pairs, count, start);
}

__global__ __launch_bounds__(1024) void token_sort_count_kernel(SortArgs a) {
    __shared__ int32_t count[16][YMK_TOKEN_MAX_E + 1];
    const int64_t p0 = (int64_t)blockIdx.x * a.per, p1 = min(a.pairs, p0 + a.per);
    sort_count<16>(a, p0, p1, count);
    for (int e = threadIdx.x; e <= a.E; e += 1024) {
        int n = 0;
        for (int i = 0; i < 16; ++i) n += count[i][e];
        a.hist[(size_t)blockIdx.x * (a.E + 1) + e] = n;
    }
}

__global__ __launch_bounds__(1024) void token_sort_place_kernel(SortArgs a) {
    __shared__ int32_t count[16][YMK_TOKEN_MAX_E + 1];
    __shared__ int32_t total[YMK_TOKEN_MAX_E + 1], mine[YMK_TOKEN_MAX_E + 1], start[YMK_TOKEN_MAX_E + 1];
    for (int e = threadIdx.x; e <= a.E; e += 1024) total[e] = mine[e] = 0;
    __syncthreads();
    // strands of workgroups per key: 1024 / (keys rounded up to a power of two), four histograms of a strand in flight, added up in LDS (integers)
    int keys = 1;
    while (keys <= a.E && keys < 512) keys <<= 1;
    const int strands = 1024 / keys, s = threadIdx.x / keys, e = threadIdx.x & (keys - 1), n = gridDim.x;
    if (e <= a.E) {
        int all = 0, before = 0;
        for (int b = s; b < n; b += 4 * strands) {
            int h[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) h[i] = b + i * strands < n ? a.hist[(size_t)(b + i * strands) * (a.E + 1) + e] : 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                all += h[i];
                before += b + i * strands < (int)blockIdx.x ? h[i] : 0;
            }
        }
        atomicAdd(&total[e], all);
        atomicAdd(&mine[e], before);
    }
    __syncthreads();
    sort_starts(total, a.E, start, blockIdx.x == 0 ? a.offsets : nullptr);
    for (int i = threadIdx.x; i <= a.E; i += 1024) start[i] += mine[i];
    __syncthreads();
    const int64_t p0 = (int64_t)blockIdx.x * a.per, p1 = min(a.pairs, p0 + a.per);
    sort_count<16>(a, p0, p1, count);
    sort_place<16>(a, p0, p1, count, start);
}

// -------------------------------------------------------------------------------------------------------- dispatch
struct MoveArgs {
    const char* x;
    char* xs;
    const float* scale;
    float* xs_scale;
    const int32_t* rows;
    int64_t ldx, ldxs, tokens;   // strides in bytes
    int32_t units, row, top_k;   // units of sizeof(U) bytes that cover a row of so many bytes
};

// One unit of a token per lane: read once, written to the rows of the token's choices.  A unit may start at any byte; the last one of a row ends with
// it, over bytes that the one before it writes as well (the same ones).
template <typename U>
__global__ __launch_bounds__(256) void token_dispatch_kernel(MoveArgs a) {
    typedef U Any __attribute__((aligned(1)));
    const int64_t n = a.tokens * a.units;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t t = n < 0x7fffffff ? (uint32_t)i / (uint32_t)a.units : i / a.units;
        const int j = (int)(i - t * a.units), at = min(j * (int)sizeof(U), a.row - (int)sizeof(U));
        const U v = *reinterpret_cast<const Any*>(a.x + t * a.ldx + at);
        for (int k = 0; k < a.top_k; ++k) {
            const int64_t r = a.rows[t * a.top_k + k];
            if ((uint64_t)r >= (uint64_t)(a.tokens * a.top_k)) continue;   // none, or no row of this plan
            *reinterpret_cast<Any*>(a.xs + r * a.ldxs + at) = v;
            if (a.scale && j == 0) a.xs_scale[r] = a.scale[t];
        }
    }
}

// --------------------------------------------------------------------------------------------------------- combine
struct CombineArgs {
    const void* ys;
    const int32_t* row;
    const float* w;
    void* y;
    int64_t tokens;
    int32_t ldys, ldy, units, C, top_k;
};

// V channels at p (any alignment): 16 bytes, or one
template <typename T, int V>
__device__ __forceinline__ void tk_load(const T* p, float (&v)[V]) {
    if constexpr (V == 1) v[0] = to_f32(*p);
    else row_widen(row_load<T, false>(p, V), v);
}
template <typename T, int V>
__device__ __forceinline__ void tk_store(T* p, const float (&v)[V]) {
    if constexpr (V == 1) from_f32(*p, v[0]);
    else row_store<T, false>(p, V, v);
}

// V channels of a token per lane (the last ones of a row end with it, over channels that the lane before has as well), KU choices in flight at a time,
// added in their order in fp32.  A pair without a row reads row 0 (there is one: the token's own pairs count) and takes nothing of it.
template <typename T, int V, int KU>
__global__ __launch_bounds__(256) void token_combine_kernel(CombineArgs a) {
    const int64_t n = a.tokens * a.units;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t t = n < 0x7fffffff ? (uint32_t)i / (uint32_t)a.units : i / a.units;
        const int c = min((int)(i - t * a.units) * V, a.C - V);
        float s[V];
#pragma unroll
        for (int e = 0; e < V; ++e) s[e] = 0.f;
        for (int k0 = 0; k0 < a.top_k; k0 += KU) {
            float v[KU][V], w[KU];
            int64_t r[KU];
#pragma unroll
            for (int k = 0; k < KU; ++k) {
                r[k] = k0 + k < a.top_k ? a.row[t * a.top_k + k0 + k] : -1;
                if (r[k] >= a.tokens * a.top_k) r[k] = -1;
                w[k] = a.w && k0 + k < a.top_k ? a.w[t * a.top_k + k0 + k] : 1.0f;
            }
#pragma unroll
            for (int k = 0; k < KU; ++k) tk_load<T, V>(static_cast<const T*>(a.ys) + (r[k] < 0 ? 0 : r[k]) * a.ldys + c, v[k]);
#pragma unroll
            for (int k = 0; k < KU; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e) s[e] = r[k] < 0 ? s[e] : fmaf(w[k], v[k][e], s[e]);
        }
        tk_store<T, V>(static_cast<T*>(a.y) + t * a.ldy + c, s);
    }
}

struct CombineBwdArgs {
    const void* dy;
    const void* ys;
    const int32_t* row;
    const float* w;
    void* dys;
    float* dw;
    int64_t tokens;
    int32_t lddy, ldys, lddys, units, C, top_k, group;
};

// A token belongs to `group` lanes (8..64) of a wave: per choice they scale the token's dy into its row and add up <dy, ys>.  dy of a token stays
// in the cache over its choices.  Where the last unit of a row overlaps the one before it, the shared channels count once.
template <typename T, int V>
__global__ __launch_bounds__(256) void token_combine_backward_kernel(CombineBwdArgs a) {
    const int lane = threadIdx.x & (a.group - 1), per = 256 / a.group;
    for (int64_t t = (int64_t)blockIdx.x * per + threadIdx.x / a.group; t < a.tokens; t += (int64_t)gridDim.x * per) {
        for (int k = 0; k < a.top_k; ++k) {
            const int64_t r = a.row[t * a.top_k + k];
            float dot = 0.f;
            if ((uint64_t)r < (uint64_t)(a.tokens * a.top_k)) {
                const float w = a.w[t * a.top_k + k];
                for (int j = lane; j < a.units; j += a.group) {
                    const int c = min(j * V, a.C - V), again = j * V - c;
                    float d[V], v[V];
                    tk_load<T, V>(static_cast<const T*>(a.dy) + t * a.lddy + c, d);
                    tk_load<T, V>(static_cast<const T*>(a.ys) + r * a.ldys + c, v);
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        dot = e < again ? dot : fmaf(d[e], v[e], dot);
                        d[e] *= w;
                    }
                    tk_store<T, V>(static_cast<T*>(a.dys) + r * a.lddys + c, d);
                }
            }
            for (int o = a.group >> 1; o > 0; o >>= 1) dot += __shfl_xor(dot, o);
            if (lane == 0) a.dw[t * a.top_k + k] = dot;
        }
    }
}

inline bool tk_al(const void* p, int64_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) == 0; }
inline bool tk_bad_plan(int64_t tokens, int32_t top_k) { return tokens < 0 || tokens >= (1ll << 30) || top_k < 1 || top_k > YMK_TOKEN_MAX_K || tokens * top_k >= (1ll << 30); }
inline unsigned tk_blocks(int64_t lanes) {
    const int64_t n = (lanes + 255) / 256;
    return (unsigned)(n < TK_MAX_BLOCKS ? n : TK_MAX_BLOCKS);
}

template <typename T, int V>
int tk_combine(const CombineArgs& a, void* stream) {
    const dim3 grid(tk_blocks(a.tokens * a.units)), block(256);
    if (a.top_k == 1) hipLaunchKernelGGL((token_combine_kernel<T, V, 1>), grid, block, 0, (hipStream_t)stream, a);
    else if (a.top_k == 2) hipLaunchKernelGGL((token_combine_kernel<T, V, 2>), grid, block, 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL((token_combine_kernel<T, V, 4>), grid, block, 0, (hipStream_t)stream, a);
    return ymk_launch_status();
}

}  // namespace

extern "C" size_t ymk_token_sort_workspace_bytes(int64_t tokens, int32_t top_k, int32_t E) {
    if (tokens <= 0 || top_k <= 0 || E <= 0 || tokens * top_k <= TK_SORT_ONE) return 0;
    return (size_t)TK_SORT_BLOCKS * (E + 1) * sizeof(int32_t);
}

extern "C" int ymk_token_sort(const void* idx, int32_t idx_bytes, int64_t tokens, int32_t top_k, int32_t E, int32_t* offsets, int32_t* src, int32_t* row,
                              void* workspace, size_t workspace_bytes, void* stream) {
    if ((idx_bytes != 4 && idx_bytes != 8) || tk_bad_plan(tokens, top_k) || E < 1 || E > YMK_TOKEN_MAX_E || !offsets) return YMK_E_BADARG;
    const int64_t pairs = tokens * top_k;
    if (pairs > 0 && (!idx || !src || !row || !tk_al(idx, idx_bytes))) return YMK_E_BADARG;
    SortArgs a{idx, pairs, idx_bytes == 8, E, (int32_t)pairs, offsets, src, row, static_cast<int32_t*>(workspace)};
    if (pairs <= TK_SORT_ONE) {   // none at all still writes the offsets
        hipLaunchKernelGGL(token_sort_one_kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream, a);
        return ymk_launch_status();
    }
    if (!workspace || workspace_bytes < ymk_token_sort_workspace_bytes(tokens, top_k, E)) return YMK_E_WORKSPACE;
    int64_t blocks = (pairs + 2047) / 2048;
    if (blocks > TK_SORT_BLOCKS) blocks = TK_SORT_BLOCKS;
    a.per = (int32_t)((pairs + blocks - 1) / blocks);
    blocks = (pairs + a.per - 1) / a.per;
    hipLaunchKernelGGL(token_sort_count_kernel, dim3((unsigned)blocks), dim3(1024), 0, (hipStream_t)stream, a);
    hipLaunchKernelGGL(token_sort_place_kernel, dim3((unsigned)blocks), dim3(1024), 0, (hipStream_t)stream, a);
    return ymk_launch_status();
}

extern "C" int ymk_token_dispatch(const void* x, int64_t ldx_bytes, int64_t row_bytes, const float* scale, void* xs, int64_t ldxs_bytes, float* xs_scale,
                                  const int32_t* row, int64_t tokens, int32_t top_k, void* stream) {
    if (tk_bad_plan(tokens, top_k) || row_bytes < 1 || row_bytes > (1 << 24) || ldx_bytes < row_bytes || ldxs_bytes < row_bytes || (scale && !xs_scale))
        return YMK_E_BADARG;
    if (tokens == 0) return YMK_OK;
    if (!x || !xs || !row) return YMK_E_BADARG;
    int u = 16;   // widest unit that a row holds
    while (u > row_bytes) u >>= 1;
    const MoveArgs a{static_cast<const char*>(x), static_cast<char*>(xs), scale, xs_scale, row, ldx_bytes, ldxs_bytes, tokens, (int32_t)((row_bytes + u - 1) / u), (int32_t)row_bytes, top_k};
    const dim3 grid(tk_blocks(tokens * a.units)), block(256);
    if (u == 16) hipLaunchKernelGGL(token_dispatch_kernel<u32x4>, grid, block, 0, (hipStream_t)stream, a);
    else if (u == 8) hipLaunchKernelGGL(token_dispatch_kernel<u32x2>, grid, block, 0, (hipStream_t)stream, a);
    else if (u == 4) hipLaunchKernelGGL(token_dispatch_kernel<uint32_t>, grid, block, 0, (hipStream_t)stream, a);
    else if (u == 2) hipLaunchKernelGGL(token_dispatch_kernel<uint16_t>, grid, block, 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL(token_dispatch_kernel<uint8_t>, grid, block, 0, (hipStream_t)stream, a);
    return ymk_launch_status();
}

extern "C" int ymk_token_combine(int32_t dtype, const void* ys, int32_t ldys, const int32_t* row, const float* w, void* y, int32_t ldy, int64_t tokens,
                                 int32_t top_k, int32_t C, void* stream) {
    if ((dtype != YMK_F32 && dtype != YMK_H16) || tk_bad_plan(tokens, top_k) || C < 1 || C > TK_MAX_C || ldys < C || ldy < C) return YMK_E_BADARG;
    if (tokens == 0) return YMK_OK;
    const int es = dtype == YMK_F32 ? 4 : 2;
    if (!ys || !row || !y || !tk_al(ys, es) || !tk_al(y, es)) return YMK_E_BADARG;
    const int V = C >= 16 / es ? 16 / es : 1;
    const CombineArgs a{ys, row, w, y, tokens, ldys, ldy, (C + V - 1) / V, C, top_k};
    if (dtype == YMK_F32) return V == 1 ? tk_combine<float, 1>(a, stream) : tk_combine<float, 4>(a, stream);
    return V == 1 ? tk_combine<h16_t, 1>(a, stream) : tk_combine<h16_t, 8>(a, stream);
}

extern "C" int ymk_token_combine_backward(int32_t dtype, const void* dy, int32_t lddy, const void* ys, int32_t ldys, const int32_t* row, const float* w,
                                          void* dys, int32_t lddys, float* dw, int64_t tokens, int32_t top_k, int32_t C, void* stream) {
    if ((dtype != YMK_F32 && dtype != YMK_H16) || tk_bad_plan(tokens, top_k) || C < 1 || C > TK_MAX_C || lddy < C || ldys < C || lddys < C) return YMK_E_BADARG;
    if (tokens == 0) return YMK_OK;
    const int es = dtype == YMK_F32 ? 4 : 2;
    if (!dy || !ys || !row || !w || !dys || !dw || !tk_al(dy, es) || !tk_al(ys, es) || !tk_al(dys, es)) return YMK_E_BADARG;
    const int V = C >= 16 / es ? 16 / es : 1;
    CombineBwdArgs a{dy, ys, row, w, dys, dw, tokens, lddy, ldys, lddys, (C + V - 1) / V, C, top_k, 8};
    while (a.group < 64 && a.group < a.units) a.group *= 2;
    const dim3 grid(tk_blocks(tokens * a.group)), block(256);
    if (dtype == YMK_F32) {
        if (V == 1) hipLaunchKernelGGL((token_combine_backward_kernel<float, 1>), grid, block, 0, (hipStream_t)stream, a);
        else hipLaunchKernelGGL((token_combine_backward_kernel<float, 4>), grid, block, 0, (hipStream_t)stream, a);
    } else if (V == 1) hipLaunchKernelGGL((token_combine_backward_kernel<h16_t, 1>), grid, block, 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL((token_combine_backward_kernel<h16_t, 8>), grid, block, 0, (hipStream_t)stream, a);
    return ymk_launch_status();
}
