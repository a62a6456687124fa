// Tokens sorted by expert and back (include/ymk_tokens.h): the stable sort of the (token, choice) pairs, the move of rows into expert order and
// the weighted sum back, with their gradients.  Nothing here multiplies matrices: the sort is bound by latency (a launch, two dependent reads),
// the moves by memory — each row is read once and written once.
#include "ymk_common.h"
#include "../../include/ymk_tokens.h"

#ifndef YMK_MAX_BLOCKS
#define TK_MAX_BLOCKS (256 * 32)
#else
#define TK_MAX_BLOCKS YMK_MAX_BLOCKS
#endif
#define TK_SORT_BLOCKS 256    // most workgroups of the two-launch sort: each sums the histograms of those before it
#define TK_SORT_ONE 8192      // pairs that one workgroup sorts alone, in one launch

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

__global__ __launch_bounds__(256) void token_sort_count_kernel(SortArgs a) {
    __shared__ int32_t count[4][YMK_TOKEN_MAX_E + 1];
    const int64_t p0 = (int64_t)blockIdx.x * a.per, p1 = min(a.pairs, p0 + a.per);
    sort_count<4>(a, p0, p1, count);
    for (int e = threadIdx.x; e <= a.E; e += 256) a.hist[(size_t)blockIdx.x * (a.E + 1) + e] = count[0][e] + count[1][e] + count[2][e] + count[3][e];
}

__global__ __launch_bounds__(256) void token_sort_place_kernel(SortArgs a) {
    __shared__ int32_t count[4][YMK_TOKEN_MAX_E + 1];
    __shared__ int32_t total[YMK_TOKEN_MAX_E + 1], mine[YMK_TOKEN_MAX_E + 1], start[YMK_TOKEN_MAX_E + 1];
    for (int e = threadIdx.x; e <= a.E; e += 256) total[e] = mine[e] = 0;
    __syncthreads();
    // strands of workgroups per key: 256 / (keys rounded up to a power of two), added up in LDS (integers)
    int keys = 1;
    while (keys <= a.E && keys < 256) keys <<= 1;
    const int strands = 256 / keys, s = threadIdx.x / keys;
    for (int e = threadIdx.x & (keys - 1); e <= a.E; e += keys) {
        int all = 0, before = 0;
        for (int b = s; b < (int)gridDim.x; b += strands) {
            const int n = a.hist[(size_t)b * (a.E + 1) + e];
            all += n;
            before += b < (int)blockIdx.x ? n : 0;
        }
        atomicAdd(&total[e], all);
        atomicAdd(&mine[e], before);
    }
    __syncthreads();
    sort_starts(total, a.E, start, blockIdx.x == 0 ? a.offsets : nullptr);
    for (int e = threadIdx.x; e <= a.E; e += 256) start[e] += mine[e];
    __syncthreads();
    const int64_t p0 = (int64_t)blockIdx.x * a.per, p1 = min(a.pairs, p0 + a.per);
    sort_count<4>(a, p0, p1, count);
    sort_place<4>(a, p0, p1, count, start);
}

// -------------------------------------------------------------------------------------------------------- dispatch
struct MoveArgs {
    const char* x;
    char* xs;
    const float* scale;
    float* xs_scale;
    const int32_t* row;
    int64_t ldx, ldxs, tokens;   // strides in bytes
    int32_t units, top_k;        // units of sizeof(U) bytes a row
};

// One unit of a token per lane: read once, written to the rows of the token's choices.
template <typename U>
__global__ __launch_bounds__(256) void token_dispatch_kernel(MoveArgs a) {
    const int64_t n = a.tokens * a.units;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t t = n < 0x7fffffff ? (uint32_t)i / (uint32_t)a.units : i / a.units;
        const int j = (int)(i - t * a.units);
        const U v = *reinterpret_cast<const U*>(a.x + t * a.ldx + (int64_t)j * sizeof(U));
        for (int k = 0; k < a.top_k; ++k) {
            const int64_t r = a.row[t * a.top_k + k];
            if (r < 0) continue;
            *reinterpret_cast<U*>(a.xs + r * a.ldxs + (int64_t)j * sizeof(U)) = v;
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
    int32_t ldys, ldy, units, top_k;
};

template <typename T, int V>
__device__ __forceinline__ void tk_load(const T* p, float (&v)[V]) {
    if constexpr (V == 1) v[0] = to_f32(*p);
    else load_vec_f32(p, v);
}
template <typename T, int V>
__device__ __forceinline__ void tk_store(T* p, const float (&v)[V]) {
    if constexpr (V == 1) from_f32(*p, v[0]);
    else store_vec_f32(p, v);
}

// V channels of a token per lane, the choices added in their order in fp32
template <typename T, int V>
__global__ __launch_bounds__(256) void token_combine_kernel(CombineArgs a) {
    const int64_t n = a.tokens * a.units;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t t = n < 0x7fffffff ? (uint32_t)i / (uint32_t)a.units : i / a.units;
        const int j = (int)(i - t * a.units);
        float s[V];
#pragma unroll
        for (int e = 0; e < V; ++e) s[e] = 0.f;
        for (int k = 0; k < a.top_k; ++k) {
            const int64_t r = a.row[t * a.top_k + k];
            if (r < 0) continue;
            const float w = a.w ? a.w[t * a.top_k + k] : 1.0f;
            float v[V];
            tk_load<T, V>(static_cast<const T*>(a.ys) + r * a.ldys + (int64_t)j * V, v);
#pragma unroll
            for (int e = 0; e < V; ++e) s[e] = fmaf(w, v[e], s[e]);
        }
        tk_store<T, V>(static_cast<T*>(a.y) + t * a.ldy + (int64_t)j * V, s);
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
    int32_t lddy, ldys, lddys, units, top_k, group;
};

// A token belongs to `group` lanes (8..64) of a wave: per choice they scale the token's dy into its row and add up <dy, ys>.  dy of a token stays
// in the cache over its choices.
template <typename T, int V>
__global__ __launch_bounds__(256) void token_combine_backward_kernel(CombineBwdArgs a) {
    const int lane = threadIdx.x & (a.group - 1), per = 256 / a.group;
    for (int64_t t = (int64_t)blockIdx.x * per + threadIdx.x / a.group; t < a.tokens; t += (int64_t)gridDim.x * per) {
        for (int k = 0; k < a.top_k; ++k) {
            const int64_t r = a.row[t * a.top_k + k];
            float dot = 0.f;
            if (r >= 0) {
                const float w = a.w[t * a.top_k + k];
                for (int j = lane; j < a.units; j += a.group) {
                    float d[V], v[V];
                    tk_load<T, V>(static_cast<const T*>(a.dy) + t * a.lddy + (int64_t)j * V, d);
                    tk_load<T, V>(static_cast<const T*>(a.ys) + r * a.ldys + (int64_t)j * V, v);
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        dot = fmaf(d[e], v[e], dot);
                        d[e] *= w;
                    }
                    tk_store<T, V>(static_cast<T*>(a.dys) + r * a.lddys + (int64_t)j * V, d);
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
    int64_t blocks = (pairs + 1023) / 1024;
    if (blocks > TK_SORT_BLOCKS) blocks = TK_SORT_BLOCKS;
    a.per = (int32_t)((pairs + blocks - 1) / blocks);
    blocks = (pairs + a.per - 1) / a.per;
    hipLaunchKernelGGL(token_sort_count_kernel, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, a);
    hipLaunchKernelGGL(token_sort_place_kernel, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, a);
    return ymk_launch_status();
}

extern "C" int ymk_token_dispatch(const void* x, int64_t ldx_bytes, int64_t row_bytes, const float* scale, void* xs, int64_t ldxs_bytes, float* xs_scale,
                                  const int32_t* row, int64_t tokens, int32_t top_k, void* stream) {
    if (tk_bad_plan(tokens, top_k) || row_bytes < 1 || row_bytes > (1 << 24) || ldx_bytes < row_bytes || ldxs_bytes < row_bytes || (scale && !xs_scale))
        return YMK_E_BADARG;
    if (tokens == 0) return YMK_OK;
    if (!x || !xs || !row) return YMK_E_BADARG;
    int u = 16;   // widest unit that divides the row, both strides and both addresses
    while (row_bytes % u || ldx_bytes % u || ldxs_bytes % u || !tk_al(x, u) || !tk_al(xs, u)) u >>= 1;
    const MoveArgs a{static_cast<const char*>(x), static_cast<char*>(xs), scale, xs_scale, row, ldx_bytes, ldxs_bytes, tokens, (int32_t)(row_bytes / u), top_k};
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
    if ((dtype != YMK_F32 && dtype != YMK_H16) || tk_bad_plan(tokens, top_k) || C < 1 || ldys < C || ldy < C) return YMK_E_BADARG;
    if (tokens == 0) return YMK_OK;
    const int es = dtype == YMK_F32 ? 4 : 2;
    if (!ys || !row || !y || !tk_al(ys, es) || !tk_al(y, es)) return YMK_E_BADARG;
    int V = 16 / es;
    if (C % V || ldys % V || ldy % V || !tk_al(ys, 16) || !tk_al(y, 16)) V = 1;
    const CombineArgs a{ys, row, w, y, tokens, ldys, ldy, C / V, top_k};
    const dim3 grid(tk_blocks(tokens * a.units)), block(256);
    if (dtype == YMK_F32) {
        if (V == 1) hipLaunchKernelGGL((token_combine_kernel<float, 1>), grid, block, 0, (hipStream_t)stream, a);
        else hipLaunchKernelGGL((token_combine_kernel<float, 4>), grid, block, 0, (hipStream_t)stream, a);
    } else if (V == 1) hipLaunchKernelGGL((token_combine_kernel<h16_t, 1>), grid, block, 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL((token_combine_kernel<h16_t, 8>), grid, block, 0, (hipStream_t)stream, a);
    return ymk_launch_status();
}

extern "C" int ymk_token_combine_backward(int32_t dtype, const void* dy, int32_t lddy, const void* ys, int32_t ldys, const int32_t* row, const float* w,
                                          void* dys, int32_t lddys, float* dw, int64_t tokens, int32_t top_k, int32_t C, void* stream) {
    if ((dtype != YMK_F32 && dtype != YMK_H16) || tk_bad_plan(tokens, top_k) || C < 1 || lddy < C || ldys < C || lddys < C) return YMK_E_BADARG;
    if (tokens == 0) return YMK_OK;
    const int es = dtype == YMK_F32 ? 4 : 2;
    if (!dy || !ys || !row || !w || !dys || !dw || !tk_al(dy, es) || !tk_al(ys, es) || !tk_al(dys, es)) return YMK_E_BADARG;
    int V = 16 / es;
    if (C % V || lddy % V || ldys % V || lddys % V || !tk_al(dy, 16) || !tk_al(ys, 16) || !tk_al(dys, 16)) V = 1;
    CombineBwdArgs a{dy, ys, row, w, dys, dw, tokens, lddy, ldys, lddys, C / V, top_k, 8};
    while (a.group < 64 && a.group < a.units) a.group *= 2;
    const dim3 grid(tk_blocks(tokens * a.group)), block(256);
    if (dtype == YMK_F32) {
        if (V == 1) hipLaunchKernelGGL((token_combine_backward_kernel<float, 1>), grid, block, 0, (hipStream_t)stream, a);
        else hipLaunchKernelGGL((token_combine_backward_kernel<float, 4>), grid, block, 0, (hipStream_t)stream, a);
    } else if (V == 1) hipLaunchKernelGGL((token_combine_backward_kernel<h16_t, 1>), grid, block, 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL((token_combine_backward_kernel<h16_t, 8>), grid, block, 0, (hipStream_t)stream, a);
    return ymk_launch_status();
}
