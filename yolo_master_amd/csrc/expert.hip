// The product of rows with their expert's matrix, and its gradients (include/ymk_tokens.h), on the matrix cores.
//
// One kernel body serves the three products.  The side whose index is contiguous in the output is called N, the other M:
//     y  = x W^T    N = output channels (rows of W[e], K contiguous)         M = rows of x (K contiguous)          K = Cin
//     dx = dy W     N = input channels (columns of W[e], N contiguous)       M = rows of dy (K contiguous)         K = Cout
//     dW = dy^T x   N = input channels (columns of x, N contiguous)          M = output channels (columns of dy)   K = the expert's rows
// A k-step takes 64 bytes of K per row of a K-contiguous side, and as many rows of a side whose own index is contiguous: either way a side's tile
// of a k-step is 64 * TILE bytes.  Both are brought straight into LDS (`buffer_load_dwordx4 ... lds`), whatever lies outside the matrix as lanes out
// of the buffer's range, which the hardware answers with zeros; so tails of rows, channels and K cost no other code.  A ring of four stages keeps
// three k-steps of transfers in flight across one barrier a k-step (counted vmcnt), and the fragments of the next k-step are read while the matrix
// instructions of this one run.
//
// Fragments are those of the 32 x 32 matrix instructions: lane l holds row l % 32 and the 16-byte pieces l / 32 and 2 + l / 32 of its 64 bytes — the
// order of K within a k-step is free as long as both sides use the same.  A side whose own index is contiguous is read through the transposing LDS
// load (16-bit) or element by element (fp32).  The N side's rows are permuted so that the 16 results a lane holds of a 32 x 32 block are 16
// CONSECUTIVE output channels (16-byte stores): row i of the block is channel ((i >> 2) & 1) * 16 + (i >> 3) * 4 + (i & 3).
#include <type_traits>

#include "ymk_common.h"
#include "glds.h"
#include "../../include/ymk_tokens.h"

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

#define EX_STAGES 4

namespace {

struct E4m3 {};   // element kind of the 8-bit product

struct ExArgs {
    const char* n;            // N side: W or x
    const char* m;            // M side: x or dy
    char* out;
    const float* bias;
    const float* n_scale;     // [E][N], with m_scale [rows]: 8-bit operands
    const float* m_scale;
    const int32_t* offsets;
    float* db;
    int64_t n_expert;         // bytes from one expert's N side (or output, dW) to the next
    int64_t out_expert;
    int32_t n_ld, m_ld;       // bytes
    int32_t out_ld;           // elements
    int32_t N, M, K;          // M: output channels (dW only); K: dW takes the expert's rows
    int32_t E, rows, act;
};

template <typename T> struct ExElem { static constexpr int ES = sizeof(T); };
template <> struct ExElem<E4m3> { static constexpr int ES = 1; };

struct ExFrag { u32x4 p[2]; };   // two 16-byte pieces of a row

template <typename T>
__device__ __forceinline__ f32x16 ex_mfma(const ExFrag& a, const ExFrag& b, f32x16 c) {
    if constexpr (std::is_same<T, E4m3>::value) {
        i32x8 x, y;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = (int)a.p[0][i]; x[4 + i] = (int)a.p[1][i];
            y[i] = (int)b.p[0][i]; y[4 + i] = (int)b.p[1][i];
        }
        return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(x, y, c, 0, 0, 0, 0, 0, 0);   // both e4m3, no block scales
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t x = a.p[q][e], y = b.p[q][e];
                c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(x), __uint_as_float(y), c, 0, 0, 0);
            }
        return c;
    } else {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
#ifdef YMK_H16_F16
            c = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(hw_h16x8, a.p[q]), __builtin_bit_cast(hw_h16x8, b.p[q]), c, 0, 0, 0);
#else
            c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(hw_h16x8, a.p[q]), __builtin_bit_cast(hw_h16x8, b.p[q]), c, 0, 0, 0);
#endif
        }
        return c;
    }
}

__device__ __forceinline__ u32x2 ex_read_tr(const char* p) {
#ifdef YMK_HOST_EMU
    return hostemu_ds_read_tr16_b64(p);
#else
    typedef __attribute__((address_space(3))) s16x4* lptr;
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lptr)(p)));
#endif
}

__device__ __forceinline__ int ex_perm(int i) { return ((i >> 2) & 1) * 16 + (i >> 3) * 4 + (i & 3); }   // i < 32

// One side's tile in LDS.  KC: K contiguous.
// `spread`: rows permuted (the N side; the transposing reader permutes its columns by itself, for either side).
//   KC:  row r at r * 64, its 16-byte piece c in slot c ^ ((r >> 1) & 3): eight consecutive rows read at the same piece cover 128 bytes of banks
//   !KC: k-row k at k * TILE * ES; 16-bit pieces c in slot c ^ ((k & 1) | (k & 2) << 1): the four k-rows a transposing read takes at once do
template <typename T, bool KC, int TILE>
struct ExSide {
    static constexpr int ES = ExElem<T>::ES, WT = TILE / 64, KS = 64 / ES;
    static constexpr int LPR = KC ? 4 : TILE * ES / 16;   // lanes (16-byte pieces) of an LDS row
    static constexpr int RPI = 64 / LPR;                  // rows a wave brings with one instruction (0 is impossible: TILE * ES <= 1024)

    const char* base;
    unsigned voff[WT];
    int32_t ld, K, kpiece, krow[WT];

    // first / limit: rows (KC) or elements (!KC) of the tile's own index from `base`'s origin; K in elements
    __device__ __forceinline__ void init(const char* origin, int32_t ld_, int first, int limit, int K_, bool spread, int wave, int lane) {
        ld = ld_;
        K = K_;
        const int lr = lane / LPR, pc = lane % LPR;
        if constexpr (KC) {
            const int sc = pc ^ ((lr >> 1) & 3);
            base = origin + (int64_t)first * ld;
            kpiece = sc * (16 / ES);
#pragma unroll
            for (int j = 0; j < WT; ++j) {
                int r = (j * 4 + wave) * RPI + lr;
                if (spread) r = (r & ~31) + ex_perm(r & 31);
                voff[j] = first + r < limit ? (unsigned)(r * ld + sc * 16) : 0x80000000u;
            }
        } else {
            base = origin + (int64_t)first * ES;
#pragma unroll
            for (int j = 0; j < WT; ++j) {
                const int k = (j * 4 + wave) * RPI + lr;
                const int sc = ES == 2 ? pc ^ ((k & 1) | ((k & 2) << 1)) : pc;
                krow[j] = k;
                voff[j] = first + sc * (16 / ES) < limit ? (unsigned)(k * ld + sc * 16) : 0x80000000u;
            }
        }
    }
    // bring k-step `step` to `dst` (this side's part of a stage); steps behind the last one bring zeros
    __device__ __forceinline__ void issue(int step, char* dst, int wave) const {
        const char* b = base + (KC ? (int64_t)step * 64 : (int64_t)step * KS * ld);
        const glds_rsrc rs = GLDS_MAKE_RSRC(b, 0x7fffffff);
        const int left = K - step * KS;
#pragma unroll
        for (int j = 0; j < WT; ++j) {
            const unsigned out = (KC ? kpiece : krow[j]) < left ? 0u : 0x80000000u;
            GLDS_BUFFER_LOAD_LDS(rs, dst + (j * 4 + wave) * 1024, voff[j] | out, 0);
        }
    }
    // fragment of the 32 rows at `r0` of the tile
    static __device__ __forceinline__ ExFrag read(const char* src, int r0, int lane) {
        ExFrag f;
        if constexpr (KC) {
            const int r = r0 + (lane & 31), s = (r >> 1) & 3, h = lane >> 5;
            f.p[0] = *reinterpret_cast<const u32x4*>(src + r * 64 + ((h ^ s) * 16));
            f.p[1] = *reinterpret_cast<const u32x4*>(src + r * 64 + (((2 + h) ^ s) * 16));
        } else if constexpr (ES == 2) {
            // 16 lanes read four k-rows of 16 elements, four lanes a row and 8 bytes a lane, and each gets one column: k-row (lane % 16) / 4,
            // elements of the permuted columns 4 * (lane % 4) .. + 3 of this half of the block
            const int i = lane & 15, g = (lane >> 4) & 1, h = lane >> 5, q = i & 3, kk = i >> 2;
            const int col = r0 + (q & 1) * 16 + (2 * g + (q >> 1)) * 4;
            const int slot = (col >> 3) ^ ((kk & 1) | ((kk & 2) << 1));
            const char* p = src + (h * 8 + kk) * (TILE * 2) + slot * 16 + (col & 4) * 2;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const u32x2 lo = ex_read_tr(p + (c * 16) * (TILE * 2)), hi = ex_read_tr(p + (c * 16 + 4) * (TILE * 2));
                f.p[c] = u32x4{lo.x, lo.y, hi.x, hi.y};
            }
        } else {
            const char* p = src + ((lane >> 5) * 4) * (TILE * 4) + (r0 + ex_perm(lane & 31)) * 4;
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) f.p[c][e] = *reinterpret_cast<const uint32_t*>(p + (c * 8 + e) * (TILE * 4));
        }
        return f;
    }
};

// The tile of a workgroup among all experts' tiles, from the offsets alone (the host does not know them).  Workgroups b, b + 8, ... run on one XCD:
// each XCD takes a contiguous range of tiles, and within it GM tiles of rows against all tiles of channels before the next GM.
struct ExTile { int e, m0, mend, n0; };
template <int TILE>
__device__ __forceinline__ bool ex_find(const ExArgs& a, ExTile& t) {
    constexpr int GM = 8, CH = YMK_TOKEN_MAX_E / 64;
    const int lane = threadIdx.x & 63, nt = (a.N + TILE - 1) / TILE;
    int incl[CH], first[CH], last[CH], total = 0;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int e = c * 64 + lane;
        first[c] = last[c] = 0;
        if (e < a.E) {
            first[c] = min(max(a.offsets[e], 0), a.rows);
            last[c] = min(max(a.offsets[e + 1], first[c]), a.rows);
        }
        int s = (last[c] - first[c] + TILE - 1) / TILE;
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(s, o);
            if (lane >= o) s += v;
        }
        incl[c] = total + s;
        total += __builtin_amdgcn_readlane(s, 63);
    }
    const int all = total * nt, per = (all + 7) / 8, slot = blockIdx.x >> 3, id = (blockIdx.x & 7) * per + slot;
    if (slot >= per || id >= all) return false;
    const int g = id / (GM * nt), size = min(GM, total - g * GM), r = id - g * (GM * nt), m = g * GM + r % size;
    t.n0 = r / size * TILE;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const unsigned long long past = __ballot(incl[c] > m);   // the first of them is the expert
        if (past) {
            const int l = __ffsll(past) - 1;   // read by lane number: the results are wave-uniform registers, as buffer addresses have to be
            t.e = c * 64 + l;
            const int f = __builtin_amdgcn_readlane(first[c], l);
            t.mend = __builtin_amdgcn_readlane(last[c], l);
            const int tiles = (t.mend - f + TILE - 1) / TILE;
            t.m0 = f + (m - (__builtin_amdgcn_readlane(incl[c], l) - tiles)) * TILE;
            return true;
        }
    }
    return false;
}

__device__ __forceinline__ float ex_act(float v, int act) {
    if (act == YMK_ACT_SILU) return silu_exact(v);
    if (act == YMK_ACT_GELU) return gelu_exact(v);
    if (act == YMK_ACT_SIGMOID) return sigmoid_exact(v);
    return v;
}

// NKC / MKC: K contiguous on that side.  DW: K is the expert's rows.  TO: output type.
template <typename T, typename TO, bool NKC, bool MKC, int TILE, bool DB>
__device__ __forceinline__ void ex_body(const ExArgs& a, const ExTile& t, int K, const char* nsrc, const char* msrc) {
    constexpr int WT = TILE / 64, SIDE = TILE * 64, STAGE = 2 * SIDE, LOADS = 2 * WT;
    extern __shared__ u32x4 ex_lds[];
    char* lds = reinterpret_cast<char*>(ex_lds);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), wn = wave & 1, wm = wave >> 1;
    typedef ExSide<T, NKC, TILE> NSide;
    typedef ExSide<T, MKC, TILE> MSide;
    NSide ns;
    MSide ms;
    ns.init(nsrc, a.n_ld, t.n0, a.N, K, true, wave, lane);
    ms.init(msrc, a.m_ld, t.m0, t.mend, K, false, wave, lane);
    auto issue = [&](int step) {
        char* dst = lds + (step & (EX_STAGES - 1)) * STAGE;
        ns.issue(step, dst, wave);
        ms.issue(step, dst + SIDE, wave);
    };
    f32x16 acc[WT][WT], accb[DB ? WT : 1];
#pragma unroll
    for (int i = 0; i < WT; ++i)
#pragma unroll
        for (int j = 0; j < WT; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
#pragma unroll
    for (int j = 0; j < (DB ? WT : 1); ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) accb[j][r] = 0.f;
    ExFrag ones;   // 1 in every element: the sum over K of the M side as a matrix product
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) ones.p[c][i] = sizeof(T) == 4 ? 0x3f800000u : pack_h16x2(1.f, 1.f);
    ExFrag fn[2][WT], fm[2][WT];
    auto read = [&](int step, ExFrag (&n)[WT], ExFrag (&m)[WT]) {
        const char* src = lds + (step & (EX_STAGES - 1)) * STAGE;
#pragma unroll
        for (int i = 0; i < WT; ++i) n[i] = NSide::read(src, (wn * WT + i) * 32, lane);
#pragma unroll
        for (int j = 0; j < WT; ++j) m[j] = MSide::read(src + SIDE, (wm * WT + j) * 32, lane);
    };
    const int nk = (K + NSide::KS - 1) / NSide::KS;
    // Stage k + 1 has to have landed for every wave, and every wave has to have its fragments of stage k in registers, before stage k's slot is
    // given to stage k + 4 and the fragments of stage k + 1 are read.
#pragma unroll
    for (int s = 0; s < EX_STAGES; ++s) issue(s);
    __builtin_amdgcn_s_waitcnt(GLDS_WAITCNT_VM((EX_STAGES - 1) * LOADS));
    GLDS_COMPILER_FENCE();
    __builtin_amdgcn_s_barrier();
    GLDS_COMPILER_FENCE();
    read(0, fn[0], fm[0]);
    auto step = [&](int k, ExFrag (&n)[WT], ExFrag (&m)[WT], ExFrag (&n2)[WT], ExFrag (&m2)[WT]) {
        __builtin_amdgcn_s_waitcnt(GLDS_WAITCNT_VM((EX_STAGES - 2) * LOADS));
        GLDS_WAIT_LGKM0();
        __builtin_amdgcn_s_barrier();
        GLDS_COMPILER_FENCE();
        issue(k + EX_STAGES);
        read(k + 1, n2, m2);
#pragma unroll
        for (int i = 0; i < WT; ++i)
#pragma unroll
            for (int j = 0; j < WT; ++j) acc[i][j] = ex_mfma<T>(n[i], m[j], acc[i][j]);
        if constexpr (DB) {
#pragma unroll
            for (int j = 0; j < WT; ++j) accb[j] = ex_mfma<T>(ones, m[j], accb[j]);
        }
    };
    for (int k = 0; k < nk; k += 2) {   // a step behind the last one multiplies zeros
        step(k, fn[0], fm[0], fn[1], fm[1]);
        step(k + 1, fn[1], fm[1], fn[0], fm[0]);
    }
    __builtin_amdgcn_s_waitcnt(GLDS_WAITCNT_VM(0));   // no transfer may reach LDS after the workgroup has ended

    // lane l: output row l % 32 of block j (permuted like the N side where the M side's own index is contiguous), 16 channels of block i
    const int h = lane >> 5;
    TO* out = reinterpret_cast<TO*>(a.out + (MKC ? 0 : t.e * a.out_expert));
#pragma unroll
    for (int j = 0; j < WT; ++j) {
        const int row = t.m0 + (wm * WT + j) * 32 + (MKC ? lane & 31 : ex_perm(lane & 31));
        if (row >= t.mend) continue;
        if constexpr (DB) {
            if (wn == 0 && h == 0) a.db[(int64_t)t.e * a.M + row] = accb[j][0];
        }
        const float ms_ = a.m_scale ? a.m_scale[row] : 1.f;
#pragma unroll
        for (int i = 0; i < WT; ++i) {
            const int ch = t.n0 + (wn * WT + i) * 32 + h * 16;
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int c = ch + q * 8;
                if (c >= a.N) continue;   // N is a multiple of 8 (fp32: of 4)
                float v[8];
                const bool tail = sizeof(TO) == 4 && c + 4 >= a.N;   // only the first four exist
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = acc[i][j][q * 8 + e];
                if (a.n_scale) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] *= ms_ * a.n_scale[(int64_t)t.e * a.N + c + e];
                }
                if (a.bias) {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (e < 4 || !tail) v[e] += a.bias[(int64_t)t.e * a.N + c + e];
                }
                if (a.act != YMK_ACT_NONE) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = ex_act(v[e], a.act);
                }
                TO* p = out + (int64_t)row * a.out_ld + c;
                if constexpr (sizeof(TO) == 4) {
                    store4(reinterpret_cast<float*>(p), v[0], v[1], v[2], v[3]);
                    if (!tail) store4(reinterpret_cast<float*>(p) + 4, v[4], v[5], v[6], v[7]);
                } else {
                    store_vec_f32(p, v);
                }
            }
        }
    }
}

// y and dx
template <typename T, typename TO, bool NKC, int TILE>
__global__ __launch_bounds__(256, TILE == 256 ? 1 : 2) void expert_rows_kernel(ExArgs a) {
    ExTile t;
    if (!ex_find<TILE>(a, t)) return;
    ex_body<T, TO, NKC, true, TILE, false>(a, t, a.K, a.n + t.e * a.n_expert, a.m);
}

// dW (and, by the workgroups of the first channels, db)
template <typename T, typename TO, int TILE>
__global__ __launch_bounds__(256, TILE == 256 ? 1 : 2) void expert_dw_kernel(ExArgs a) {
    const int nt = (a.N + TILE - 1) / TILE, mt = (a.M + TILE - 1) / TILE, per = (gridDim.x + 7) / 8;
    const int id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (id >= a.E * nt * mt) return;
    ExTile t;
    t.e = id / (nt * mt);
    t.m0 = id / nt % mt * TILE;
    t.mend = a.M;
    t.n0 = id % nt * TILE;
    const int first = min(max(a.offsets[t.e], 0), a.rows), last = min(max(a.offsets[t.e + 1], first), a.rows);
    const char* n = a.n + (int64_t)first * a.n_ld;
    const char* m = a.m + (int64_t)first * a.m_ld;
    if (a.db && t.n0 == 0) ex_body<T, TO, false, false, TILE, true>(a, t, last - first, n, m);
    else ex_body<T, TO, false, false, TILE, false>(a, t, last - first, n, m);
}

template <auto Kernel>
int ex_launch(const ExArgs& a, int64_t blocks, size_t lds, void* stream) {
    if (blocks <= 0) return YMK_OK;
    if (blocks > 0x7fffffff) return YMK_E_BADARG;
    static YmkOncePerDevice once;
    if (once.need()) {
        if (hipFuncSetAttribute(reinterpret_cast<const void*>(Kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess) return YMK_E_LAUNCH;
        once.done();
    }
    hipLaunchKernelGGL(Kernel, dim3((unsigned)blocks), dim3(256), lds, (hipStream_t)stream, a);
    return ymk_launch_status();
}

// workgroups that hold every tile of rows whatever the offsets say, in whole rounds of the 8 XCDs
inline int64_t ex_blocks(int64_t rows, int E, int N, int tile) {
    const int64_t mt = rows / tile + (rows < E ? rows : E), nt = (N + tile - 1) / tile;
    return (mt * nt + 7) / 8 * 8;
}

template <typename T, typename TO, bool NKC>
int ex_rows(const ExArgs& a, void* stream) {
    constexpr int TILE = 128;
    return ex_launch<expert_rows_kernel<T, TO, NKC, TILE>>(a, ex_blocks(a.rows, a.E, a.N, TILE), EX_STAGES * 2 * TILE * 64, stream);
}
template <typename T, typename TO>
int ex_dw(const ExArgs& a, void* stream) {
    constexpr int TILE = 128;
    const int64_t blocks = (int64_t)a.E * ((a.N + TILE - 1) / TILE) * ((a.M + TILE - 1) / TILE);
    return ex_launch<expert_dw_kernel<T, TO, TILE>>(a, (blocks + 7) / 8 * 8, EX_STAGES * 2 * TILE * 64, stream);
}

inline bool ex_bad16(const void* p) { return !p || (reinterpret_cast<uintptr_t>(p) & 15); }
inline bool ex_bad_ld(int64_t ld, int64_t C, int es) { return ld < C || ld * es % 16 || ld * es >= (1 << 23); }
inline bool ex_bad_sizes(int64_t rows, int32_t E, int32_t Cin, int32_t Cout) {
    return rows < 0 || rows >= (1ll << 30) || E < 1 || E > YMK_TOKEN_MAX_E || Cin < 1 || Cout < 1;
}

}  // namespace

extern "C" int ymk_expert_linear(int32_t dtype, int32_t out_dtype, const void* x, int32_t ldx, const float* x_scale, const void* w, const float* w_scale,
                                 const float* bias, const int32_t* offsets, void* y, int32_t ldy, int64_t rows, int32_t E, int32_t Cin, int32_t Cout,
                                 int32_t act, void* stream) {
    const bool f8 = dtype == YMK_E4M3;
    if ((dtype != YMK_F32 && dtype != YMK_H16 && !f8) || (out_dtype != dtype && !(f8 && (out_dtype == YMK_F32 || out_dtype == YMK_H16))) ||
        ex_bad_sizes(rows, E, Cin, Cout) || act < YMK_ACT_NONE || act > YMK_ACT_GELU || !offsets || (f8 && (!x_scale || !w_scale)) || (!f8 && (x_scale || w_scale)))
        return YMK_E_BADARG;
    const int es = f8 ? 1 : dtype == YMK_F32 ? 4 : 2, eo = out_dtype == YMK_F32 ? 4 : 2;
    if (rows == 0) return YMK_OK;
    if (Cin * es % 16 || Cout % (f8 ? 8 : 16 / es) || ex_bad16(x) || ex_bad16(w) || ex_bad16(y) || ex_bad_ld(ldx, Cin, es) || ex_bad_ld(Cin, Cin, es) || ex_bad_ld(ldy, Cout, eo))
        return YMK_E_BADARG;
    const ExArgs a{static_cast<const char*>(w), static_cast<const char*>(x), static_cast<char*>(y), bias, w_scale, x_scale, offsets, nullptr,
                   (int64_t)Cout * Cin * es, 0, Cin * es, ldx * es, ldy, Cout, 0, Cin, E, (int32_t)rows, act};
    if (f8) return out_dtype == YMK_F32 ? ex_rows<E4m3, float, true>(a, stream) : ex_rows<E4m3, h16_t, true>(a, stream);
    return dtype == YMK_F32 ? ex_rows<float, float, true>(a, stream) : ex_rows<h16_t, h16_t, true>(a, stream);
}

extern "C" int ymk_expert_linear_dx(int32_t dtype, const void* dy, int32_t lddy, const void* w, const int32_t* offsets, void* dx, int32_t lddx,
                                    int64_t rows, int32_t E, int32_t Cin, int32_t Cout, void* stream) {
    if ((dtype != YMK_F32 && dtype != YMK_H16) || ex_bad_sizes(rows, E, Cin, Cout) || !offsets) return YMK_E_BADARG;
    const int es = dtype == YMK_F32 ? 4 : 2;
    if (rows == 0) return YMK_OK;
    if (Cin * es % 16 || Cout * es % 16 || ex_bad16(dy) || ex_bad16(w) || ex_bad16(dx) || ex_bad_ld(lddy, Cout, es) || ex_bad_ld(Cin, Cin, es) || ex_bad_ld(lddx, Cin, es))
        return YMK_E_BADARG;
    const ExArgs a{static_cast<const char*>(w), static_cast<const char*>(dy), static_cast<char*>(dx), nullptr, nullptr, nullptr, offsets, nullptr,
                   (int64_t)Cout * Cin * es, 0, Cin * es, lddy * es, lddx, Cin, 0, Cout, E, (int32_t)rows, YMK_ACT_NONE};
    return dtype == YMK_F32 ? ex_rows<float, float, false>(a, stream) : ex_rows<h16_t, h16_t, false>(a, stream);
}

extern "C" int ymk_expert_linear_dw(int32_t dtype, int32_t dw_dtype, const void* dy, int32_t lddy, const void* x, int32_t ldx, const int32_t* offsets,
                                    void* dw, float* db, int64_t rows, int32_t E, int32_t Cin, int32_t Cout, void* stream) {
    if ((dtype != YMK_F32 && dtype != YMK_H16) || (dw_dtype != dtype && dw_dtype != YMK_F32) || ex_bad_sizes(rows, E, Cin, Cout) || !offsets || ex_bad16(dw))
        return YMK_E_BADARG;
    const int es = dtype == YMK_F32 ? 4 : 2, eo = dw_dtype == YMK_F32 ? 4 : 2;
    if (Cin * es % 16 || Cout * es % 16 || ex_bad_ld(Cin, Cin, eo)) return YMK_E_BADARG;
    if (rows > 0 && (ex_bad16(dy) || ex_bad16(x) || ex_bad_ld(lddy, Cout, es) || ex_bad_ld(ldx, Cin, es))) return YMK_E_BADARG;
    const ExArgs a{static_cast<const char*>(x), static_cast<const char*>(dy), static_cast<char*>(dw), nullptr, nullptr, nullptr, offsets, db,
                   0, (int64_t)Cout * Cin * eo, ldx * es, lddy * es, Cin, Cin, Cout, 0, E, (int32_t)rows, YMK_ACT_NONE};
    if (dtype == YMK_F32) return ex_dw<float, float>(a, stream);
    return dw_dtype == YMK_F32 ? ex_dw<h16_t, float>(a, stream) : ex_dw<h16_t, h16_t>(a, stream);
}
