// The product of rows with their expert's matrix, and its gradients (include/ymk_tokens.h), on the matrix cores.
//
// One kernel body serves the three products.  The side whose index is contiguous in the output is called N, the other M:
//     y  = x W^T    N = output channels (rows of W[e], K contiguous)         M = rows of x (K contiguous)          K = Cin
//     dx = dy W     N = input channels (columns of W[e], N contiguous)       M = rows of dy (K contiguous)         K = Cout
//     dW = dy^T x   N = input channels (columns of x, N contiguous)          M = output channels (columns of dy)   K = the expert's rows
// A k-step takes 128 bytes of K per row of a K-contiguous side (whole cache lines: with 64-byte steps the same bytes took twice the requests and the
// transfers alone ran at 10 instead of 13 TB/s), and as many rows of a side whose own index is contiguous: either way a side's tile of a k-step is
// 128 * TILE bytes.  Both are brought straight into LDS (`buffer_load_dwordx4 ... lds`), whatever lies outside the matrix as lanes out of the
// buffer's range, which the hardware answers with zeros; so tails of rows, channels and K cost no other code.  A k-step is multiplied in two
// halves: while the matrix instructions of one run, the fragments of the next are read into the other half of the registers.  A side's tile of a step is
// a unit of a ring of five: the M side's unit of a step is brought during an earlier step's second half and the N side's during a first half, so that
// transfers (and their LDS writes) go on evenly all the time, two to three halves ahead, with one barrier a step.
//
// Measured (MI355X, two cards; a large library product reaches 1440 TFLOP/s in bf16, 2710 in e4m3, 154 in fp32, a large copy 5.0-5.4 TB/s): 32768 rows over 8
// experts, 1024 -> 4096 in bf16: y 291-296 us (930-945 TFLOP/s), dx 308-315, dW and db 283-288; 4096 -> 4096: 872-924 us (1190-1260); 65532 rows over 32
// experts, 2048 -> 4096 in e4m3 with SiLU 614-641 us (1720-1790).  What bounds it: the transfers (copies of the kernel without its matrix instructions took 0.85
// of the whole, without its transfers 0.8) and, where K is short, the results' turn and the activation, which the one workgroup of a CU does not overlap with
// anything.  Workgroups that take tile after tile and bring the next one's first step under the results of the last gained nothing (292 against 293 us,
// e4m3 778 against 568).
//
// Fragments are those of the 32 x 32 matrix instructions: lane l holds row l % 32 and the 16-byte pieces l / 32 and 2 + l / 32 of a half's 64 bytes — the
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

#define EX_UNITS 5
#ifdef YMK_HOST_EMU
#define EX_SCHED_FENCE() ((void)0)
#else
#define EX_SCHED_FENCE() __builtin_amdgcn_sched_barrier(0)
#endif

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

// Part q of a 16-byte piece of e4m3 codes in bfloat16: exact (4 bits of 8, and the exponents fit), so are the products in 32 bits.  The 8-bit matrix
// instructions add 16 products at the largest one's exponent and drop what lies below 2^-13 of it (a 2048-deep sum of normal values is off by 1.5e-5 rms,
// through bfloat16 by 9e-8).  DEEP sums go through the 16-bit instructions at half the rate: those of fp32 outputs, whose half step is 2^-24 (65532 rows over 32
// experts, 2048 -> 4096: 829 us at 8 bits, 1219), and those of tiles of up to 64 rows, which wait for the weights anyway (6 rows of 64 experts 15.0 and 15.7 us,
// 128 of 8 14.7 and 15.8, 992 of 32 14.9 and 16.5).  With more rows and 16-bit outputs the loss is far below the output's own rounding (error against 64 bits
// in bfloat16 1.679e-3 either way, in binary16 2.099e-4 for 2.094e-4) and the 8-bit instruction stays.
__device__ __forceinline__ u32x4 ex_widen(const u32x4& p, int q) {
    typedef __bf16 pair __attribute__((ext_vector_type(2)));
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t codes = p[2 * q + i];
        const pair lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, 1.0f, false), hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, 1.0f, true);
        w[2 * i] = __builtin_bit_cast(uint32_t, lo);
        w[2 * i + 1] = __builtin_bit_cast(uint32_t, hi);
    }
    return w;
}
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

template <typename T, bool DEEP>
__device__ __forceinline__ f32x16 ex_mfma(const ExFrag& a, const ExFrag& b, f32x16 c) {
    if constexpr (std::is_same<T, E4m3>::value && DEEP) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, ex_widen(a.p[i >> 1], i & 1)), __builtin_bit_cast(bf16x8, ex_widen(b.p[i >> 1], i & 1)), c, 0, 0, 0);
        return c;
    } else if constexpr (std::is_same<T, E4m3>::value) {
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

// c + the elements of a fragment
template <typename T>
__device__ __forceinline__ float ex_sum(const ExFrag& f, float c) {
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w = f.p[q][i];
            if constexpr (sizeof(T) == 4) c += __uint_as_float(w);
            else c = dot2_h16(w, pack_h16x2(1.f, 1.f), c);
        }
    return c;
}
// hi + v with its rounding error added to lo (the two-sum of Knuth, The Art of Computer Programming 2, 4.2.2).  K of db is the expert's rows: as one running
// sum, 12617 normal values in fp32 were 1.4e-6 off.  Four steps (64 additions of one value, or of two 16-bit ones) are a sum of their own, which goes into
// hi and lo: 1.5e-7.  (Every fragment into hi and lo took dW and db of 32768 rows over 8 experts, 1024 -> 4096 in bf16 from 264 to 287 us, this costs nothing.)
__device__ __forceinline__ void ex_add(float& hi, float& lo, float v) {
    const float t = hi + v, w = t - hi;
    lo += (hi - (t - w)) + (v - w);
    hi = t;
}

// A raw buffer at p (an offset with bit 31 set is out of its range: zeros, no access), and 16 bytes a lane from it to LDS at dst (wave-uniform) + lane * 16.
// The transfer is written as assembly because the compiler waits for ALL transfers before any transposing LDS read when it knows of them (dx of 32768 x
// 4096 by 1024 in bf16: 530 us).  It has no register result; this kernel's counted waits and barriers order it against the reads of its bytes.
#ifdef YMK_HOST_EMU
typedef hostemu_rsrc ExBuffer;
__device__ __forceinline__ ExBuffer ex_buffer(const char* p) { return GLDS_MAKE_RSRC(p, 0x7fffffff); }
__device__ __forceinline__ void ex_load_lds(const ExBuffer& b, char* dst, unsigned voff) { GLDS_BUFFER_LOAD_LDS(b, dst, voff, 0); }
#else
typedef u32x4 ExBuffer;
__device__ __forceinline__ ExBuffer ex_buffer(const char* p) {
    const uint64_t a = reinterpret_cast<uint64_t>(p);
    ExBuffer b{(uint32_t)a, (uint32_t)(a >> 32) & 0xffffu, 0x7fffffffu, 0x00020000u};
    asm volatile("s_nop 4" : "+s"(b));   // a scalar register that a vector instruction has written may be read by a transfer five wait states later
    return b;
}
__device__ __forceinline__ void ex_load_lds(const ExBuffer& b, char* dst, unsigned voff) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"((uint32_t)(uintptr_t)(glds_lptr)dst), "v"(voff), "s"(b) : "memory", "m0");   // M0 needs one wait state
}
#endif

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
//   KC:  row r at r * 128, its 16-byte piece c in slot c ^ ((r >> 1) & 7): the 16 rows that a 16-byte read serves at once (0-3, 12-15, 20-23, 24-27 and
//        their complement, or 16 in a row) cover all 64 banks
//   !KC: k-row k at k * TILE * ES; 16-bit pieces c in slot c ^ ((k & 3) << 2), in rows of 128 bytes c ^ (k & 2) << 1: the four k-rows by 64 bytes that half
//        a wave's transposing read takes do
template <typename T, bool KC, int TILE>
struct ExSide {
    static constexpr int ES = ExElem<T>::ES, KS = 128 / ES;   // elements of K a step
    static constexpr int LPR = KC ? 8 : TILE * ES / 16;        // lanes (16-byte pieces) of an LDS row
    static constexpr int RPI = 64 / LPR;                       // rows a wave brings with one transfer (TILE * ES <= 1024)
    static constexpr int LOADS = TILE / 32;                    // transfers of a wave a step

    static __device__ __forceinline__ int swizzle(int k) { return TILE >= 128 ? (k & 3) << 2 : (k & 2) << 1; }

    const char* base;
    unsigned voff[LOADS];
    int32_t ld, K, kfirst[KC ? 1 : LOADS];

    // first / limit: the tile's own index, counted from `origin`; K in elements
    __device__ __forceinline__ void init(const char* origin, int32_t ld_, int first, int limit, int K_, bool spread, int wave, int lane) {
        ld = ld_;
        K = K_;
        const int lr = lane / LPR, pc = lane % LPR;
        if constexpr (KC) {
            const int sc = pc ^ ((((wave & 1) * 8 + lr) >> 1) & 7);   // row (j * 4 + wave) * 8 + lr
            base = origin + (int64_t)first * ld;
            kfirst[0] = sc * (16 / ES);
#pragma unroll
            for (int j = 0; j < LOADS; ++j) {
                int r = (j * 4 + wave) * RPI + lr;
                if (spread) r = (r & ~31) + ex_perm(r & 31);
                voff[j] = first + r < limit ? (unsigned)(r * ld + sc * 16) : 0x80000000u;
            }
        } else {
            base = origin + (int64_t)first * ES;
#pragma unroll
            for (int j = 0; j < LOADS; ++j) {
                const int k = (j * 4 + wave) * RPI + lr;
                const int sc = ES == 2 ? pc ^ swizzle(k) : pc;
                kfirst[j] = k;
                voff[j] = first + sc * (16 / ES) < limit ? (unsigned)(k * ld + sc * 16) : 0x80000000u;
            }
        }
    }
    // k-step `step` as a buffer; steps behind the last one bring zeros
    struct Step { ExBuffer rs; int left; };
    __device__ __forceinline__ Step at(int step) const {
        return {ex_buffer(base + (KC ? (int64_t)step * 128 : (int64_t)step * KS * ld)), K - step * KS};
    }
    // bring transfer j of it to `dst` (this side's part of a slot)
    __device__ __forceinline__ void issue(const Step& s, int j, char* dst, int wave) const {
        const unsigned out = kfirst[KC ? 0 : j] < s.left ? 0u : 0x80000000u;
        ex_load_lds(s.rs, dst + (j * 4 + wave) * 1024, voff[j] | out);
    }
    // fragment of the 32 rows at `r0` of the tile, half `half` of the step
    static __device__ __forceinline__ ExFrag read(const char* src, int r0, int half, int lane) {
        ExFrag f;
        if constexpr (KC) {
            const int r = r0 + (lane & 31), s = (r >> 1) & 7, c = half * 4 + (lane >> 5);
            f.p[0] = *reinterpret_cast<const u32x4*>(src + r * 128 + ((c ^ s) * 16));
            f.p[1] = *reinterpret_cast<const u32x4*>(src + r * 128 + (((c + 2) ^ s) * 16));
        } else if constexpr (ES == 2) {
            // 16 lanes read four k-rows of 16 elements, four lanes a row and 8 bytes a lane, and each gets one column: k-row (lane % 16) / 4,
            // elements of the permuted columns 4 * (lane % 4) .. + 3 of this half of the block
            const int i = lane & 15, g = (lane >> 4) & 1, h = lane >> 5, q = i & 3, kk = i >> 2;
            const int col = r0 + (q & 1) * 16 + (2 * g + (q >> 1)) * 4;
            const int slot = (col >> 3) ^ swizzle(kk);
            const char* p = src + (half * 32 + h * 8 + kk) * (TILE * 2) + slot * 16 + (col & 4) * 2;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const u32x2 lo = ex_read_tr(p + (c * 16) * (TILE * 2)), hi = ex_read_tr(p + (c * 16 + 4) * (TILE * 2));
                f.p[c] = u32x4{lo.x, lo.y, hi.x, hi.y};
            }
        } else {
            const char* p = src + (half * 16 + (lane >> 5) * 4) * (TILE * 4) + (r0 + ex_perm(lane & 31)) * 4;
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
template <int TM, int TN>
__device__ __forceinline__ bool ex_find(const ExArgs& a, ExTile& t) {
    constexpr int GM = 8, CH = YMK_TOKEN_MAX_E / 64;
    const int lane = threadIdx.x & 63, nt = (a.N + TN - 1) / TN;
    int incl[CH], first[CH], last[CH], total = 0;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int e = c * 64 + lane;
        first[c] = last[c] = incl[c] = 0;
        if (c * 64 >= a.E) continue;   // for the whole wave
        if (e < a.E) {
            first[c] = min(max(a.offsets[e], 0), a.rows);
            last[c] = min(max(a.offsets[e + 1], first[c]), a.rows);
        }
        int s = (last[c] - first[c] + TM - 1) / TM;
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(s, o);
            if (lane >= o) s += v;
        }
        incl[c] = total + s;
        total += __builtin_amdgcn_readlane(s, 63);
    }
    if ((int64_t)total * nt > 0x7ffffff0) return false;   // offsets that are no offsets: the host's grid holds every tile of ascending ones
    const int all = total * nt, per = (all + 7) / 8, slot = blockIdx.x >> 3, id = (blockIdx.x & 7) * per + slot;
    if (slot >= per || id >= all) return false;
    const int g = id / (GM * nt), size = min(GM, total - g * GM), r = id - g * (GM * nt), m = g * GM + r % size;
    t.n0 = r / size * TN;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const unsigned long long past = __ballot(incl[c] > m);   // the first of them is the expert
        if (past) {
            const int l = __ffsll(past) - 1;   // read by lane number: the results are wave-uniform registers, as buffer addresses have to be
            t.e = c * 64 + l;
            const int f = __builtin_amdgcn_readlane(first[c], l);
            t.mend = __builtin_amdgcn_readlane(last[c], l);
            const int tiles = (t.mend - f + TM - 1) / TM;
            t.m0 = f + (m - (__builtin_amdgcn_readlane(incl[c], l) - tiles)) * TM;
            return true;
        }
    }
    return false;
}

// The activation of an fp32 output in the exact forms; of a 16-bit one in short forms (the exact ones take about 50 instructions an element, more
// than the products of a 2048-wide row): a few units of 2^-23 around zero, up to 2^-17 where the exponential's argument is near its end (rounded at 2^-18
// there), zero for results below 2^-118 (a reciprocal that is subnormal).  GELU = x Phi(x) through erfc(z) = t exp(-z^2 + p(t)), t = 1 / (1 + z / 2): the Chebyshev fit
// of Press et al., Numerical Recipes (2nd ed., 6.2), relative error 1.2e-7 everywhere, so the negative tail keeps its digits.
template <int ACT, bool SHORT>
__device__ __forceinline__ float ex_act(float v) {
    if constexpr (ACT == YMK_ACT_SILU) return SHORT ? silu_f(v) : silu_exact(v);
    else if constexpr (ACT == YMK_ACT_SIGMOID) return SHORT ? __builtin_amdgcn_rcpf(1.0f + __expf(-v)) : sigmoid_exact(v);
    else if constexpr (ACT == YMK_ACT_GELU) {
        if constexpr (!SHORT) return gelu_exact(v);
        const float z = fabsf(v) * 0.70710678118654752f, t = __builtin_amdgcn_rcpf(fmaf(z, 0.5f, 1.0f));
        float p = 0.17087277f;
        p = fmaf(p, t, -0.82215223f);
        p = fmaf(p, t, 1.48851587f);
        p = fmaf(p, t, -1.13520398f);
        p = fmaf(p, t, 0.27886807f);
        p = fmaf(p, t, -0.18628806f);
        p = fmaf(p, t, 0.09678418f);
        p = fmaf(p, t, 0.37409196f);
        p = fmaf(p, t, 1.00002368f);
        p = fmaf(p, t, -1.26551223f);
        const float half_erfc = 0.5f * t * __expf(fmaf(-z, z, p));
        return v * (v > 0.f ? 1.0f - half_erfc : half_erfc);   // +infinity stays: v - v * 0 would be no number
    } else return v;
}

// NKC / MKC: K contiguous on that side (of dW, whose K is the expert's rows, neither).  TO: output type.  DB: the sums of the M side's rows over K as well.
template <typename T, typename TO, bool NKC, bool MKC, int TILE, bool DB>
__device__ __forceinline__ void ex_body(const ExArgs& a, const ExTile& t, int K, const char* nsrc, const char* msrc) {
    constexpr int WT = TILE / 64, UNIT = TILE * 128, LOADS = TILE / 32, CHUNKS = 2 * WT;
    constexpr bool DEEP = sizeof(TO) == 4 || TILE == 64;   // of 8-bit products
    extern __shared__ u32x4 ex_lds[];
    char* lds = reinterpret_cast<char*>(ex_lds);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), wn = wave & 1, wm = wave >> 1;
    typedef ExSide<T, NKC, TILE> NSide;
    typedef ExSide<T, MKC, TILE> MSide;
    NSide ns;
    MSide ms;
    ns.init(nsrc, a.n_ld, t.n0, a.N, K, true, wave, lane);
    ms.init(msrc, a.m_ld, t.m0, t.mend, K, false, wave, lane);
    constexpr int CH = WT * 32, LPR = CH / 8, RPI = 64 / LPR;   // a wave's channels, the lanes of an output row and the rows of a store
    const int c0 = t.n0 + wn * CH + (lane % LPR) * 8;
    float bias[8], scale[8], mscale[WT];   // fetched here: their latency is not the epilogue's
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        bias[e] = a.bias && c0 + e < a.N ? a.bias[(int64_t)t.e * a.N + c0 + e] : 0.f;
        scale[e] = a.n_scale && c0 + e < a.N ? a.n_scale[(int64_t)t.e * a.N + c0 + e] : 1.f;
    }
#pragma unroll
    for (int j = 0; j < WT; ++j) {
        const int row = t.m0 + (wm * WT + j) * 32 + (lane & 31);
        mscale[j] = a.m_scale && row < t.mend ? a.m_scale[row] : 1.f;
    }
    f32x16 acc[WT][WT];
    float accb[WT], sumb[WT], lowb[WT];   // DB: this lane's part of the sum over K of its M-side rows: the last steps', those before, and what their sum rounded off
#pragma unroll
    for (int i = 0; i < WT; ++i)
#pragma unroll
        for (int j = 0; j < WT; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
#pragma unroll
    for (int j = 0; j < WT; ++j) accb[j] = sumb[j] = lowb[j] = 0.f;
    // An fp32 matrix instruction adds two products: every 512 of K the accumulators go into sums of their own, so that no chain of additions is longer than
    // 256 or the number of such blocks.  dW, whose K is the expert's rows, of 53499 rows of normal values: 4.5e-7 off relative to the result, 4.1e-6 as one
    // chain; y of 4096 channels 4.1e-7 and 1.15e-6.  The accumulators of 256 x 256 leave no registers for it.  16-bit operands come 16 an instruction.
    constexpr bool FOLD = std::is_same<T, float>::value && TILE <= 128;
    f32x16 far[FOLD ? WT : 1][FOLD ? WT : 1];
    if constexpr (FOLD) {
#pragma unroll
        for (int i = 0; i < WT; ++i)
#pragma unroll
            for (int j = 0; j < WT; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) far[i][j][r] = 0.f;
    }
    auto fold = [&] {
#pragma unroll
        for (int i = 0; i < WT; ++i)
#pragma unroll
            for (int j = 0; j < WT; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    far[i][j][r] += acc[i][j][r];
                    acc[i][j][r] = 0.f;
                }
    };
    ExFrag fn[2][WT], fm[2][WT];   // the fragments of a step's two halves
    const int steps = (K + NSide::KS - 1) / NSide::KS;
    // Units in the order they are brought: N of step 0, M of step 0, N of 1, ...; unit u lies at (u % 5) * UNIT.  Step k's are free once every wave has the
    // fragments of its second half, which the barrier between the halves of step k says.  Before it unit 2 k + 4 (N of k + 2) may be brought, to where M
    // of k - 1 was; after it unit 2 k + 5 (M of k + 2), to where N of k was.  At the barrier all units up to 2 k + 3 have to have landed: those of step
    // k + 1, whose first half is read next.
    int un = 0;   // (2 k) % 5
    auto unit = [&](int u) { return lds + (u >= EX_UNITS ? u - EX_UNITS : u) * UNIT; };
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const auto n = ns.at(q);
        const auto m = ms.at(q);
#pragma unroll
        for (int j = 0; j < LOADS; ++j) ns.issue(n, j, lds + 2 * q * UNIT, wave);
#pragma unroll
        for (int j = 0; j < LOADS; ++j) ms.issue(m, j, lds + (2 * q + 1) * UNIT, wave);
    }
    __builtin_amdgcn_s_waitcnt(GLDS_WAITCNT_VM(2 * LOADS));
    GLDS_COMPILER_FENCE();
    __builtin_amdgcn_s_barrier();
    GLDS_COMPILER_FENCE();
#pragma unroll
    for (int i = 0; i < WT; ++i) {
        fn[0][i] = NSide::read(lds, (wn * WT + i) * 32, 0, lane);
        fm[0][i] = MSide::read(lds + UNIT, (wm * WT + i) * 32, 0, lane);
    }
    // The matrix instructions of half `h` with, between every few of them, the reads of one fragment of the next half and a transfer, in this order: left
    // to itself the compiler moves the matrix instructions (they need no memory) to the reads of their own fragments, and the transfers before them all.
    auto half = [&](auto H, const char* nsrc_, const char* msrc_, char* dst, const auto& next) {
        constexpr int h = decltype(H)::value;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            EX_SCHED_FENCE();
#pragma unroll
            for (int q = c * (WT * WT) / CHUNKS; q < (c + 1) * (WT * WT) / CHUNKS; ++q)
                acc[q / WT][q % WT] = ex_mfma<T, DEEP>(fn[h][q / WT], fm[h][q % WT], acc[q / WT][q % WT]);
            EX_SCHED_FENCE();
#pragma unroll
            for (int j = c * LOADS / CHUNKS; j < (c + 1) * LOADS / CHUNKS; ++j) {
                if constexpr (h == 0) ns.issue(next, j, dst, wave);
                else ms.issue(next, j, dst, wave);
            }
            if (c < WT) {
                fn[1 - h][c] = NSide::read(nsrc_, (wn * WT + c) * 32, 1 - h, lane);
                if constexpr (DB) accb[c] = ex_sum<T>(fm[h][c], accb[c]);
            } else {
                fm[1 - h][c - WT] = MSide::read(msrc_, (wm * WT + c - WT) * 32, 1 - h, lane);
            }
        }
        EX_SCHED_FENCE();
    };
    for (int k = 0; k < steps; ++k) {
        half(std::integral_constant<int, 0>{}, unit(un), unit(un + 1), unit(un + 4), ns.at(k + 2));
        __builtin_amdgcn_s_waitcnt(GLDS_WAITCNT_VM(LOADS));   // all but the unit that was brought last
        GLDS_WAIT_LGKM0();
        __builtin_amdgcn_s_barrier();
        GLDS_COMPILER_FENCE();
        half(std::integral_constant<int, 1>{}, unit(un + 2), unit(un + 3), unit(un), ms.at(k + 2));
        un = un + 2 >= EX_UNITS ? un + 2 - EX_UNITS : un + 2;
        if constexpr (FOLD) {
            if ((k & 15) == 15) fold();
        }
        if constexpr (DB) {
            if ((k & 3) == 3 || k == steps - 1) {
#pragma unroll
                for (int j = 0; j < WT; ++j) {
                    ex_add(sumb[j], lowb[j], accb[j]);
                    accb[j] = 0.f;
                }
            }
        }
    }
    if constexpr (FOLD) {
        fold();
#pragma unroll
        for (int i = 0; i < WT; ++i)
#pragma unroll
            for (int j = 0; j < WT; ++j) acc[i][j] = far[i][j];
    }
    __builtin_amdgcn_s_waitcnt(GLDS_WAITCNT_VM(0));   // the transfers of zeros behind the last step have landed: LDS is free once every wave is here
    __syncthreads();

    // Lane l holds output row l % 32 of block j (permuted like the N side where the M side's own index is contiguous) and 16 channels of block i.
    // A wave turns one block of 32 rows at a time through its own part of LDS, so that a row leaves as whole lines and the scales, the bias and
    // the activation are code of a short loop (inlined per accumulator they would overflow the instruction cache).
    constexpr int LD = CH + 4;   // 16 bytes of padding: eight rows written at once meet eight different banks
    float* turn = reinterpret_cast<float*>(lds) + wave * (32 * LD);
    static_assert(4 * 32 * LD * 4 <= EX_UNITS * UNIT, "the turning buffers fit the units");
    const int h = lane >> 5;
    TO* out = reinterpret_cast<TO*>(a.out + (MKC ? 0 : t.e * a.out_expert));
#pragma unroll
    for (int j = 0; j < WT; ++j) {
        const int row0 = t.m0 + (wm * WT + j) * 32;
        if (row0 >= t.mend) break;
        if constexpr (DB) {
            const int row = row0 + (MKC ? lane & 31 : ex_perm(lane & 31));
            float sum = sumb[j], low = lowb[j];   // lanes l and l + 32 hold the same row's other halves of K
            ex_add(sum, low, __shfl_xor(sumb[j], 32));
            low += __shfl_xor(lowb[j], 32);
            sum = fabsf(sum) < __uint_as_float(0x7f800000u) ? sum + low : sum;   // what an infinite sum rounds off is no number
            if (wn == 0 && h == 0 && row < t.mend) a.db[(int64_t)t.e * a.M + row] = sum;
        }
        float* w = turn + (MKC ? lane & 31 : ex_perm(lane & 31)) * LD + h * 16;
#pragma unroll
        for (int i = 0; i < WT; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = std::is_same<T, E4m3>::value ? acc[i][j][q * 4 + e] * mscale[j] : acc[i][j][q * 4 + e];
                store4(w + i * 32 + q * 4, v[0], v[1], v[2], v[3]);
            }
        __builtin_amdgcn_wave_barrier();   // only this wave's part: LDS operations of a wave stay in order
        auto some = [&](int r0, auto ACT) {   // RPI rows
            const int r = r0 + lane / LPR, row = row0 + r;
            float v[8];
            load4(turn + r * LD + (lane % LPR) * 8, v[0], v[1], v[2], v[3]);
            load4(turn + r * LD + (lane % LPR) * 8 + 4, v[4], v[5], v[6], v[7]);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[e] = std::is_same<T, E4m3>::value ? fmaf(v[e], scale[e], bias[e]) : v[e] + bias[e];
                v[e] = ex_act<decltype(ACT)::value, sizeof(TO) == 2>(v[e]);
            }
            if (row >= t.mend || c0 >= a.N) return;
            TO* p = out + (int64_t)row * a.out_ld + c0;
            if constexpr (sizeof(TO) == 4) {
                store4(reinterpret_cast<float*>(p), v[0], v[1], v[2], v[3]);
                if (c0 + 4 < a.N) store4(reinterpret_cast<float*>(p) + 4, v[4], v[5], v[6], v[7]);   // fp32 channels come in fours, the others in eights
            } else {
                store_vec_f32(p, v);
            }
        };
        auto block = [&](auto ACT) {
#pragma unroll 2
            for (int r0 = 0; r0 < 32; r0 += RPI) some(r0, ACT);
        };
        if (!MKC || !NKC || a.act == YMK_ACT_NONE) {
#pragma unroll
            for (int r0 = 0; r0 < 32; r0 += RPI) some(r0, std::integral_constant<int, YMK_ACT_NONE>{});
        } else if (a.act == YMK_ACT_SILU) block(std::integral_constant<int, YMK_ACT_SILU>{});
        else if (a.act == YMK_ACT_GELU) block(std::integral_constant<int, YMK_ACT_GELU>{});
        else block(std::integral_constant<int, YMK_ACT_SIGMOID>{});
        __builtin_amdgcn_wave_barrier();
    }
}

// y and dx
template <typename T, typename TO, bool NKC, int TILE>
__global__ __launch_bounds__(256, TILE == 256 ? 1 : TILE == 128 ? 2 : 4) void expert_rows_kernel(ExArgs a) {
    ExTile t;
    if (!ex_find<TILE, TILE>(a, t)) return;
    ex_body<T, TO, NKC, true, TILE, false>(a, t, a.K, a.n + t.e * a.n_expert, a.m);
}

// y for few rows an expert: bound by the bytes of the experts' matrices.  A workgroup takes 16 rows by 32 channels; its four waves take the 128-byte pieces
// of K in turn, EX_FEW_AHEAD of them in flight, straight from memory into the operands of the 16 x 16 matrix instructions (no LDS: nothing of W is used
// twice), and add their sums up through LDS in the order of the waves.  8 tokens by two of 8 experts, 2048 -> 4096 in bf16: 27 us, 4.9 TB/s of weights.
#define EX_FEW_N 32
#define EX_FEW_AHEAD 4
template <typename T>
__device__ __forceinline__ f32x4 ex_mfma16(const ExFrag& a, const ExFrag& b, f32x4 c) {
    if constexpr (std::is_same<T, E4m3>::value) {   // deep sums
#pragma unroll
        for (int i = 0; i < 4; ++i)
            c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, ex_widen(a.p[i >> 1], i & 1)), __builtin_bit_cast(bf16x8, ex_widen(b.p[i >> 1], i & 1)), c, 0, 0, 0);
        return c;
    } else {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t x = a.p[q][e], y = b.p[q][e];
                    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(x), __uint_as_float(y), c, 0, 0, 0);
                }
            } else c = mfma16x16x32_h16(a.p[q], b.p[q], c);
        }
        return c;
    }
}

template <typename T, typename TO>
__global__ __launch_bounds__(256) void expert_few_rows_kernel(ExArgs a) {
    constexpr int ES = ExElem<T>::ES, NB = EX_FEW_N / 16;
    __shared__ float part[4][16][EX_FEW_N + 1];   // [wave][row][channel]
    ExTile t;
    if (!ex_find<16, EX_FEW_N>(a, t)) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), r = lane & 15, piece = (lane >> 4) * 16;
    // rows and channels behind the last one repeat it: their results are not stored
    const char* xp = a.m + (int64_t)min(t.m0 + r, t.mend - 1) * a.m_ld;
    const char* wp[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) wp[i] = a.n + t.e * a.n_expert + (int64_t)min(t.n0 + i * 16 + r, a.N - 1) * a.n_ld;
    // the epilogue's two channels of a row a thread; what it needs is fetched here
    const int row = min(t.m0 + ((int)threadIdx.x >> 4), t.mend - 1), c = t.n0 + ((int)threadIdx.x & 15) * 2, ca = min(c, a.N - 2);   // N is even
    const float ms = a.m_scale ? a.m_scale[row] : 1.f;
    float scale[2], bias[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        scale[e] = a.n_scale ? a.n_scale[(int64_t)t.e * a.N + ca + e] : 1.f;
        bias[e] = a.bias ? a.bias[(int64_t)t.e * a.N + ca + e] : 0.f;
    }
    const int bytes = a.K * ES, full = bytes >> 7;   // whole pieces of K; the rest is less than one
    f32x4 acc[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto load = [&](const char* p, int at) {
        ExFrag f;
        f.p[0] = *reinterpret_cast<const u32x4*>(p + at + piece);
        f.p[1] = *reinterpret_cast<const u32x4*>(p + at + 64 + piece);
        return f;
    };
    constexpr bool FOLD = std::is_same<T, float>::value;   // as in ex_body, every 128 of K (32 additions of four products)
    f32x4 far[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) far[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    int k = wave;
    for (; k + 4 * (EX_FEW_AHEAD - 1) < full; k += 4 * EX_FEW_AHEAD) {
        ExFrag x[EX_FEW_AHEAD], w[EX_FEW_AHEAD][NB];
#pragma unroll
        for (int u = 0; u < EX_FEW_AHEAD; ++u) {
            x[u] = load(xp, (k + 4 * u) * 128);
#pragma unroll
            for (int i = 0; i < NB; ++i) w[u][i] = load(wp[i], (k + 4 * u) * 128);
        }
        EX_SCHED_FENCE();   // all of them are on their way before the first is waited for
#pragma unroll
        for (int u = 0; u < EX_FEW_AHEAD; ++u)
#pragma unroll
            for (int i = 0; i < NB; ++i) acc[i] = ex_mfma16<T>(w[u][i], x[u], acc[i]);
        if constexpr (FOLD) {
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                far[i] += acc[i];
                acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
        }
    }
    for (; k < full; k += 4) {
        const ExFrag x = load(xp, k * 128);
#pragma unroll
        for (int i = 0; i < NB; ++i) acc[i] = ex_mfma16<T>(load(wp[i], k * 128), x, acc[i]);
    }
    if (k == full && (bytes & 127)) {   // the last piece: 16-byte parts behind K are zeros on both sides
        auto tail = [&](const char* p) {
            ExFrag f;
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int at = full * 128 + q * 64 + piece;
                const u32x4 v = *reinterpret_cast<const u32x4*>(p + (at < bytes ? at : 0));
                f.p[q] = at < bytes ? v : u32x4{0, 0, 0, 0};
            }
            return f;
        };
        const ExFrag x = tail(xp);
#pragma unroll
        for (int i = 0; i < NB; ++i) acc[i] = ex_mfma16<T>(tail(wp[i]), x, acc[i]);
    }
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) part[wave][r][i * 16 + (lane >> 4) * 4 + q] = FOLD ? far[i][q] + acc[i][q] : acc[i][q];
    __syncthreads();
    if (t.m0 + ((int)threadIdx.x >> 4) >= t.mend || c >= a.N) return;
    float v[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const float(*p)[16][EX_FEW_N + 1] = part;
        const int q = threadIdx.x >> 4, k = c - t.n0 + e;
        v[e] = (p[0][q][k] + p[1][q][k]) + (p[2][q][k] + p[3][q][k]);
        v[e] = std::is_same<T, E4m3>::value ? fmaf(v[e] * ms, scale[e], bias[e]) : v[e] + bias[e];   // the scales' product may be subnormal
        if (a.act == YMK_ACT_SILU) v[e] = ex_act<YMK_ACT_SILU, sizeof(TO) == 2>(v[e]);
        else if (a.act == YMK_ACT_GELU) v[e] = ex_act<YMK_ACT_GELU, sizeof(TO) == 2>(v[e]);
        else if (a.act == YMK_ACT_SIGMOID) v[e] = ex_act<YMK_ACT_SIGMOID, sizeof(TO) == 2>(v[e]);
    }
    TO* out = reinterpret_cast<TO*>(a.out) + (int64_t)row * a.out_ld + c;
    if constexpr (sizeof(TO) == 4) *reinterpret_cast<f32x2*>(out) = f32x2{v[0], v[1]};
    else *reinterpret_cast<uint32_t*>(out) = pack_h16x2(v[0], v[1]);
}

// dW (and, by the workgroups of the first channels, db)
template <typename T, typename TO, int TILE>
__global__ __launch_bounds__(256, TILE == 256 ? 1 : TILE == 128 ? 2 : 4) void expert_dw_kernel(ExArgs a) {
    // Experts differ in rows, so each expert's tiles are split over all XCDs: eight runs of neighbouring tiles, one an XCD (32768 rows over 8 experts
    // drawn with a spread of 0.3, 1024 by 4096: an expert an XCD took 324 us, this 278 us); fewer than eight tiles go round in turn.
    const int nt = (a.N + TILE - 1) / TILE, mt = (a.M + TILE - 1) / TILE, all = nt * mt, run = (all + 7) / 8;
    const int slot = all < 8 ? blockIdx.x : blockIdx.x >> 3;
    ExTile t;
    t.e = slot / (all < 8 ? all : run);
    const int id = all < 8 ? slot % all : (blockIdx.x & 7) * run + slot % run;
    if (t.e >= a.E || id >= all) return;
    t.m0 = id / nt * TILE;
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
    if (blocks > 0x7ffffff0) return YMK_E_BADARG;
    static YmkOncePerDevice once;
    if (once.need()) {
        if (hipFuncSetAttribute(reinterpret_cast<const void*>(Kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess) return YMK_E_LAUNCH;
        once.done();
    }
    hipLaunchKernelGGL(Kernel, dim3((unsigned)blocks), dim3(256), lds, (hipStream_t)stream, a);
    return ymk_launch_status();
}

// workgroups that hold every tile of rows whatever the offsets say, in whole rounds of the 8 XCDs
inline int64_t ex_blocks(int64_t rows, int E, int N, int tm, int tn) {
    const int64_t mt = rows / tm + (rows < E ? rows : E), nt = (N + tn - 1) / tn;
    return (mt * nt + 7) / 8 * 8;
}

// Wider tiles bring fewer bytes to LDS for a product, but leave CUs idle when there are few of them and waste rows when experts have few.  Both sides, us a
// call, the weights from memory (600 MB of them in turn):
//     rows an expert   shape (16-bit unless said)              16     64    128    256
//     1                6 rows of 64 experts, 4096 -> 2048 e4m3 16.0   21.5   22.3   39.4
//     2                16 of 8, 2048 -> 4096                   29.7   34.7   34.8   43.3
//     16               128 of 8, 2048 -> 4096                  31.3   35.0   35.0   43.1
//     16               128 of 8, 2048 -> 4096 e4m3             17.8   17.5   15.7   24.0
//     64               512 of 8, 2048 -> 4096                  91.7   35.3   37.0   45.5
//     64               512 of 8, 2048 -> 4096 e4m3             52.7   19.3   17.7   26.3
//     64               1024 of 16, 1024 -> 2048                52.7   16.9   17.2   26.0
//     200              3202 of 16, 256 -> 520 fp32             27.9   18.4   22.9   69.2
//     256              4096 of 16, 512 -> 2048                113.7   25.2   20.4   23.0
//     4096             32768 of 8, 4096 -> 4096                              1099    886
// The rule knows the average only: an expert that got most of the rows of a small call walks its matrix once per 16 of them.
inline int ex_tile(int64_t rows, int E, int N) {
    auto tiles = [&](int tile) { return (rows / tile + E / 2) * ((N + tile - 1) / tile); };
    if (rows <= 16 || rows <= 4ll * E) return 16;
    if (rows >= 192ll * E && tiles(256) >= 256) return 256;
    if (rows >= 32ll * E && tiles(128) >= 256) return 128;
    return 64;
}

// A/B and test switch, read at first use: YMK_EXPERT_TILE=16|64|128|256 takes that tile for every size (16: y only, the others then take 64; 256: 8-bit
// rows with an fp32 output and an fp32 dW take 128)
inline int ex_forced() {
    static const int tile = [] {
        const char* s = getenv("YMK_EXPERT_TILE");
        const int v = s ? atoi(s) : 0;
        return v == 16 || v == 64 || v == 128 || v == 256 ? v : 0;
    }();
    return tile;
}
template <typename T, typename TO, bool NKC, int TILE>
int ex_rows_tile(const ExArgs& a, void* stream) {
    return ex_launch<expert_rows_kernel<T, TO, NKC, TILE>>(a, ex_blocks(a.rows, a.E, a.N, TILE, TILE), EX_UNITS * TILE * 128, stream);
}
template <typename T, typename TO, bool NKC>
int ex_rows(const ExArgs& a, void* stream) {
    const int tile = ex_forced() ? ex_forced() : ex_tile(a.rows, a.E, a.N);
    constexpr bool WIDE = !(std::is_same<T, E4m3>::value && sizeof(TO) == 4);   // the widened operands of 256 x 256 do not fit the registers
    if constexpr (NKC) {
        if (tile == 16) {
            const int64_t blocks = ex_blocks(a.rows, a.E, a.N, 16, EX_FEW_N);
            if (blocks > 0x7ffffff0) return YMK_E_BADARG;
            hipLaunchKernelGGL((expert_few_rows_kernel<T, TO>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, a);
            return ymk_launch_status();
        }
    }
    if constexpr (WIDE) {
        if (tile == 256) return ex_rows_tile<T, TO, NKC, 256>(a, stream);
    }
    if (tile >= 128) return ex_rows_tile<T, TO, NKC, 128>(a, stream);
    return ex_rows_tile<T, TO, NKC, 64>(a, stream);
}
inline int64_t ex_dw_blocks(const ExArgs& a, int tile) {
    const int64_t all = (int64_t)((a.N + tile - 1) / tile) * ((a.M + tile - 1) / tile);
    return all < 8 ? all * a.E : (all + 7) / 8 * 8 * a.E;
}
template <typename T, typename TO>
int ex_dw(const ExArgs& a, void* stream) {
    // us at 64 / 128 / 256: 200 rows an expert, 16 of 520 x 256 fp32 18.3 / 25.5 / 65; 64 rows, 16 of 2048 x 1024 29.9 / 23.4 / 25.9; 256 rows, 16 of
    // 2048 x 512 25.1 / 21.5 / 21.3; 4096 rows, 8 of 4096 x 4096 - / 1250 / 974.  K is not split: the workgroups are tiles times experts however many
    // rows there are, so many rows over few small matrices leave CUs idle.
    const int tile = ex_forced() ? ex_forced() : a.rows >= 1024ll * a.E && ex_dw_blocks(a, 256) >= 512 ? 256 : ex_dw_blocks(a, 128) >= 512 ? 128 : 64;
    // Two sets of fp32 accumulators of 256 x 256 do not fit the registers; 128 is as fast there: 4096 rows, 8 of 4096 x 1024 2049 / 2056 us at 256 / 128 before
    if constexpr (!std::is_same<T, float>::value) {
        if (tile == 256) return ex_launch<expert_dw_kernel<T, TO, 256>>(a, ex_dw_blocks(a, 256), EX_UNITS * 256 * 128, stream);
    }
    if (tile >= 128) return ex_launch<expert_dw_kernel<T, TO, 128>>(a, ex_dw_blocks(a, 128), EX_UNITS * 128 * 128, stream);
    return ex_launch<expert_dw_kernel<T, TO, 64>>(a, ex_dw_blocks(a, 64), EX_UNITS * 64 * 128, stream);
}

inline bool ex_bad16(const void* p) { return !p || (reinterpret_cast<uintptr_t>(p) & 15); }
inline bool ex_bad_ld(int64_t ld, int64_t C, int es) { return ld < C || ld * es % 16 || ld * es >= (1 << 23); }
inline bool ex_bad_sizes(int64_t rows, int32_t E, int32_t Cin, int32_t Cout) {
    return rows < 0 || rows >= (1ll << 26) || E < 1 || E > YMK_TOKEN_MAX_E || Cin < 1 || Cout < 1;
}

}  // namespace

extern "C" int ymk_expert_linear(int32_t dtype, int32_t out_dtype, const void* x, int32_t ldx, const float* x_scale, const void* w, const float* w_scale,
                                 const float* bias, const int32_t* offsets, void* y, int32_t ldy, int64_t rows, int32_t E, int32_t Cin, int32_t Cout,
                                 int32_t act, void* stream) {
    const bool f8 = dtype == YMK_E4M3;
    if ((dtype != YMK_F32 && dtype != YMK_H16 && !f8) || (out_dtype != dtype && !(f8 && (out_dtype == YMK_F32 || out_dtype == YMK_H16))) ||
        ex_bad_sizes(rows, E, Cin, Cout) || act < YMK_ACT_NONE || act > YMK_ACT_GELU || !offsets)
        return YMK_E_BADARG;
    const int es = f8 ? 1 : dtype == YMK_F32 ? 4 : 2, eo = out_dtype == YMK_F32 ? 4 : 2;
    if (rows == 0) return YMK_OK;
    if ((f8 && (!x_scale || !w_scale)) || (!f8 && (x_scale || w_scale))) return YMK_E_BADARG;
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
