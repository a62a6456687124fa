// TEST INFRASTRUCTURE — a host stand-in for <hip/hip_runtime.h>, just large enough to compile the config-5 kernel
// sources (csrc/mixture.hip, csrc/mixattn.hip) for the CPU and run them lane by lane: workgroups run one after another,
// the lanes of a workgroup are fibers that switch at barriers, __shfl_xor() exchanges through a per-lane buffer between
// two barriers, __shared__ storage is function-static (tests/hostemu/build.py rewrites the qualifier).  It checks the
// kernels' LOGIC (indexing, reductions, barriers, numerics) before they ever reach an MI355X; it says nothing about
// occupancy, LDS limits or speed.
#pragma once
#include <ucontext.h>

#include <cmath>
#include <cstdint>
#include <cstdlib>
#include <cstring>
#include <functional>

#define __global__ static
#define __device__
#define __host__
#define __forceinline__ inline
#define __launch_bounds__(...)
#ifndef INFINITY
#define INFINITY __builtin_inff()
#endif

struct dim3 {
    unsigned x, y, z;
    dim3(unsigned x_ = 1, unsigned y_ = 1, unsigned z_ = 1) : x(x_), y(y_), z(z_) {}
};
struct int4 { int x, y, z, w; };
typedef void* hipStream_t;
typedef int hipError_t;
enum { hipSuccess = 0 };
static inline hipError_t hipGetLastError() { return hipSuccess; }

// Lanes are FIBERS of one OS thread (ucontext): the scheduler resumes every unfinished lane of the workgroup in turn and
// a lane runs until it has to wait.  Two kinds of rendezvous, each with its own arrival counter and generation number:
// `block_sync` (__syncthreads / s_barrier: every unfinished lane of the workgroup) and `wave_sync` (the exchange points of
// __shfl_xor and of the matrix-core builtins: the 64 lanes of one wave).  Waves may therefore execute different numbers of
// wave-level exchanges between two workgroup barriers (a wave with fewer MFMA steps than its neighbours), as on the GPU.
// Kernels whose lanes skip a barrier other lanes take are not supported (and would be broken on the GPU as well).
namespace hostemu {
constexpr unsigned MAX_LANES = 1024;          // the largest workgroup any emulated kernel uses (the NMS ordering kernels)
constexpr size_t STACK = 128 * 1024;
struct Fiber {
    ucontext_t ctx;
    bool done;
};
inline Fiber fibers[MAX_LANES];
inline ucontext_t sched;
inline char* stacks = nullptr;
inline unsigned cur = 0;
inline dim3 g_threadIdx, g_blockIdx, g_blockDim, g_gridDim;
inline uint64_t xch[MAX_LANES];               // shuffle exchange, one (up to 64-bit) slot per lane
alignas(16) inline float dyn_lds[40960];     // dynamic LDS of `extern __shared__` kernels (160 KB: one CU's LDS)
inline std::function<void()> job;

inline unsigned n_alive = 0, blk_arrived = 0, blk_gen = 0;
inline unsigned wave_arrived[MAX_LANES / 64], wave_gen[MAX_LANES / 64], wave_alive[MAX_LANES / 64];
inline void yield() { swapcontext(&fibers[cur].ctx, &sched); }
inline void block_sync() {
    const unsigned g = blk_gen;
    ++blk_arrived;
    while (blk_gen == g) {
        if (blk_arrived >= n_alive) { blk_arrived = 0; ++blk_gen; break; }   // the last lane to arrive (or lanes finished meanwhile) opens it
        yield();
    }
}
inline void wave_sync() {
    const unsigned w = cur / 64, g = wave_gen[w];
    ++wave_arrived[w];
    while (wave_gen[w] == g) {
        if (wave_arrived[w] >= wave_alive[w]) { wave_arrived[w] = 0; ++wave_gen[w]; break; }   // lanes that returned do not take part
        yield();
    }
}
inline void entry() {
    job();
    fibers[cur].done = true;
    --n_alive;
    --wave_alive[cur / 64];
    swapcontext(&fibers[cur].ctx, &sched);
}
template <typename F>
void launch(F&& body, dim3 grid, dim3 block) {
    if (block.y != 1 || block.z != 1 || block.x % 64 || block.x > MAX_LANES) abort();   // 1-D workgroups of whole waves
    if (!stacks) stacks = static_cast<char*>(malloc(MAX_LANES * STACK));
    g_blockDim = block;
    g_gridDim = grid;
    job = body;
    for (unsigned bz = 0; bz < grid.z; ++bz)
        for (unsigned by = 0; by < grid.y; ++by)
            for (unsigned bx = 0; bx < grid.x; ++bx) {
                g_blockIdx = dim3(bx, by, bz);
                for (unsigned t = 0; t < block.x; ++t) {
                    getcontext(&fibers[t].ctx);
                    fibers[t].ctx.uc_stack.ss_sp = stacks + (size_t)t * STACK;
                    fibers[t].ctx.uc_stack.ss_size = STACK;
                    fibers[t].ctx.uc_link = nullptr;
                    fibers[t].done = false;
                    makecontext(&fibers[t].ctx, entry, 0);
                }
                n_alive = block.x;
                blk_arrived = 0;
                for (unsigned w = 0; w < MAX_LANES / 64; ++w) { wave_arrived[w] = 0; wave_alive[w] = 64; }
                for (unsigned alive = block.x; alive;) {   // one pass = one phase between barriers
                    alive = 0;
                    for (unsigned t = 0; t < block.x; ++t) {
                        if (fibers[t].done) continue;
                        cur = t;
                        g_threadIdx = dim3(t, 0, 0);
                        swapcontext(&sched, &fibers[t].ctx);
                        alive += !fibers[t].done;
                    }
                }
            }
}
}  // namespace hostemu
#define threadIdx hostemu::g_threadIdx
#define blockIdx hostemu::g_blockIdx
#define blockDim hostemu::g_blockDim
#define gridDim hostemu::g_gridDim

static inline void __syncthreads() { hostemu::block_sync(); }
// Wave-level exchanges: every lane publishes its 32-bit value, the wave meets, every lane reads the lane it asked for, the
// wave meets again (so the slot can be reused).  A source lane that has already returned reads as the asking lane's own value.
namespace hostemu {
template <typename T, typename F>
inline T exchange(T v, F&& src_lane) {
    static_assert(sizeof(T) <= 8, "32- and 64-bit exchanges");
    const unsigned t = cur;
    std::memcpy(&xch[t], &v, sizeof(T));
    wave_sync();
    const unsigned s = (t & ~63u) | ((unsigned)src_lane(t & 63u) & 63u);
    T r = v;
    if (!fibers[s].done) std::memcpy(&r, &xch[s], sizeof(T));
    wave_sync();
    return r;
}
}  // namespace hostemu
template <typename T> static inline T __shfl_xor(T v, int mask, int = 64) { return hostemu::exchange(v, [&](unsigned l) { return l ^ (unsigned)mask; }); }
template <typename T> static inline T __shfl_up(T v, unsigned delta, int = 64) { return hostemu::exchange(v, [&](unsigned l) { return l >= delta ? l - delta : l; }); }
template <typename T> static inline T __shfl_down(T v, unsigned delta, int = 64) { return hostemu::exchange(v, [&](unsigned l) { return l + delta < 64 ? l + delta : l; }); }
template <typename T> static inline T __shfl(T v, int lane, int = 64) { return hostemu::exchange(v, [&](unsigned) { return (unsigned)lane; }); }
static inline int __builtin_amdgcn_readlane(int v, int lane) { return __shfl(v, lane); }
static inline int __builtin_amdgcn_readfirstlane(int v) {   // the lowest lane of the wave that is still running
    const unsigned w0 = hostemu::cur & ~63u;
    return hostemu::exchange(v, [&](unsigned) { unsigned l = 0; while (l < 63 && hostemu::fibers[w0 + l].done) ++l; return l; });
}
static inline unsigned long long __ballot(int pred) {
    unsigned long long m = 0;
    for (unsigned l = 0; l < 64; ++l) {   // 64 rounds of a one-bit exchange (test infrastructure: clarity over speed)
        const int b = hostemu::exchange(pred ? 1 : 0, [&](unsigned) { return l; });
        const bool alive = !hostemu::fibers[(hostemu::cur & ~63u) + l].done;
        if (alive && b) m |= 1ull << l;
    }
    return m;
}
static inline int __popcll(unsigned long long v) { return __builtin_popcountll(v); }
static inline int __popc(unsigned v) { return __builtin_popcount(v); }
static inline void __threadfence_block() {}
static inline void __builtin_amdgcn_wave_barrier() { hostemu::wave_sync(); }
// v_permlane16_swap / v_permlane32_swap (gfx950): rows of 16 lanes; swap odd rows of the first operand with even rows of the second /
// the upper half of the first with the lower half of the second.  Returns {new first, new second}.
typedef unsigned hostemu_u32x2 __attribute__((ext_vector_type(2)));
static inline hostemu_u32x2 __builtin_amdgcn_permlane16_swap(unsigned a, unsigned b, bool, bool) {
    const unsigned row = (hostemu::cur & 63u) >> 4;
    const unsigned pa = hostemu::exchange(a, [&](unsigned l) { return l ^ 16u; });   // partner row's first operand
    const unsigned pb = hostemu::exchange(b, [&](unsigned l) { return l ^ 16u; });
    hostemu_u32x2 r;
    r.x = (row & 1u) ? pb : a;     // odd rows of a receive the even row below them of b
    r.y = (row & 1u) ? b : pa;     // even rows of b receive the odd row above them of a
    return r;
}
static inline hostemu_u32x2 __builtin_amdgcn_permlane32_swap(unsigned a, unsigned b, bool, bool) {
    const unsigned hi = (hostemu::cur & 63u) >> 5;
    const unsigned pa = hostemu::exchange(a, [&](unsigned l) { return l ^ 32u; });
    const unsigned pb = hostemu::exchange(b, [&](unsigned l) { return l ^ 32u; });
    hostemu_u32x2 r;
    r.x = hi ? pb : a;
    r.y = hi ? b : pa;
    return r;
}
static inline int atomicOr(int* p, int v) { const int o = *p; *p = o | v; return o; }
static inline unsigned long long atomicOr(unsigned long long* p, unsigned long long v) { const unsigned long long o = *p; *p = o | v; return o; }
static inline int atomicMin(int* p, int v) { const int o = *p; if (v < o) *p = v; return o; }
static inline float __uint_as_float(uint32_t u) { float f; std::memcpy(&f, &u, 4); return f; }
static inline uint32_t __float_as_uint(float f) { uint32_t u; std::memcpy(&u, &f, 4); return u; }
static inline int __float_as_int(float f) { int u; std::memcpy(&u, &f, 4); return u; }
static inline float __int_as_float(int u) { float f; std::memcpy(&f, &u, 4); return f; }
static inline int atomicAdd(int* p, int v) { const int o = *p; *p = o + v; return o; }
static inline unsigned atomicAdd(unsigned* p, unsigned v) { const unsigned o = *p; *p = o + v; return o; }
static inline float atomicAdd(float* p, float v) { const float o = *p; *p = o + v; return o; }
static inline double atomicAdd(double* p, double v) { const double o = *p; *p = o + v; return o; }
static inline unsigned atomicMax(unsigned* p, unsigned v) { const unsigned o = *p; if (v > o) *p = v; return o; }
#define __builtin_amdgcn_exp2f(x) exp2f(x)
#define __expf(x) expf(x)   // glibc declares __expf itself
#define __builtin_amdgcn_rcpf(x) (1.0f / (x))
using std::isfinite;
using std::max;
using std::min;

#define hipLaunchKernelGGL(kernel, grid, block, shmem, stream, ...) \
    hostemu::launch([&] { kernel(__VA_ARGS__); }, grid, block)

// ---- what the tiled-GEMM design probes (tools/micro/conv256.hip) need on top -----------------------------------------
// Matrix core: v_mfma_f32_16x16x32_bf16.  Lane l of the wave holds A[l % 16][(l / 16) * 8 .. + 7], B[(l / 16) * 8 .. + 7][l % 16]
// and D[(l / 16) * 4 + r][l % 16], r = 0..3 (CDNA3/4 ISA; the layout the library's kernels were validated with on hardware).
typedef __bf16 hostemu_bf16x8 __attribute__((ext_vector_type(8)));
typedef float hostemu_f32x4 __attribute__((ext_vector_type(4)));
namespace hostemu {
inline float mfma_a[MAX_LANES][8], mfma_b[MAX_LANES][8];
}
static inline hostemu_f32x4 __builtin_amdgcn_mfma_f32_16x16x32_bf16(hostemu_bf16x8 a, hostemu_bf16x8 b, hostemu_f32x4 c, int, int, int) {
    const unsigned t = hostemu::cur, w0 = t & ~63u, l = t & 63u;
    for (int e = 0; e < 8; ++e) {
        hostemu::mfma_a[t][e] = (float)a[e];
        hostemu::mfma_b[t][e] = (float)b[e];
    }
    hostemu::wave_sync();
    for (int r = 0; r < 4; ++r) {
        const unsigned i = (l / 16) * 4 + r, j = l % 16;
        float s = 0.f;
        for (unsigned k = 0; k < 32; ++k) s += hostemu::mfma_a[w0 + (k / 8) * 16 + i][k % 8] * hostemu::mfma_b[w0 + (k / 8) * 16 + j][k % 8];
        c[r] += s;
    }
    hostemu::wave_sync();
    return c;
}
// v_mfma_f32_16x16x32_f16: the same operand layout with IEEE binary16 elements (the fp16 build, -DYMK_H16_F16)
typedef _Float16 hostemu_f16x8 __attribute__((ext_vector_type(8)));
static inline hostemu_f32x4 __builtin_amdgcn_mfma_f32_16x16x32_f16(hostemu_f16x8 a, hostemu_f16x8 b, hostemu_f32x4 c, int, int, int) {
    const unsigned t = hostemu::cur, w0 = t & ~63u, l = t & 63u;
    for (int e = 0; e < 8; ++e) {
        hostemu::mfma_a[t][e] = (float)a[e];
        hostemu::mfma_b[t][e] = (float)b[e];
    }
    hostemu::wave_sync();
    for (int r = 0; r < 4; ++r) {
        const unsigned i = (l / 16) * 4 + r, j = l % 16;
        float s = 0.f;
        for (unsigned k = 0; k < 32; ++k) s += hostemu::mfma_a[w0 + (k / 8) * 16 + i][k % 8] * hostemu::mfma_b[w0 + (k / 8) * 16 + j][k % 8];
        c[r] += s;
    }
    hostemu::wave_sync();
    return c;
}
// v_mfma_f32_16x16x4_f32: lane l holds A[l % 16][l / 16], B[l / 16][l % 16]; D as above.
static inline hostemu_f32x4 __builtin_amdgcn_mfma_f32_16x16x4f32(float a, float b, hostemu_f32x4 c, int, int, int) {
    const unsigned t = hostemu::cur, w0 = t & ~63u, l = t & 63u;
    hostemu::mfma_a[t][0] = a;
    hostemu::mfma_b[t][0] = b;
    hostemu::wave_sync();
    for (int r = 0; r < 4; ++r) {
        const unsigned i = (l / 16) * 4 + r, j = l % 16;
        float s = 0.f;
        for (unsigned k = 0; k < 4; ++k) s += hostemu::mfma_a[w0 + k * 16 + i][0] * hostemu::mfma_b[w0 + k * 16 + j][0];
        c[r] += s;
    }
    hostemu::wave_sync();
    return c;
}
// The 32x32 forms: lane l holds row l % 32 of its operand, elements (l / 32) * n .. + n - 1 of K (n elements a lane); D[(r / 4) * 8 + (l / 32) * 4 + r % 4][l % 32],
// r = 0..15 (CDNA3/4 ISA; for the 64-deep 8-bit form the order of K is the operands' own, the same for both).
typedef float hostemu_f32x16 __attribute__((ext_vector_type(16)));
typedef int hostemu_i32x8 __attribute__((ext_vector_type(8)));
namespace hostemu {
inline float mfma_wide_a[MAX_LANES][32], mfma_wide_b[MAX_LANES][32];
inline hostemu_f32x16 mfma32(int n, hostemu_f32x16 c) {   // operands published by the caller
    const unsigned w0 = cur & ~63u, l = cur & 63u;
    wave_sync();
    for (int r = 0; r < 16; ++r) {
        const unsigned i = (r / 4) * 8 + (l / 32) * 4 + r % 4, j = l % 32;
        float s = 0.f;
        for (unsigned h = 0; h < 2; ++h)
            for (int e = 0; e < n; ++e) s += mfma_wide_a[w0 + h * 32 + i][e] * mfma_wide_b[w0 + h * 32 + j][e];
        c[r] += s;
    }
    wave_sync();
    return c;
}
// OCP e4m3: bias 7, subnormals at 2^-9, 0x7f / 0xff NaN, no infinities
inline float from_e4m3(unsigned v) {
    const int e = (v >> 3) & 15, m = v & 7;
    if (e == 15 && m == 7) return __builtin_nanf("");
    const float a = e ? std::ldexp((float)(8 + m), e - 10) : std::ldexp((float)m, -9);
    return v & 0x80 ? -a : a;
}
inline unsigned to_e4m3(float f) {   // round to nearest even; beyond 464 NaN, as the hardware's conversion without clamping gives
    const unsigned s = std::signbit(f) ? 0x80u : 0u;
    const float a = std::fabs(f);
    if (!(a <= 464.f)) return s | 0x7fu;
    if (a >= 448.f) return s | 0x7eu;
    int e;
    std::frexp(a, &e);
    const int q = a < std::ldexp(1.f, -6) ? -9 : e - 4;   // exponent of one step
    const float n = std::nearbyint(std::ldexp(a, -q));    // 0..16 steps
    if (a < std::ldexp(1.f, -6)) return s | (unsigned)n;  // 8 steps are the smallest normal number
    unsigned m = (unsigned)n, ex = (unsigned)(q + 10);
    if (m == 16) { m = 8; ++ex; }
    return s | (ex << 3) | (m - 8);
}
}  // namespace hostemu
static inline hostemu_f32x16 __builtin_amdgcn_mfma_f32_32x32x16_bf16(hostemu_bf16x8 a, hostemu_bf16x8 b, hostemu_f32x16 c, int, int, int) {
    for (int e = 0; e < 8; ++e) { hostemu::mfma_wide_a[hostemu::cur][e] = (float)a[e]; hostemu::mfma_wide_b[hostemu::cur][e] = (float)b[e]; }
    return hostemu::mfma32(8, c);
}
static inline hostemu_f32x16 __builtin_amdgcn_mfma_f32_32x32x16_f16(hostemu_f16x8 a, hostemu_f16x8 b, hostemu_f32x16 c, int, int, int) {
    for (int e = 0; e < 8; ++e) { hostemu::mfma_wide_a[hostemu::cur][e] = (float)a[e]; hostemu::mfma_wide_b[hostemu::cur][e] = (float)b[e]; }
    return hostemu::mfma32(8, c);
}
static inline hostemu_f32x16 __builtin_amdgcn_mfma_f32_32x32x2f32(float a, float b, hostemu_f32x16 c, int, int, int) {
    hostemu::mfma_wide_a[hostemu::cur][0] = a;
    hostemu::mfma_wide_b[hostemu::cur][0] = b;
    return hostemu::mfma32(1, c);
}
static inline hostemu_f32x16 __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(hostemu_i32x8 a, hostemu_i32x8 b, hostemu_f32x16 c, int fmt_a, int fmt_b, int, int, int, int) {
    if (fmt_a || fmt_b) abort();   // e4m3 only
    for (int e = 0; e < 32; ++e) {
        hostemu::mfma_wide_a[hostemu::cur][e] = hostemu::from_e4m3(((unsigned)a[e / 4] >> (e % 4 * 8)) & 255u);
        hostemu::mfma_wide_b[hostemu::cur][e] = hostemu::from_e4m3(((unsigned)b[e / 4] >> (e % 4 * 8)) & 255u);
    }
    return hostemu::mfma32(32, c);
}
static inline hostemu_f32x4 __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(hostemu_i32x8 a, hostemu_i32x8 b, hostemu_f32x4 c, int fmt_a, int fmt_b, int, int, int, int) {
    if (fmt_a || fmt_b) abort();   // e4m3 only
    const unsigned t = hostemu::cur, w0 = t & ~63u, l = t & 63u;
    for (int e = 0; e < 32; ++e) {
        hostemu::mfma_wide_a[t][e] = hostemu::from_e4m3(((unsigned)a[e / 4] >> (e % 4 * 8)) & 255u);
        hostemu::mfma_wide_b[t][e] = hostemu::from_e4m3(((unsigned)b[e / 4] >> (e % 4 * 8)) & 255u);
    }
    hostemu::wave_sync();
    for (int r = 0; r < 4; ++r) {
        const unsigned i = (l / 16) * 4 + r, j = l % 16;
        float s = 0.f;
        for (unsigned h = 0; h < 4; ++h)
            for (int e = 0; e < 32; ++e) s += hostemu::mfma_wide_a[w0 + h * 16 + i][e] * hostemu::mfma_wide_b[w0 + h * 16 + j][e];
        c[r] += s;
    }
    hostemu::wave_sync();
    return c;
}
static inline int __builtin_amdgcn_cvt_pk_fp8_f32(float x, float y, int old, bool high) {
    const unsigned v = hostemu::to_e4m3(x) | (hostemu::to_e4m3(y) << 8);
    return (int)(high ? ((unsigned)old & 0xffffu) | (v << 16) : ((unsigned)old & 0xffff0000u) | v);
}
// two e4m3 codes of a word (its lower or upper half) times scale in bfloat16
typedef __bf16 hostemu_bf16x2 __attribute__((ext_vector_type(2)));
static inline hostemu_bf16x2 __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(unsigned codes, float scale, bool high) {
    const unsigned v = high ? codes >> 16 : codes;
    return hostemu_bf16x2{(__bf16)(hostemu::from_e4m3(v & 255u) * scale), (__bf16)(hostemu::from_e4m3((v >> 8) & 255u) * scale)};
}
// ds_read_b64_tr_b16: the 16 lanes of a group read four rows of 16 16-bit elements, lane i the elements 4 (i % 4) .. + 3 of row i / 4 at its own
// address, and lane i receives column i of them
static inline hostemu_u32x2 hostemu_ds_read_tr16_b64(const char* p) {
    uint64_t mine;
    std::memcpy(&mine, p, 8);
    const unsigned i = hostemu::cur & 15u;
    uint64_t out = 0;
    for (unsigned r = 0; r < 4; ++r) {
        const uint64_t v = hostemu::exchange(mine, [&](unsigned l) { return (l & ~15u) + r * 4 + i / 4; });
        out |= ((v >> (i % 4 * 16)) & 0xffffull) << (r * 16);
    }
    hostemu_u32x2 r;
    r.x = (unsigned)out;
    r.y = (unsigned)(out >> 32);
    return r;
}
static inline int __ffsll(unsigned long long v) { return __builtin_ffsll((long long)v); }
// LDS-DMA: 16 bytes per lane from the lane's global address to (wave-uniform LDS base) + lane * 16.  Completes at once
// here, so counted-vmcnt mistakes are invisible; addressing, swizzles and masks are not.
static inline void hostemu_global_load_lds16(const void* g, void* lds_base) {
    std::memcpy(static_cast<char*>(lds_base) + (hostemu::cur & 63u) * 16, g, 16);
}
#define __builtin_amdgcn_global_load_lds(g, l, size, off, aux) hostemu_global_load_lds16((const void*)(g), (void*)(l))
#define __builtin_amdgcn_s_waitcnt(x) ((void)0)
static inline void __builtin_amdgcn_s_barrier() { hostemu::block_sync(); }
// raw buffer resource (stride 0) and `buffer_load_dwordx4 ... offen lds`: 16 bytes per lane from base + voffset + soffset to (wave-uniform
// LDS base) + lane * 16; a lane whose voffset + 16 exceeds num_records - soffset reads zeros (the hardware's range check of raw
// buffers compares the VGPR offset alone against num_records - SGPR offset: an offset with bit 31 set is always out of range)
struct hostemu_rsrc { const char* base; unsigned num_records; };
static inline hostemu_rsrc hostemu_make_rsrc(const void* p, unsigned n) { return hostemu_rsrc{static_cast<const char*>(p), n}; }
static inline void hostemu_buffer_load_lds16(hostemu_rsrc r, void* lds_base, unsigned voff, unsigned soff) {
    char* d = static_cast<char*>(lds_base) + (hostemu::cur & 63u) * 16;
    const unsigned lim = r.num_records >= soff ? r.num_records - soff : 0u;
    if ((unsigned long long)voff + 16ull > (unsigned long long)lim) std::memset(d, 0, 16);
    else std::memcpy(d, r.base + voff + soff, 16);
}

// the slice of the HIP runtime API the probes' main() uses
enum hipMemcpyKind { hipMemcpyHostToDevice, hipMemcpyDeviceToHost };
enum hipFuncAttribute { hipFuncAttributeMaxDynamicSharedMemorySize };
typedef int hipEvent_t;
template <typename T> static inline hipError_t hipMalloc(T** p, size_t n) { *p = static_cast<T*>(malloc(n)); return hipSuccess; }
static inline hipError_t hipFree(void* p) { free(p); return hipSuccess; }
static inline hipError_t hipMemcpy(void* d, const void* s, size_t n, hipMemcpyKind) { std::memcpy(d, s, n); return hipSuccess; }
static inline hipError_t hipMemset(void* d, int v, size_t n) { std::memset(d, v, n); return hipSuccess; }
static inline hipError_t hipDeviceSynchronize() { return hipSuccess; }
static inline hipError_t hipFuncSetAttribute(const void*, hipFuncAttribute, int) { return hipSuccess; }
static inline hipError_t hipGetDevice(int* d) { *d = 0; return hipSuccess; }
enum hipDeviceAttribute_t { hipDeviceAttributeMultiprocessorCount = 63 };
static inline hipError_t hipDeviceGetAttribute(int* v, hipDeviceAttribute_t, int) { *v = 256; return hipSuccess; }
template <typename K> static inline hipError_t hipOccupancyMaxActiveBlocksPerMultiprocessor(int* n, K, int, size_t) { *n = 1; return hipSuccess; }
static inline const char* hipGetErrorString(hipError_t) { return "host emulation"; }
static inline hipError_t hipEventCreate(hipEvent_t*) { return hipSuccess; }
static inline hipError_t hipEventDestroy(hipEvent_t) { return hipSuccess; }
static inline hipError_t hipEventRecord(hipEvent_t) { return hipSuccess; }
static inline hipError_t hipEventSynchronize(hipEvent_t) { return hipSuccess; }
static inline hipError_t hipEventElapsedTime(float* ms, hipEvent_t, hipEvent_t) { *ms = 1.0f; return hipSuccess; }
