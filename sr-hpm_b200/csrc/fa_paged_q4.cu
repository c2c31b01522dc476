// Attention of a batch's new tokens over a paged cache of q4_0 rows (srhpm_flash_attn_paged), on the 5th-generation tensor
// cores, with the cached tokens along the products' long side:
//   S^T = K Q^T        M = 128 tokens, N rows; K as f16 in tensor memory (a lane per token), Q in shared memory
//   softmax            a thread has one token's scores; a row's maximum is raised only when a score exceeds it by 2^8, which all
//                      threads of the row learn through one barrier with a vote; p = 2^(s - m + 7) as f16 into shared memory
//   O^T += V^T P^T     M = 128 dims, N rows, K = 128 tokens: V as it lies, a row of f16 per token
// The rows of a sequence and KV head (query heads of its group x new tokens) are the narrow side, so 4 rows of a decoding step
// cost a product of N = 16, not one of 64 or 128 rows that mostly are none, and 4-bit numbers are unpacked once for all rows of
// a tile. Unpacking goes where it costs least: K's into tensor memory, whose writes take no shared memory bandwidth, V's into
// the 128-byte swizzled rows that the product reads.
//
// Measured: 9 f32 rows over 131072 tokens, 24 / 4 heads of 256: 123 us, 54 of 64 rows used; a tile of 128 tokens takes 7300 cycles on
// its SM: the MMA warp waits for V 1400 (shared memory holds one tile of it) and issues P V for 2300, the softmax warps wait for
// that 1900 and spend 1800 on O's way out and the rest. Tiles of 96 rows, 2048 rows over 32768 tokens: 6500 cycles, unpacking 2700 of
// them, raw rows late by 1300 to 1900 (2.69 ms; with 128 rows a tile 2.75, with 8 softmax warps besides 2.96).
//
// Work: as in fa_paged.cu, all items' units of 128 tokens stand in one line that is cut into equal parts, one per CTA.
// Roles: 16 softmax warps (four groups, a quarter of the rows each: with half of them a thread's scores and sums did not fit its
// registers, and the chain from scores to P took 6000 cycles of a tile), 1 MMA warp, 2 producer warps (K's and V's raw rows by TMA, 64
// tokens at a time, row boxes of 16-byte multiples; layouts that TMA does not take come by cp.async, 9 pieces a row), and 8 warps
// that unpack, K's and V's, 32 tokens of a tile each.
// f32 rows (PREC): Q and P as sums of two f16 parts, and as the tensor cores' sums are truncated (a shrink of 2^-25 per product
// step, measured: 2e-5 after 400), O is taken out every kFlush tiles and summed up in f32 in the item's record.
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "fa_paged.cuh"
#include "fastdiv.cuh"
#include "internal.h"
#include "launch.cuh"
#include "ptx.cuh"
#include "q4.cuh"
#include "tc.cuh"

namespace srhpm {
using namespace fap;
using namespace q4;
namespace {

constexpr int      kTile   = 128;  // tokens of a tile and of a unit of work
constexpr int      kSm     = 16;   // softmax warps, in groups of four
constexpr int      kConv   = 8;    // unpacking warps: K's four, V's four
constexpr int      kThr    = (kSm + 4 + kConv) * 32;
constexpr int      kRawTok = 64;   // tokens of a raw stage
constexpr int      kFlush  = 8;    // tiles
constexpr float    kUnset  = -3e38f;    // a row's reference before its first score

template <int D, int N, bool PREC> struct LayT {
    static constexpr int parts = PREC ? 2 : 1;
    static constexpr int MT    = D == 256 ? 2 : 1;             // products along the dims
    static constexpr int MM    = D == 64 ? 64 : 128;           // dims of a product
    static constexpr int NP    = N < 32 ? 32 : N;              // tensor-memory columns of N
    static constexpr int chunk = 32 * D * 2;                   // a warp's tokens of V
    static constexpr int VT    = D == 256 ? 1 : 2;             // V tiles in the ring
    static constexpr int KB    = D / 2 * 2 + MT * NP + 2 * NP <= 512 ? 2 : 1;   // K tiles in tensor memory
    static constexpr int SB    = KB * D / 2 + MT * NP + 2 * NP <= 512 ? 2 : 1;  // score buffers
    static constexpr int qtile = N * D * 2;
    static constexpr int planes = (N + 63) / 64;
    static constexpr int ptile = planes * kTile * 128;         // one part of P
    static constexpr int q     = 0;
    static constexpr int ring  = q + parts * qtile;
    static constexpr int p     = ring + VT * 4 * chunk;
    static constexpr int rowb  = D / 16 * 9;
    static constexpr int CB    = D / 16;
    static constexpr int RS    = row_stride(D);
    static constexpr int stage = kRawTok * RS;
    static constexpr int tail  = 3 * 1024 + 24 * N;            // barriers, rows' numbers
    // P buffers: two where shared memory has room for them beside the raw rows of two tiles
    static constexpr int PB    = 232448 - tail - p - 2 * parts * ptile >= 8 * stage ? 2 : 1;
    static constexpr int raw   = p + PB * parts * ptile;
    static constexpr int room  = (232448 - tail - raw) / stage;
    static constexpr int NK    = room >= 12 ? 6 : room >= 6 ? 4 : 2;  // raw stages of K and of V (even: a slot is one half's of the tiles)
    static constexpr int NV    = room >= 12 ? 6 : room >= 8 ? 4 : 2;
    static constexpr int rows  = raw + (NK + NV) * stage;         // off, m, fac, frec: f32 [N]; lo, hi: int [N]
    static constexpr int red   = rows + 24 * N;                // f32 [4][4][32]
    static constexpr int bar   = red + 2048;
    static constexpr int nbar  = 2 * KB + 8 * VT + 2 * SB + PB + 2 + 2 + 2 * (NK + NV);
    static constexpr int misc  = bar + nbar * 8;
    static constexpr int total = misc + 80;
    static constexpr int CW    = N / 4;                        // columns (rows of Q) of a softmax thread
    static constexpr uint32_t tO = 0, tS = MT * NP, tK = tS + SB * NP;
    static_assert(total <= 232448 && raw % 128 == 0 && rows >= kMaxSeqs * 8, "shared memory");
    static_assert(tK + KB * D / 2 <= 512, "tensor memory");
    // registers of the softmax warps, of the MMA's and the producers', of the unpacking ones: the launch's 72 a thread, shared out anew
    static constexpr int rs = N == 96 ? 88 : N == 64 ? 80 : 72, rm = N == 96 ? 40 : 56, ru = N == 96 ? 56 : N == 64 ? 64 : 80;
    static_assert(kSm * 32 * rs + 128 * rm + kConv * 32 * ru <= kThr * 72, "registers");
};

// A from tensor memory (K-major f16 pairs, lane = row)
__device__ __forceinline__ void mma_f16_ta(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(id), "r"(accumulate), "r"(0u)
        : "memory");
}
__device__ __forceinline__ void wait_bar(uint64_t * bar, uint32_t parity, int32_t * status, bool & bad) {
    if (bad) return;
    for (uint32_t i = 0; i < kProbes; i++) {
        if (mbar_try_wait(bar, parity)) return;
    }
    bad = true;  // this thread waits for nothing more: its results are void, its accesses stay in bounds
    atomicExch(status, kErrWaitFull);
}
// true for all `count` threads of barrier `id` if one of them says so
__device__ __forceinline__ bool bar_any(int id, int count, bool v) {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %3, 0;\n\tbar.red.or.pred q, %1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(r)
                 : "r"(id), "r"(count), "r"((uint32_t) v)
                 : "memory");
    return r != 0;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// o += what the record holds of it, times the factors that its rows were rescaled by since; all loads in flight at once
template <int W> __device__ __forceinline__ void add_record(uint32_t (&o)[W], const float * rec, int stride, int n, const float * f) {
    float x[W];
#pragma unroll
    for (int e = 0; e < W; e++) x[e] = e < n ? rec[e * stride] : 0.0f;
#pragma unroll
    for (int e = 0; e < W; e++) o[e] = __float_as_uint(fmaf(x[e], f[e], __uint_as_float(o[e])));
}

// W columns (a power of two, or 24) over the warp's 32 lanes: afterwards lane l has the result of column l % W in x[0]
template <int W, class T, class F> __device__ __forceinline__ float fold(T (&x)[W], F f) {
    if constexpr (W == 24) {
        T y[32];
#pragma unroll
        for (int k = 0; k < 32; k++) y[k] = k < 24 ? x[k < 24 ? k : 0] : x[0];
        return fold(y, f);
    }
    const int lane = threadIdx.x & 31;
    int       n = W;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        if (o >= W) {
#pragma unroll
            for (int k = 0; k < W; k++) x[k] = f(x[k], __shfl_xor_sync(0xffffffffu, x[k], o));
        } else {
            n = o;
#pragma unroll
            for (int k = 0; k < W / 2; k++) {
                if (k < n) {
                    const T keep = (lane & o) ? x[k + n] : x[k], give = (lane & o) ? x[k] : x[k + n];
                    x[k]             = f(keep, __shfl_xor_sync(0xffffffffu, give, o));
                }
            }
        }
    }
    if constexpr (sizeof(T) == 4 && !std::is_same<T, float>::value) {
        return __uint_as_float(x[0]);
    } else {
        return x[0];
    }
}

template <int D, int N, bool PREC>
__global__ void __launch_bounds__(kThr, 1)
    fa_paged_q4_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv, const __grid_constant__ PArgs a,
                       const __grid_constant__ Pool4 kp, const __grid_constant__ Pool4 vp) {
    using Ly           = LayT<D, N, PREC>;
    constexpr int KB = Ly::KB, SB = Ly::SB, PB = Ly::PB, VT = Ly::VT, NK = Ly::NK, NV = Ly::NV, CW = Ly::CW;
    extern __shared__ __align__(1024) uint8_t sm[];
    uint64_t * kfull  = reinterpret_cast<uint64_t *>(sm + Ly::bar);
    uint64_t * kempty = kfull + KB;
    uint64_t * vfull  = kempty + KB;
    uint64_t * vempty = vfull + 4 * VT;
    uint64_t * sfull  = vempty + 4 * VT;
    uint64_t * sfree  = sfull + SB;
    uint64_t * pfull  = sfree + SB;
    uint64_t * pvdone = pfull + PB;  // [2] in turn
    uint64_t * qfull  = pvdone + 2;
    uint64_t * qempty = qfull + 1;
    uint64_t * rfull  = qempty + 1;         // K's NK, V's NV
    uint64_t * rempty = rfull + NK + NV;
    uint32_t * tptr   = reinterpret_cast<uint32_t *>(sm + Ly::misc);
    int *      first  = reinterpret_cast<int *>(sm + Ly::misc + 16);
    int64_t *  range  = reinterpret_cast<int64_t *>(sm + Ly::misc + 32);
    uint64_t * mdone  = reinterpret_cast<uint64_t *>(sm + Ly::misc + 64);  // all products

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    bool      bad = false;
    if (smem_u32(sm) & 1023u) {  // the swizzled operands need it; the linker places the only shared array so
        if (tid == 0) atomicExch(a.status, kErrWaitFull);
        pdl_wait();
        return;
    }
    if (tid == 0) {
        for (int i = 0; i < KB; i++) {
            mbar_init(&kfull[i], kConv / 2);
            mbar_init(&kempty[i], 1);
        }
        for (int i = 0; i < 4 * VT; i++) {
            mbar_init(&vfull[i], 1);
            mbar_init(&vempty[i], 1);
        }
        for (int i = 0; i < SB; i++) {
            mbar_init(&sfull[i], 1);
            mbar_init(&sfree[i], kSm);
        }
        for (int i = 0; i < PB; i++) mbar_init(&pfull[i], kSm);
        for (int i = 0; i < 2; i++) mbar_init(&pvdone[i], 1);
        mbar_init(qfull, kSm);
        mbar_init(qempty, 1);
        mbar_init(mdone, 1);
        for (int i = 0; i < NK + NV; i++) {
            mbar_init(&rfull[i], a.box ? 1 : 32);
            mbar_init(&rempty[i], 2);
        }
        fence_mbar_init();
        first[0] = -1;
    }
    if (warp == kSm) tc::tmem_alloc(tptr, 512);
    pdl_launch_dependents();
    pdl_wait();
    plan_part<N, kTile, true>(a, reinterpret_cast<int *>(sm), reinterpret_cast<int *>(sm + Ly::red), first, range);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tb = *tptr;
    if (tid == 0) a.desc[2 * blockIdx.x] = make_int4(0, 0, 0, 0);
    Walk w;
    w.s         = first[0];
    bool active = w.s >= 0;
    if (active) {
        w.h   = first[1];
        w.rt  = first[2];
        w.off = first[3];
        w.rem = w.part = range[1] - range[0];
        walk_load<N>(a, w);
        walk_item<N, kTile>(a, w);
    }

    if (warp < kSm) {
        if constexpr (Ly::rs > 72) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Ly::rs));
        // ---------------- softmax ----------------
        const int wg = warp >> 2, wq = warp & 3, tg = tid & 127, bid = 1 + wg, g0 = wg * CW;  // rows g0 .. g0 + CW - 1
        float *   off = reinterpret_cast<float *>(sm + Ly::rows) + g0, *mrow = off + N, *fac = mrow + N, *frec = fac + N;
        int *     rlo = reinterpret_cast<int *>(frec + N), *rhi = rlo + N;
        float *   red = reinterpret_cast<float *>(sm + Ly::red) + wg * 128;
        // dim of this lane's row of O^T, of each product along the dims
        const int  od   = D == 64 ? q4::value_at(16 * wq + (lane & 15)) : 64 * (wq >> 1) + q4::value_at(32 * (wq & 1) + lane);
        const bool mine = D != 64 || lane < 16;
        uint32_t   gi = 0, pvw = 0, items = 0;
        auto       pv_wait = [&](uint32_t upto) {
            for (; pvw < upto; pvw++) wait_bar(&pvdone[pvw & 1], (pvw >> 1) & 1, a.status, bad);
        };
        // Q of an item: 16-byte pieces of 8 dims in K's order, 128-byte swizzle; rows that are none as zeros
        auto bring_q = [&](const Walk & w) {
            if (w.sp.nkv == 0) return;
            const int rb = w.rt * N, rows = min(N, w.n * a.G - rb);
            if (items > 0) wait_bar(qempty, (items - 1) & 1, a.status, bad);
            items++;
#pragma unroll 1
            for (int v = tid; v < N * (D / 8); v += kSm * 32) {
                const int row = v / (D / 8), pc = v % (D / 8), odd = (pc >> 2) & 1, word = pc & 3;
                uint2     x[4];
#pragma unroll
                for (int e = 0; e < 4; e++) x[e] = make_uint2(0u, 0u);
                if (row < rows) {
                    const int       tok = a.byG.div(rb + row), h = w.h * a.G + (rb + row - tok * a.G);
                    const uint8_t * src = a.q + (int64_t) (w.r0 + tok) * a.qnb1 + (int64_t) h * a.qnb2;
#pragma unroll
                    for (int e = 0; e < 4; e++) {  // pairs of neighbouring dims: bytes 0, 1 and 2, 3, low and high halves
                        const int d = (pc >> 2) * 32 + q4::byte_of(odd, word, 2 * (e & 1)) + 16 * (e >> 1);
                        if constexpr (PREC) {
                            x[e] = *reinterpret_cast<const uint2 *>(src + 4 * d);
                        } else {
                            x[e].x = *reinterpret_cast<const uint32_t *>(src + 2 * d);
                        }
                    }
                }
                uint8_t * to = sm + Ly::q + (pc >> 3) * (N * 128) + row * 128 + (((pc & 7) ^ (row & 7)) << 4);
                uint32_t  hw[4], lw[4];
#pragma unroll
                for (int e = 0; e < 2; e++) {  // low halves, high halves
                    const uint2 A = x[2 * e], B = x[2 * e + 1];
                    if constexpr (PREC) {
                        const float f[4] = { __uint_as_float(A.x), __uint_as_float(B.x), __uint_as_float(A.y), __uint_as_float(B.y) };
#pragma unroll
                        for (int m = 0; m < 2; m++) {
                            const __half2 h2 = __floats2half2_rn(f[2 * m], f[2 * m + 1]);
                            const __half2 l2 = __floats2half2_rn(f[2 * m] - __low2float(h2), f[2 * m + 1] - __high2float(h2));
                            hw[2 * e + m] = *reinterpret_cast<const uint32_t *>(&h2);
                            lw[2 * e + m] = *reinterpret_cast<const uint32_t *>(&l2);
                        }
                    } else {
                        hw[2 * e]     = q4::prmt(A.x, B.x, 0x5410u);
                        hw[2 * e + 1] = q4::prmt(A.x, B.x, 0x7632u);
                    }
                }
                *reinterpret_cast<uint4 *>(to) = make_uint4(hw[0], hw[1], hw[2], hw[3]);
                if constexpr (PREC) *reinterpret_cast<uint4 *>(to + Ly::qtile) = make_uint4(lw[0], lw[1], lw[2], lw[3]);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(qfull);
        };
        // O's part of this group: f(values, product along the dims, place)
        auto each_o = [&](auto f) {
#pragma unroll 1
            for (int mt = 0; mt < Ly::MT; mt++) {
                uint32_t       o[CW];
                const uint32_t at = tc::taddr(tb + Ly::tO + mt * Ly::NP + g0, wq, 0);
                tc::ld_cols<CW>(at, o);
                tc::wait_ld();
                f(o, mt, at);
            }
        };
        const float qs = a.softcap_l2 != 0.0f ? 1.0f : a.qscale;
        if (active) bring_q(w);
        while (active) {
            const int  n = w.sp.nkv ? w.take : 0, rb = w.rt * N, rows = min(N, w.n * a.G - rb);
            const int  slot = 2 * blockIdx.x + (w.off == 0 ? 1 : 0);
            const bool whole = w.off == 0 && w.take == w.sp.units;
            if (tg < CW) {
                const bool is = g0 + tg < rows;
                const int  pos = w.kv - w.n + a.byG.div(rb + (is ? g0 + tg : 0));
                rhi[tg]  = is ? min(pos + 1, w.sp.hi) : 0;
                rlo[tg]  = a.window > 0 ? max(w.sp.lo, (int) max((int64_t) INT32_MIN, (int64_t) pos - a.window + 1)) : w.sp.lo;
                off[tg]  = is ? kUnset : INFINITY;  // rows that are none: p = 0
                mrow[tg] = is ? -INFINITY : INFINITY;
                frec[tg] = 1.0f;
            }
            named_bar_sync(bid, 128);
            // tokens that every row sees
            const int pmin = w.kv - w.n + a.byG.div(rb), pmax = w.kv - w.n + a.byG.div(rb + rows - 1);
            const int ahi = min(pmin + 1, w.sp.hi), alo = a.window > 0 ? (int) max((int64_t) 0, (int64_t) pmax - a.window + 1) : w.sp.lo;
            float     l[CW];
#pragma unroll
            for (int e = 0; e < CW; e++) l[e] = 0.0f;
#pragma unroll 1
            for (int i = 0; i < n; i++, gi++) {
                const uint32_t sb = gi % SB, pb = gi % PB;
                const int      t0 = w.tile(i) * kTile, pos = t0 + 32 * wq + lane;
                const bool     mask = t0 < alo || t0 + kTile > ahi;
                wait_bar(&sfull[sb], (gi / SB) & 1, a.status, bad);
                tc::fence_after();
                if constexpr (PREC) {
                    if (i > 0 && i % kFlush == 0) {  // O so far to the record
                        pv_wait(gi);
                        tc::fence_after();
                        each_o([&](uint32_t (&o)[CW], int mt, uint32_t) {
                            float *   rec = a.part_acc + ((int64_t) slot * a.prow + g0) * D + 128 * mt + od;
                            const int nr  = mine ? rows - g0 : 0;
                            if (i > kFlush) add_record(o, rec, D, nr, frec);
#pragma unroll
                            for (int e = 0; e < CW; e++) {
                                if (e < nr) rec[e * D] = __uint_as_float(o[e]);
                            }
                        });
                        named_bar_sync(bid, 128);
                        if (tg < CW) frec[tg] = 1.0f;
                    }
                }
                const uint32_t ts = tc::taddr(tb + Ly::tS + sb * Ly::NP + g0, wq, 0);
                uint32_t       s[CW];
                auto           scores = [&]() {
                    tc::ld_cols<CW>(ts, s);
                    tc::wait_ld();
                    if (a.softcap_l2 != 0.0f) {
#pragma unroll
                        for (int e = 0; e < CW; e++) s[e] = __float_as_uint(a.softcap_l2 * tanhf(__uint_as_float(s[e]) * a.qscale));
                    }
                    if (mask) {
#pragma unroll
                        for (int e = 0; e < CW; e++) {
                            if (pos < rlo[e] || pos >= rhi[e]) s[e] = __float_as_uint(-INFINITY);
                        }
                    }
                };
                auto shifted = [&]() {
                    float top = -INFINITY;
#pragma unroll
                    for (int e = 0; e < CW; e += 4) {
                        const float4 o = *reinterpret_cast<const float4 *>(off + e);
                        float        x0, x1, x2, x3;
                        f2_unpack(f2_fma(f2_pack(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), f2_pack(qs, qs), f2_pack(-o.x, -o.y)), x0, x1);
                        f2_unpack(f2_fma(f2_pack(__uint_as_float(s[e + 2]), __uint_as_float(s[e + 3])), f2_pack(qs, qs), f2_pack(-o.z, -o.w)), x2, x3);
                        s[e] = __float_as_uint(x0); s[e + 1] = __float_as_uint(x1); s[e + 2] = __float_as_uint(x2); s[e + 3] = __float_as_uint(x3);
                        top = max3(max3(top, x0, x1), x2, x3);
                    }
                    return top;
                };
                scores();
                const float top = shifted();
                if (bar_any(bid, 128, top > kLazy + kShift)) {
                    // raise the rows' references: largest scores over the tile's tokens
                    scores();
                    const float best = qs * fold(s, [](uint32_t u, uint32_t v) { return __float_as_uint(fmaxf(__uint_as_float(u), __uint_as_float(v))); });
                    if (lane < CW) red[wq * 32 + lane] = best;
                    named_bar_sync(bid, 128);
                    if (tg < CW) {
                        const float v = fmaxf(fmaxf(red[tg], red[32 + tg]), fmaxf(red[64 + tg], red[96 + tg])), mo = mrow[tg];
                        float       f = 1.0f;
                        if (v > mo + kLazy) {  // of -inf: any score
                            f        = exp2a(mo - v);
                            mrow[tg] = v;
                            off[tg]  = v - kShift;
                            frec[tg] *= f;
                        }
                        fac[tg] = f;
                    }
                    named_bar_sync(bid, 128);
#pragma unroll
                    for (int e = 0; e < CW; e++) l[e] *= fac[e];
                    if (i > 0 && (!PREC || i % kFlush)) {
                        pv_wait(gi);
                        tc::fence_after();
                        each_o([&](uint32_t (&o)[CW], int, uint32_t at) {
#pragma unroll
                            for (int e = 0; e < CW; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * fac[e]);
                            tc::st_cols<CW>(at, o);
                        });
                        tc::wait_st();
                    }
                    scores();
                    shifted();
                }
                tc::fence_before();  // S is read
                __syncwarp();
                if (lane == 0) mbar_arrive(&sfree[sb]);
                uint8_t * pr = sm + Ly::p + pb * Ly::parts * Ly::ptile + (32 * wq + lane) * 128;
                uint32_t  hi[CW / 2];
                [[maybe_unused]] uint32_t lo[CW / 2];
#pragma unroll
                for (int k = 0; k < CW / 2; k++) {
                    const float x0 = exp2a(__uint_as_float(s[2 * k])), x1 = exp2a(__uint_as_float(s[2 * k + 1]));
                    f2_unpack(f2_add(f2_pack(l[2 * k], l[2 * k + 1]), f2_pack(x0, x1)), l[2 * k], l[2 * k + 1]);
                    const __half2 h2 = __floats2half2_rn(x0, x1);
                    hi[k]            = *reinterpret_cast<const uint32_t *>(&h2);
                    if constexpr (PREC) {
                        const __half2 r2 = __floats2half2_rn(x0 - __low2float(h2), x1 - __high2float(h2));
                        lo[k]            = *reinterpret_cast<const uint32_t *>(&r2);
                    }
                }
                pv_wait(gi + 1 > PB ? gi + 1 - PB : 0);  // the product that read this P buffer
                if constexpr (CW >= 8) {
#pragma unroll
                    for (int k = 0; k < CW / 2; k += 4) {
                        uint8_t * to = pr + ((g0 + 2 * k) >> 6) * (kTile * 128) + (((((g0 + 2 * k) >> 3) & 7) ^ (lane & 7)) << 4);
                        *reinterpret_cast<uint4 *>(to) = make_uint4(hi[k], hi[k + 1], hi[k + 2], hi[k + 3]);
                        if constexpr (PREC) *reinterpret_cast<uint4 *>(to + Ly::ptile) = make_uint4(lo[k], lo[k + 1], lo[k + 2], lo[k + 3]);
                    }
                } else {  // four rows: half a piece
                    uint8_t * to = pr + (((g0 >> 3) ^ (lane & 7)) << 4) + 2 * (g0 & 7);
                    *reinterpret_cast<uint2 *>(to) = make_uint2(hi[0], hi[1]);
                    if constexpr (PREC) *reinterpret_cast<uint2 *>(to + Ly::ptile) = make_uint2(lo[0], lo[1]);
                }
                fence_proxy_async_smem();
                tc::fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&pfull[pb]);
            }
            // ---------------- the item's end; the next one's Q before it, so that its products start meanwhile ----------------
            Walk       nw   = w;
            const bool more = walk_next<N, kTile>(a, nw);
            if (more) bring_q(nw);
            const float sum = fold(l, [](float u, float v) { return u + v; });
            if (lane < CW) red[wq * 32 + lane] = sum;
            named_bar_sync(bid, 128);
            if (tg < CW && g0 + tg < rows) {
                const int   r = g0 + tg, tok = a.byG.div(rb + r), h = w.h * a.G + (rb + r - tok * a.G);
                float       L = (red[tg] + red[32 + tg]) + (red[64 + tg] + red[96 + tg]);
                const float M = mrow[tg];
                float       f = 1.0f;
                if (!whole) {
                    a.part_ms[(int64_t) slot * a.prow + r] = make_float2(M, L);
                } else {
                    if (a.sinks) {  // relative to the larger of the two
                        const float sk = a.sinks[h] * kLog2e;
                        if (sk > M) {
                            f = M == -INFINITY ? 0.0f : exp2a(M - sk);
                            L = L * f + exp2f(kShift);
                        } else if (sk > -INFINITY) {
                            L += exp2a(sk - M + kShift);
                        }
                    }
                    f = L == 0.0f ? 0.0f : f / L;  // a NaN stays one
                }
                fac[tg] = f;
            }
            named_bar_sync(bid, 128);
            if (n > 0) {
                pv_wait(gi);
                tc::fence_after();
            }
            if (g0 < rows) {
                auto put = [&](uint32_t (&o)[CW], int mt, uint32_t) {
                    float * rec = a.part_acc + ((int64_t) slot * a.prow + g0) * D + 128 * mt + od;
                    if (PREC && n > kFlush) add_record(o, rec, D, mine ? rows - g0 : 0, frec);
#pragma unroll
                    for (int e = 0; e < CW; e++) {
                        const int r = g0 + e;
                        if (!mine || r >= rows) continue;
                        float x = __uint_as_float(o[e]);
                        if (!whole) {
                            rec[e * D] = x;
                            continue;
                        }
                        const float f = fac[e];
                        x             = f != 0.0f ? x * f : 0.0f;
                        const int tok = a.byG.div(rb + r), h = w.h * a.G + (rb + r - tok * a.G);
                        uint8_t * dst = a.dst + (int64_t) h * a.dnb1 + (int64_t) (w.r0 + tok) * a.dnb2;
                        if constexpr (PREC) {
                            reinterpret_cast<float *>(dst)[128 * mt + od] = x;
                        } else {
                            reinterpret_cast<__half *>(dst)[128 * mt + od] = __float2half_rn(x);
                        }
                    }
                };
                if (n > 0) {
                    each_o(put);
                } else {
                    uint32_t o[CW];
#pragma unroll
                    for (int e = 0; e < CW; e++) o[e] = 0;
                    for (int mt = 0; mt < Ly::MT; mt++) put(o, mt, 0);
                }
            }
            tc::fence_before();  // O is read: the next item's products may write it
            if (tid == 0 && !whole && w.off == 0) {
                // this CTA opens an item that others go on with: parts of it, for the join
                const int64_t end = range[0] + (range[1] - range[0] - w.rem) + w.sp.units;
                const int     e   = part_of_end(range[2], range[3], end, blockIdx.x);
                a.desc[2 * blockIdx.x + 1] = make_int4(rb, rows, 0, 0);
                a.desc[2 * blockIdx.x]     = make_int4(e - (int) blockIdx.x + 1, w.h, w.r0, 0);
            }
            named_bar_sync(bid, 128);  // the rows' numbers are read
            w      = nw;
            active = more;
        }
    } else if (warp < kSm + 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Ly::rm));
        if (warp == kSm) {
            // ---------------- MMA ----------------
            constexpr uint32_t idqk = tc::idesc(tc::kD_F32, tc::kAB_F16, tc::kAB_F16, tc::kKMajor, tc::kKMajor, N, 128);
            constexpr uint32_t idpv = tc::idesc(tc::kD_F32, tc::kAB_F16, tc::kAB_F16, tc::kMNMajor, tc::kMNMajor, N, Ly::MM);
            constexpr uint64_t sw   = 2ull << 61;  // 128-byte swizzle
            const uint64_t     qd0  = tc::sdesc(smem_u32(sm + Ly::q), 16, 1024) | sw;  // addresses step by bytes / 16
            const uint64_t     vd0  = tc::sdesc(smem_u32(sm + Ly::ring), 32 * 128, 1024) | sw;
            const uint64_t     pd0  = tc::sdesc(smem_u32(sm + Ly::p), kTile * 128, 1024) | sw;
            uint32_t           gi = 0, items = 0;
            for (; active; active = walk_next<N, kTile>(a, w)) {
                const int n = __shfl_sync(0xffffffffu, w.sp.nkv ? w.take : 0, 0);
                if (n == 0) continue;
                wait_bar(qfull, items & 1, a.status, bad);
                items++;
                auto qk = [&](int i) {
                    const uint32_t g = gi + i, kb = g % KB, sb = g % SB;
                    wait_bar(&kfull[kb], (g / KB) & 1, a.status, bad);
                    if (g >= SB) wait_bar(&sfree[sb], (g / SB - 1) & 1, a.status, bad);
                    tc::fence_after();
                    __syncwarp();
                    if (elect_one()) {
                        // a plane of 64 dims at a time: the descriptors of all products at once would not fit the registers
                        uint64_t qd = qd0;
                        uint32_t ka = tb + Ly::tK + kb * (D / 2);
#pragma unroll 1
                        for (int pl = 0; pl < Ly::parts * (D / 64); pl++) {
#pragma unroll
                            for (int j = 0; j < 4; j++) {
                                mma_f16_ta(tb + Ly::tS + sb * Ly::NP, ka + 8 * j, qd + 2 * j, idqk, (uint32_t) (pl > 0 || j > 0));
                            }
                            qd += N * 128 / 16;
                            ka = pl + 1 == D / 64 ? ka + 32 - D / 2 : ka + 32;
                        }
                        tc::commit(&kempty[kb]);
                        tc::commit(&sfull[sb]);
                        if (i == n - 1) tc::commit(qempty);
                    }
                    __syncwarp();
                };
                qk(0);
                for (int i = 0; i < n; i++) {
                    if (i + 1 < n) qk(i + 1);
                    const uint32_t g = gi + i, pb = g % PB;
                    const bool     fresh = PREC ? i % kFlush == 0 : i == 0;
                    wait_bar(&pfull[pb], (g / PB) & 1, a.status, bad);
#pragma unroll 1
                    for (int ch = 0; ch < 4; ch++) {
                        const uint32_t sl = g % VT * 4 + ch;
                        wait_bar(&vfull[sl], (g / VT) & 1, a.status, bad);
                        tc::fence_after();
                        __syncwarp();
                        if (elect_one()) {
#pragma unroll
                            for (int mt = 0; mt < Ly::MT; mt++) {
                                const uint64_t vd = vd0 + (sl * Ly::chunk + mt * 2 * (32 * 128)) / 16;
                                const uint64_t pd = pd0 + (pb * Ly::parts * Ly::ptile + ch * 4096) / 16;
#pragma unroll
                                for (int k = 0; k < 2; k++) {
#pragma unroll
                                    for (int part = 0; part < Ly::parts; part++) {
                                        tc::mma_f16(tb + Ly::tO + mt * Ly::NP, vd + k * 2048 / 16, pd + (part * Ly::ptile + k * 2048) / 16, idpv,
                                                    (uint32_t) (!fresh || ch > 0 || k > 0 || part > 0));
                                    }
                                }
                            }
                            tc::commit(&vempty[sl]);
                            if (ch == 3) tc::commit(&pvdone[g & 1]);
                        }
                        __syncwarp();
                    }
                }
                gi += n;
            }
            if (elect_one()) tc::commit(mdone);
        } else if (warp < kSm + 3) {
            // ---------------- producers: raw rows, 64 tokens at a time ----------------
            const bool isk = warp == kSm + 1;
            const int  NR = isk ? NK : NV;
            uint64_t * rf = rfull + (isk ? 0 : NK), *re = rempty + (isk ? 0 : NK);
            const uint32_t raw0 = smem_u32(sm + Ly::raw + (isk ? 0 : NK * Ly::stage));
            const Pool4 &  pool = isk ? kp : vp;
            uint32_t       c = 0;  // stages so far
            for (; active; active = walk_next<N, kTile>(a, w)) {
                const int n = w.sp.nkv ? w.take : 0;
                for (int i0 = 0; i0 < n; i0 += 4) {
                    // lane j: page of tokens 16 (j % 8) .. of tile i0 + j / 8: four tiles' at a time, as an entry takes 700 cycles
                    int       ent = -1, y = 0;  // -1: no row sees them
                    const int ti  = i0 + (lane >> 3);
                    if (ti < n) {
                        const int tok = w.tile(ti) * kTile + 16 * (lane & 7);
                        if (tok < w.sp.hi && tok + 16 > w.sp.lo) {
                            const int e = a.byPage.div(tok);
                            y           = tok - e * a.page;
                            ent         = reinterpret_cast<const int32_t *>(a.table + (int64_t) w.s * a.tstride)[e];
                            if (ent < 0 || ent >= a.n_pages) {  // no page: reads as zeros
                                atomicExch(a.status, kErrPage);
                                ent = a.n_pages;
                            }
                        }
                    }
                    for (int st = 0; st < 2 * min(4, n - i0); st++, c++) {
                        const uint32_t sl = c % NR;
                        if (c >= (uint32_t) NR) wait_bar(&re[sl], (c / NR - 1) & 1, a.status, bad);
                        bad = __any_sync(0xffffffffu, bad);  // the warp gives up as one: the lanes shuffle below
                        if (bad) break;
                        const uint32_t to = raw0 + sl * Ly::stage;
                        int            pg[4], yy[4];
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            pg[k] = __shfl_sync(0xffffffffu, ent, 4 * st + k);
                            yy[k] = __shfl_sync(0xffffffffu, y, 4 * st + k);
                        }
                        if (a.box) {
                            // boxes of 16, 32 or 64 tokens, as pages hold them; one that no row sees is left out
                            const int bs = a.box >> 4, x = (w.h * Ly::rowb) & ~15;
                            int       nb = 0;
#pragma unroll
                            for (int k = 0; k < 4; k++) {
                                // a box's entry and place stand with its first 16 tokens; where those are not seen, with a later 16
                                if (k % bs == 0) {
                                    for (int e = 1; e < bs; e++) {
                                        if (pg[k] < 0 && pg[(k + e) & 3] >= 0) {
                                            pg[k] = pg[(k + e) & 3];
                                            yy[k] = yy[(k + e) & 3] - 16 * e;
                                        }
                                    }
                                    nb += pg[k] >= 0;
                                }
                            }
                            if (elect_one()) {
                                mbar_arrive_expect_tx(&rf[sl], nb * a.box * Ly::RS);
#pragma unroll
                                for (int k = 0; k < 4; k++) {
                                    if (k % bs == 0 && pg[k] >= 0) tma_rows(to + 16 * k * Ly::RS, isk ? &mk : &mv, x, yy[k], pg[k], &rf[sl]);
                                }
                            }
                            __syncwarp();
                        } else {
                            const int64_t hb = w.h * pool.nb2;
#pragma unroll 1
                            for (int k = 0; k < kRawTok * 9; k += 32) {
                                const int     idx = k + lane, tk = idx / 9, pc = idx - 9 * tk, q = tk >> 4;
                                const int     p = q < 2 ? (q ? pg[1] : pg[0]) : q == 2 ? pg[2] : pg[3], yq = (q < 2 ? (q ? yy[1] : yy[0]) : q == 2 ? yy[2] : yy[3]) + (tk & 15);
                                const bool    ok = p >= 0 && p < a.n_pages;
                                const int64_t o = ok ? p * pool.nb3 + yq * pool.nb1 + hb + pc * Ly::CB : 0;
                                q4::copy_async<Ly::CB>(to + tk * Ly::RS + pc * Ly::CB, pool.p + o, ok ? Ly::CB : 0);
                            }
                            asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&rf[sl])) : "memory");
                        }
                    }
                    if (bad) break;
                }
                if (bad) break;
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            // The loads land before this CTA's shared memory goes, those too that a warp whose wait ran out does not take. Nobody else
            // fills this warp's ring, so each slot's last phase is the one waited for.
            for (uint32_t k = c > (uint32_t) NR ? c - NR : 0; a.box && k < c; k++) mbar_wait(&rf[k % NR], (k / NR) & 1);
        }
    } else {
        if constexpr (Ly::ru < 72) {
            asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Ly::ru));
        } else {
            asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Ly::ru));
        }
        // ---------------- unpacking: K into tensor memory, V into swizzled rows ----------------
        const int  wq = warp & 3, th = wq >> 1;  // 32 tokens of the tile
        const bool isk = warp < kSm + 4 + kConv / 2;
        const int  NR = isk ? NK : NV;
        uint64_t * rf = rfull + (isk ? 0 : NK), *re = rempty + (isk ? 0 : NK);
        const uint8_t * raw = sm + Ly::raw + (isk ? 0 : NK * Ly::stage) + (32 * (wq & 1) + lane) * Ly::RS;
        uint32_t        gi = 0;
        for (; active; active = walk_next<N, kTile>(a, w)) {
            const int n = w.sp.nkv ? w.take : 0;
            const int lead = a.box ? (w.h * Ly::rowb) & 15 : 0;
            for (int i = 0; i < n; i++, gi++) {
                const uint32_t c = 2 * gi + th, sl = c % NR, kb = gi % KB, vs = gi % VT * 4 + wq;
                wait_bar(&rf[sl], (c / NR) & 1, a.status, bad);
                __syncwarp();
                const uint8_t * row = raw + sl * Ly::stage + lead;
                uint32_t        W[9];  // of a pair of blocks
                auto            words = [&](int k, int odd) {
                    const uint8_t * r = row + 36 * k;
                    if constexpr (D == 64) {
#pragma unroll
                        for (int e = 0; e < 9; e++) W[e] = *reinterpret_cast<const uint32_t *>(r + 4 * e);
                    } else if (odd == 0) {  // 8-byte loads where they stand on 8 bytes
#pragma unroll
                        for (int e = 0; e < 8; e += 2) {
                            const uint2 x = *reinterpret_cast<const uint2 *>(r + 4 * e);
                            W[e] = x.x; W[e + 1] = x.y;
                        }
                        W[8] = *reinterpret_cast<const uint32_t *>(r + 32);
                    } else {
                        W[0] = *reinterpret_cast<const uint32_t *>(r);
#pragma unroll
                        for (int e = 1; e < 9; e += 2) {
                            const uint2 x = *reinterpret_cast<const uint2 *>(r + 4 * e);
                            W[e] = x.x; W[e + 1] = x.y;
                        }
                    }
                };
                auto release = [&]() {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&re[sl]);
                };
                constexpr int NP2 = D / 64, U2 = NP2 < 2 ? NP2 : 2;  // pairs
                uint32_t      v[16];
                if (isk) {
                    const uint32_t at = tc::taddr(tb + Ly::tK + kb * (D / 2), wq, 0);
                    if (gi >= KB) wait_bar(&kempty[kb], (gi / KB - 1) & 1, a.status, bad);
                    tc::fence_after();
                    __syncwarp();
#pragma unroll 1
                    for (int k0 = 0; k0 < NP2; k0 += U2) {  // not unrolled: the roles' loops share the instruction cache
#pragma unroll
                        for (int e = 0; e < U2; e++) {
                            words(k0 + e, e);
                            if (k0 + e == NP2 - 1) release();
                            q4::unpack<false>(W, v);
                            tc::st16(at + 32 * (k0 + e), v);
                            q4::unpack<true>(W, v);
                            tc::st16(at + 32 * (k0 + e) + 16, v);
                        }
                    }
                    tc::wait_st();
                    tc::fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&kfull[kb]);
                } else {
                    const int  tok  = w.tile(i) * kTile + 32 * wq + lane;
                    const bool none = tok < w.sp.lo || tok >= w.sp.hi;  // no row sees it: zeros, as 0 * NaN is NaN
                    uint8_t *  to   = sm + Ly::ring + vs * Ly::chunk + lane * 128;
                    auto       put  = [&](int plane, int c0) {
                        uint8_t * pl = to + plane * (32 * 128);
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            *reinterpret_cast<uint4 *>(pl + (((c0 + e) ^ (lane & 7)) << 4)) = make_uint4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
                        }
                    };
                    if (gi >= VT) wait_bar(&vempty[vs], (gi / VT - 1) & 1, a.status, bad);
                    __syncwarp();
#pragma unroll 1
                    for (int k0 = 0; k0 < NP2; k0 += U2) {
#pragma unroll
                        for (int e = 0; e < U2; e++) {
                            words(k0 + e, e);
                            if (k0 + e == NP2 - 1) release();
                            if (none) {
#pragma unroll
                                for (int x = 0; x < 9; x++) W[x] = 0;
                            }
                            q4::unpack<false>(W, v);
                            put(k0 + e, 0);
                            q4::unpack<true>(W, v);
                            put(k0 + e, 4);
                        }
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&vfull[vs]);
                }
            }
        }
    }
    __syncwarp();
    tc::fence_before();
    __syncthreads();
    if (warp == kSm) {
        // the softmax warps wait for the last products, unless a wait of theirs ran out
        mbar_wait(mdone, 0);
        tc::tmem_free(tb, 512);
    }
}

template <int D, int N, bool PREC>
int launch_t(srhpm_ctx * ctx, const PArgs & a, const CUtensorMap & mk, const CUtensorMap & mv, const Pool4 & k, const Pool4 & v,
             cudaStream_t stream) {
    using Ly = LayT<D, N, PREC>;
    auto                         kern = fa_paged_q4_kernel<D, N, PREC>;
    static std::atomic<unsigned> done{ 0 };
    const unsigned               bit = 1u << (ctx->device & 31);
    if (!(done.load() & bit)) {
        const int st = cuda_status(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Ly::total));
        if (st != SRHPM_OK) return st;
        done.fetch_or(bit);
    }
    const int st = cuda_status(launch_k_pdl(kern, dim3(ctx->num_sms), dim3(kThr), Ly::total, stream, mk, mv, a, k, v));
    ctx->launches.fetch_add(1);
    if (st != SRHPM_OK) return st;
    return merge_launch(ctx, a, D, PREC, std::min(32, a.prow), stream);
}
template <int D>
int launch_d(srhpm_ctx * ctx, int rows, bool f32, const PArgs & a, const CUtensorMap & mk, const CUtensorMap & mv, const Pool4 & k,
             const Pool4 & v, cudaStream_t stream) {
    if (f32) return rows == 16 ? launch_t<D, 16, true>(ctx, a, mk, mv, k, v, stream) : launch_t<D, 64, true>(ctx, a, mk, mv, k, v, stream);
    return rows == 16   ? launch_t<D, 16, false>(ctx, a, mk, mv, k, v, stream)
           : rows == 64 ? launch_t<D, 64, false>(ctx, a, mk, mv, k, v, stream)
                        : launch_t<D, 96, false>(ctx, a, mk, mv, k, v, stream);
}

}  // namespace

// Rows of a tile, from the average of rows per sequence and KV head, padding included. 16 sequences of 4000 tokens, us by tile:
//   rows per sequence          8     16     64     96
//   24 / 4 heads of 256   6    44     54     70     85    (32 / 8 heads of 128, 8 rows: 38, 77, 87, 106)
//                        12    72     54     71     85    (16 rows: 66, 76, 88, 108; one sequence of 30000 tokens 57, 43, 50, 60)
//                        24   100     88     72     86
//                        60   212    156     77     92
//                        96          224    121     95
//                       126                 122    145
//                       192                 176    150
// A tile of 96 takes 1.2 times one of 64, so the fewer tiles win above that. f32 rows have two parts of each operand, for which shared
// memory holds 64 rows.
int fap::q4_rows(int T, int S, int G, bool f32) {
    const int64_t R = ((int64_t) T * G + S - 1) / S;
    if (R <= 8) return 8;
    if (R <= 16) return 16;
    return f32 || (R + 63) / 64 * 5 <= (R + 95) / 96 * 6 ? 64 : 96;
}

int fap::q4_parts(int rows, int D) { return rows == 8 ? (D == 256 ? 8 : 16) : 1; }

int fap::q4_run(srhpm_ctx * ctx, PArgs & a, const PagedCache & c, int rows, bool f32, cudaStream_t stream) {
    const Pool4 k{ c.k, c.knb1, c.knb2, c.knb3 }, v{ c.v, c.vnb1, c.vnb2, c.vnb3 };
    CUtensorMap maps[2] = {}, &mk = maps[0], &mv = maps[1];
    const int   box = row_stride(c.D);
    // TMA takes the rows where a token's heads stand side by side and tokens and pages start on 16 bytes; other layouts come in
    // pieces by cp.async
    const int rowb = c.D / 16 * 9;
    auto      fits = [&](const Pool4 & p) {
        return (p.nb2 == rowb || c.Hkv == 1) && c.Hkv * rowb >= box && p.nb1 % 16 == 0 && p.nb3 % 16 == 0 &&
               reinterpret_cast<uintptr_t>(p.p) % 16 == 0 && p.nb1 >= (int64_t) c.Hkv * rowb;
    };
    a.box = 0;
    if (fits(k) && fits(v)) {
        // within a page, and within a stage: of the few-row kernel's steps 32 tokens, 16 of 256 values
        a.box = c.page % 32 || (rows == 8 && c.D == 256) ? 16 : c.page % 64 || rows == 8 ? 32 : 64;
        for (const Pool4 * p : { &k, &v }) {
            // a dimension of one element never steps: any valid stride
            const int64_t s3 = c.n_pages > 1 ? p->nb3 : p->nb1 * c.page;
            if (!encode_rows(p == &k ? &mk : &mv, p->p, (uint64_t) c.Hkv * rowb, c.page, c.n_pages, p->nb1, s3, box, a.box)) {
                return SRHPM_ERR_INVALID;
            }
        }
    }
    if (rows == 8) return q4_few_run(ctx, a, maps, c, f32, stream);
    if (c.D == 64) return launch_d<64>(ctx, rows, f32, a, mk, mv, k, v, stream);
    if (c.D == 128) return launch_d<128>(ctx, rows, f32, a, mk, mv, k, v, stream);
    return launch_d<256>(ctx, rows, f32, a, mk, mv, k, v, stream);
}

}  // namespace srhpm
