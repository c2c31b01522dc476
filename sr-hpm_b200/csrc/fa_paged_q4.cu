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
// Work: as in fa_paged.cu, all items' units of 128 tokens stand in one line that is cut into equal parts, one per CTA.
// Roles: 8 softmax warps (two groups, half of the rows each), 1 MMA warp, 3 warps that bring Q, 4 that unpack K and 4 that
// unpack V. An unpacking warp has 32 tokens of each tile and brings their bytes itself, by cp.async into a ring of its own,
// several tiles ahead and across items: 9 pieces make a row of 64 or 128 values, whatever the strides are.
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
namespace {

constexpr int      kTile   = 128;  // tokens of a tile and of a unit of work
constexpr int      kSm     = 8;    // softmax warps
constexpr int      kQW     = 3;    // warps that bring Q
constexpr int      kThr    = (kSm + 1 + kQW + 8) * 32;
constexpr int      kFlush  = 4;    // tiles
constexpr uint32_t kProbes = 1u << 19;  // of a wait before it gives up: about 2 s
constexpr float    kUnset  = -3e38f;    // a row's reference before its first score

struct Pool4 {
    const uint8_t * p;
    int64_t         nb1, nb2, nb3;
};

// a stage's rows: HD values of a token in RS bytes, of which TMA fills all (its boxes start on 16 bytes, a row up to 12 later)
constexpr int row_values(int D) { return D < 128 ? D : 128; }
constexpr int row_stride(int D) { return D < 128 ? 48 : 80; }

template <int D, int N, bool PREC> struct LayT {
    static constexpr int parts = PREC ? 2 : 1;
    static constexpr int MT    = D == 256 ? 2 : 1;             // products along the dims
    static constexpr int MM    = D == 64 ? 64 : 128;           // dims of a product
    static constexpr int NP    = N < 32 ? 32 : N;              // tensor-memory columns of N
    static constexpr int CH    = D == 256 ? 2 : 1;             // chunks of a V tile, 32 KB at most
    static constexpr int vtok  = kTile / CH;
    static constexpr int chunk = vtok * D * 2;
    static constexpr int VS    = 2;                            // chunks in the ring
    static constexpr int KB    = D / 2 * 2 + MT * NP + 2 * NP <= 512 ? 2 : 1;   // K tiles in tensor memory
    static constexpr int SB    = KB * D / 2 + MT * NP + 2 * NP <= 512 ? 2 : 1;  // score buffers
    static constexpr int qtile = N * D * 2;
    static constexpr int planes = (N + 63) / 64;
    static constexpr int ptile = planes * kTile * 128;         // one part of P
    static constexpr int q     = 0;
    static constexpr int ring  = q + parts * qtile;
    static constexpr int p     = ring + VS * chunk;
    // P buffers: two where shared memory has room for them beside three stages of raw rows
    static constexpr int HD    = row_values(D);
    static constexpr int SPT   = D / HD;                       // stages of a tile
    static constexpr int rowb  = HD / 16 * 9;
    static constexpr int CB    = HD / 16;
    static constexpr int RS    = row_stride(D);
    static constexpr int stage = 32 * RS;                      // of one warp
    static constexpr int tail  = 2560 + 24 * N;                // barriers, rows' numbers
    static constexpr int PB    = 232448 - tail - p - 2 * parts * ptile >= 4 * 8 * stage ? 2 : 1;
    static constexpr int raw   = p + PB * parts * ptile;
    static constexpr int room  = (232448 - tail - raw) / (8 * stage);
    static constexpr int ST    = room < 6 * SPT ? room : 6 * SPT;
    static constexpr int rows  = raw + ST * 8 * stage;         // off, m, fac, frec: f32 [N]; lo, hi: int [N]
    static constexpr int red   = rows + 24 * N;                // f32 [2][4][32]
    static constexpr int bar   = red + 1024;
    static constexpr int nbar  = 2 * KB + 2 * VS + 2 * SB + PB + 2 + 2 + 8 * ST;
    static constexpr int misc  = bar + nbar * 8;
    static constexpr int total = misc + 80;
    static constexpr int CW    = N / 2 < 32 ? N / 2 : 32;      // columns that a softmax thread takes at a time
    static constexpr int NC    = N / 2 / CW;
    static constexpr uint32_t tO = 0, tS = MT * NP, tK = tS + SB * NP;
    static_assert(total <= 232448 && ST >= 2 && raw % 16 == 0 && rows >= kMaxSeqs * 8, "shared memory");
    static_assert(tK + KB * D / 2 <= 512, "tensor memory");
    // registers of the softmax warps, of the MMA's and Q's, of the unpacking ones: the launch's 96 a thread, shared out anew
    static constexpr int rs = N == 128 ? 144 : 120, rm = N == 128 ? 72 : 56, ru = N == 128 ? 56 : 88;
    static_assert(256 * rs + 128 * rm + 256 * ru <= kThr * 96, "registers");
};

__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
// A from tensor memory (K-major f16 pairs, lane = row)
__device__ __forceinline__ void mma_f16_ta(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(id), "r"(accumulate), "r"(0u)
        : "memory");
}
__device__ __forceinline__ float exp2a(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ void wait_bar(uint64_t * bar, uint32_t parity, int32_t * status, bool & bad) {
    if (bad) return;
    for (uint32_t i = 0; i < kProbes; i++) {
        if (mbar_try_wait(bar, parity)) return;
    }
    bad = true;  // this thread waits for nothing more: its results are void, its accesses stay in bounds
    atomicExch(status, kErrWaitFull);
}
__device__ __forceinline__ void tma_rows(uint32_t dst, const CUtensorMap * m, int x, int y, int z, uint64_t * bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(m), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
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

template <int W> __device__ __forceinline__ void ld_t(uint32_t t, uint32_t (&r)[W]) {
    if constexpr (W == 32) {
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
            "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
              "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
              "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
              "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
            : "r"(t));
    } else {
        tc::ld8(t, r);
    }
}
template <int W> __device__ __forceinline__ void st_t(uint32_t t, const uint32_t (&r)[W]) {
    if constexpr (W == 32) {
        tc::st16(t, *reinterpret_cast<const uint32_t(*)[16]>(&r[0]));
        tc::st16(t + 16, *reinterpret_cast<const uint32_t(*)[16]>(&r[16]));
    } else {
        tc::st8(t, r);
    }
}

// o += what the record holds of it, times the factors that its rows were rescaled by since; all loads in flight at once
template <int W> __device__ __forceinline__ void add_record(uint32_t (&o)[W], const float * rec, int stride, int n, const float * f) {
    float x[W];
#pragma unroll
    for (int e = 0; e < W; e++) x[e] = e < n ? rec[e * stride] : 0.0f;
#pragma unroll
    for (int e = 0; e < W; e++) o[e] = __float_as_uint(fmaf(x[e], f[e], __uint_as_float(o[e])));
}

// W columns over the warp's 32 lanes: afterwards lane l has the result of column l % W in x[0]
template <int W, class T, class F> __device__ __forceinline__ float fold(T (&x)[W], F f) {
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
    constexpr int KB = Ly::KB, SB = Ly::SB, PB = Ly::PB, VS = Ly::VS, CH = Ly::CH, ST = Ly::ST, CW = Ly::CW, NC = Ly::NC;
    extern __shared__ __align__(1024) uint8_t sm[];
    uint64_t * kfull  = reinterpret_cast<uint64_t *>(sm + Ly::bar);
    uint64_t * kempty = kfull + KB;
    uint64_t * vfull  = kempty + KB;
    uint64_t * vempty = vfull + VS;
    uint64_t * sfull  = vempty + VS;
    uint64_t * sfree  = sfull + SB;
    uint64_t * pfull  = sfree + SB;
    uint64_t * pvdone = pfull + PB;  // [2] in turn
    uint64_t * qfull  = pvdone + 2;
    uint64_t * qempty = qfull + 1;
    uint64_t * rawfull = qempty + 1;  // [8][ST]
    uint32_t * tptr   = reinterpret_cast<uint32_t *>(sm + Ly::misc);
    int *      first  = reinterpret_cast<int *>(sm + Ly::misc + 16);
    int64_t *  range  = reinterpret_cast<int64_t *>(sm + Ly::misc + 32);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    bool      bad = false;
    if (smem_u32(sm) & 1023u) {  // the swizzled operands need it; the linker places the only shared array so
        if (tid == 0) atomicExch(a.status, kErrWaitFull);
        pdl_wait();
        return;
    }
    if (tid == 0) {
        for (int i = 0; i < KB; i++) {
            mbar_init(&kfull[i], 4);
            mbar_init(&kempty[i], 1);
        }
        for (int i = 0; i < VS; i++) {
            mbar_init(&vfull[i], 4 / CH);
            mbar_init(&vempty[i], 1);
        }
        for (int i = 0; i < SB; i++) {
            mbar_init(&sfull[i], 1);
            mbar_init(&sfree[i], kSm);
        }
        for (int i = 0; i < PB; i++) mbar_init(&pfull[i], kSm);
        for (int i = 0; i < 2; i++) mbar_init(&pvdone[i], 1);
        mbar_init(qfull, kQW);
        mbar_init(qempty, 1);
        for (int i = 0; i < 8 * ST; i++) mbar_init(&rawfull[i], a.box ? 1 : 32);
        fence_mbar_init();
        first[0] = -1;
    }
    if (warp == kSm) tc::tmem_alloc(tptr, 512);
    pdl_launch_dependents();
    pdl_wait();
    plan_part<N, kTile>(a, reinterpret_cast<int *>(sm), reinterpret_cast<int *>(sm + Ly::red), first, range);
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
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Ly::rs));
        // ---------------- softmax ----------------
        const int wg = warp >> 2, wq = warp & 3, tg = tid & 127, bid = 1 + wg;
        float *   off = reinterpret_cast<float *>(sm + Ly::rows), *mrow = off + N, *fac = mrow + N, *frec = fac + N;
        int *     rlo = reinterpret_cast<int *>(frec + N), *rhi = rlo + N;
        float *   red = reinterpret_cast<float *>(sm + Ly::red) + wg * 128;
        const int g0  = wg * (N / 2);  // this group's rows
        // dim of this lane's row of O^T, of each product along the dims
        const int  od   = D == 64 ? q4::value_at(16 * wq + (lane & 15)) : 64 * (wq >> 1) + q4::value_at(32 * (wq & 1) + lane);
        const bool mine = D != 64 || lane < 16;
        uint32_t   gi = 0, pvw = 0;
        auto       pv_wait = [&](uint32_t upto) {
            for (; pvw < upto; pvw++) wait_bar(&pvdone[pvw & 1], (pvw >> 1) & 1, a.status, bad);
        };
        for (; active; active = walk_next<N, kTile>(a, w)) {
            const int  n = w.sp.nkv ? w.take : 0, rb = w.rt * N, rows = min(N, w.n * a.G - rb);
            const int  slot = 2 * blockIdx.x + (w.off == 0 ? 1 : 0);
            const bool whole = w.off == 0 && w.take == w.sp.units;
            if (tg < N / 2) {
                const int  r = g0 + tg;
                const bool is = r < rows;
                const int  pos = w.kv - w.n + a.byG.div(rb + (is ? r : 0));
                rhi[r]  = is ? min(pos + 1, w.sp.hi) : 0;
                rlo[r]  = a.window > 0 ? max(w.sp.lo, (int) max((int64_t) INT32_MIN, (int64_t) pos - a.window + 1)) : w.sp.lo;
                off[r]  = is ? kUnset : INFINITY;  // rows that are none: p = 0
                mrow[r] = is ? -INFINITY : INFINITY;
                frec[r] = 1.0f;
            }
            named_bar_sync(bid, 128);
            // tokens that every row sees
            const int pmin = w.kv - w.n + a.byG.div(rb), pmax = w.kv - w.n + a.byG.div(rb + rows - 1);
            const int ahi = min(pmin + 1, w.sp.hi), alo = a.window > 0 ? (int) max((int64_t) 0, (int64_t) pmax - a.window + 1) : w.sp.lo;
            float     l[NC][CW];
#pragma unroll
            for (int c = 0; c < NC; c++) {
#pragma unroll
                for (int e = 0; e < CW; e++) l[c][e] = 0.0f;
            }
            const float qs = a.softcap_l2 != 0.0f ? 1.0f : a.qscale;
            // O's part of one chunk of columns: f(values, product along the dims)
            auto each_o = [&](int c0, auto f) {
#pragma unroll 1
                for (int mt = 0; mt < Ly::MT; mt++) {
                    uint32_t       o[CW];
                    const uint32_t at = tc::taddr(tb + Ly::tO + mt * Ly::NP + c0, wq, 0);
                    ld_t<CW>(at, o);
                    tc::wait_ld();
                    f(o, mt, at);
                }
            };
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
#pragma unroll 1
                        for (int c = 0; c < NC; c++) {
                            each_o(g0 + c * CW, [&](uint32_t (&o)[CW], int mt, uint32_t) {
                                float *   rec = a.part_acc + ((int64_t) slot * a.prow + g0 + c * CW) * D + 128 * mt + od;
                                const int nr  = mine ? rows - (g0 + c * CW) : 0;
                                if (i > kFlush) add_record(o, rec, D, nr, frec + g0 + c * CW);
#pragma unroll
                                for (int e = 0; e < CW; e++) {
                                    if (e < nr) rec[e * D] = __uint_as_float(o[e]);
                                }
                            });
                        }
                        named_bar_sync(bid, 128);
                        if (tg < N / 2) frec[g0 + tg] = 1.0f;
                    }
                }
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    const int      c0 = g0 + c * CW;
                    const uint32_t ts = tc::taddr(tb + Ly::tS + sb * Ly::NP + c0, wq, 0);
                    uint32_t       s[CW];
                    auto           scores = [&]() {
                        ld_t<CW>(ts, s);
                        tc::wait_ld();
                        if (a.softcap_l2 != 0.0f) {
#pragma unroll
                            for (int e = 0; e < CW; e++) s[e] = __float_as_uint(a.softcap_l2 * tanhf(__uint_as_float(s[e]) * a.qscale));
                        }
                        if (mask) {
#pragma unroll
                            for (int e = 0; e < CW; e++) {
                                if (pos < rlo[c0 + e] || pos >= rhi[c0 + e]) s[e] = __float_as_uint(-INFINITY);
                            }
                        }
                    };
                    auto shifted = [&]() {
                        float top = -INFINITY;
#pragma unroll
                        for (int e = 0; e < CW; e += 4) {
                            const float4 o = *reinterpret_cast<const float4 *>(off + c0 + e);
                            float        x0, x1, x2, x3;
                            f2_unpack(f2_fma(f2_pack(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), f2_pack(qs, qs), f2_pack(-o.x, -o.y)), x0, x1);
                            f2_unpack(f2_fma(f2_pack(__uint_as_float(s[e + 2]), __uint_as_float(s[e + 3])), f2_pack(qs, qs), f2_pack(-o.z, -o.w)), x2, x3);
                            s[e] = __float_as_uint(x0); s[e + 1] = __float_as_uint(x1); s[e + 2] = __float_as_uint(x2); s[e + 3] = __float_as_uint(x3);
                            top = fmaxf(fmaxf(top, fmaxf(x0, x1)), fmaxf(x2, x3));
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
                            const float v = fmaxf(fmaxf(red[tg], red[32 + tg]), fmaxf(red[64 + tg], red[96 + tg])), mo = mrow[c0 + tg];
                            float       f = 1.0f;
                            if (v > mo + kLazy) {  // of -inf: any score
                                f             = exp2a(mo - v);
                                mrow[c0 + tg] = v;
                                off[c0 + tg]  = v - kShift;
                                frec[c0 + tg] *= f;
                            }
                            fac[c0 + tg] = f;
                        }
                        named_bar_sync(bid, 128);
#pragma unroll
                        for (int e = 0; e < CW; e++) l[c][e] *= fac[c0 + e];
                        if (i > 0 && (!PREC || i % kFlush)) {
                            pv_wait(gi);
                            tc::fence_after();
                            each_o(c0, [&](uint32_t (&o)[CW], int, uint32_t at) {
#pragma unroll
                                for (int e = 0; e < CW; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * fac[c0 + e]);
                                st_t<CW>(at, o);
                            });
                            tc::wait_st();
                        }
                        scores();
                        shifted();
                    }
                    if (c == NC - 1) {  // S is read
                        tc::fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sfree[sb]);
                    }
                    if (c == 0) pv_wait(gi + 1 > PB ? gi + 1 - PB : 0);  // the product that read this P buffer
                    uint8_t * pr = sm + Ly::p + pb * Ly::parts * Ly::ptile + (c0 >> 6) * (kTile * 128) + (32 * wq + lane) * 128;
#pragma unroll
                    for (int e = 0; e < CW; e += 8) {
                        uint32_t hi[4], lo[4];
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const float x0 = exp2a(__uint_as_float(s[e + 2 * k])), x1 = exp2a(__uint_as_float(s[e + 2 * k + 1]));
                            f2_unpack(f2_add(f2_pack(l[c][e + 2 * k], l[c][e + 2 * k + 1]), f2_pack(x0, x1)), l[c][e + 2 * k], l[c][e + 2 * k + 1]);
                            const __half2 h2 = __floats2half2_rn(x0, x1);
                            hi[k]            = *reinterpret_cast<const uint32_t *>(&h2);
                            if constexpr (PREC) {
                                const __half2 r2 = __floats2half2_rn(x0 - __low2float(h2), x1 - __high2float(h2));
                                lo[k]            = *reinterpret_cast<const uint32_t *>(&r2);
                            }
                        }
                        uint8_t * to = pr + (((((c0 + e) >> 3) & 7) ^ (lane & 7)) << 4);
                        *reinterpret_cast<uint4 *>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                        if constexpr (PREC) *reinterpret_cast<uint4 *>(to + Ly::ptile) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                    }
                }
                fence_proxy_async_smem();
                tc::fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&pfull[pb]);
            }
            // ---------------- the item's end ----------------
#pragma unroll
            for (int c = 0; c < NC; c++) {
                const int   c0 = g0 + c * CW;
                const float sum = fold(l[c], [](float u, float v) { return u + v; });
                if (lane < CW) red[wq * 32 + lane] = sum;
                named_bar_sync(bid, 128);
                if (tg < CW && c0 + tg < rows) {
                    const int   r = c0 + tg, tok = a.byG.div(rb + r), h = w.h * a.G + (rb + r - tok * a.G);
                    float       L = (red[tg] + red[32 + tg]) + (red[64 + tg] + red[96 + tg]);
                    const float M = mrow[r];
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
                    fac[r] = f;
                }
                named_bar_sync(bid, 128);
            }
            if (n > 0) {
                pv_wait(gi);
                tc::fence_after();
            }
#pragma unroll 1
            for (int c = 0; c < NC; c++) {
                const int c0 = g0 + c * CW;
                if (c0 >= rows) break;
                auto put = [&](uint32_t (&o)[CW], int mt, uint32_t) {
                    float * rec = a.part_acc + ((int64_t) slot * a.prow + c0) * D + 128 * mt + od;
                    if (PREC && n > kFlush) add_record(o, rec, D, mine ? rows - c0 : 0, frec + c0);
#pragma unroll
                    for (int e = 0; e < CW; e++) {
                        const int r = c0 + e;
                        if (!mine || r >= rows) continue;
                        float x = __uint_as_float(o[e]);
                        if (!whole) {
                            rec[e * D] = x;
                            continue;
                        }
                        const float f = fac[r];
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
                    each_o(c0, put);
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
                int           e   = blockIdx.x;
                while (range[2] * (e + 1) / range[3] < end) e++;
                a.desc[2 * blockIdx.x + 1] = make_int4(rb, rows, 0, 0);
                a.desc[2 * blockIdx.x]     = make_int4(e - (int) blockIdx.x + 1, w.h, w.r0, 0);
            }
            named_bar_sync(bid, 128);  // the rows' numbers are read
        }
    } else if (warp < kSm + 1 + kQW) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Ly::rm));
        if (warp == kSm) {
            // ---------------- MMA ----------------
            constexpr uint32_t idqk = tc::idesc(tc::kD_F32, tc::kAB_F16, tc::kAB_F16, tc::kKMajor, tc::kKMajor, N, 128);
            constexpr uint32_t idpv = tc::idesc(tc::kD_F32, tc::kAB_F16, tc::kAB_F16, tc::kMNMajor, tc::kMNMajor, N, Ly::MM);
            constexpr uint64_t sw   = 2ull << 61;  // 128-byte swizzle
            const uint64_t     qd0  = tc::sdesc(smem_u32(sm + Ly::q), 16, 1024) | sw;  // addresses step by bytes / 16
            const uint64_t     vd0  = tc::sdesc(smem_u32(sm + Ly::ring), Ly::vtok * 128, 1024) | sw;
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
#pragma unroll
                    for (int ch = 0; ch < CH; ch++) wait_bar(&vfull[(g * CH + ch) % VS], ((g * CH + ch) / VS) & 1, a.status, bad);
                    wait_bar(&pfull[pb], (g / PB) & 1, a.status, bad);
                    tc::fence_after();
                    __syncwarp();
                    if (elect_one()) {
#pragma unroll
                        for (int ch = 0; ch < CH; ch++) {
                            const uint32_t sl = (g * CH + ch) % VS;
#pragma unroll 1
                            for (int mt = 0; mt < Ly::MT; mt++) {
                                uint64_t vd = vd0 + (sl * Ly::chunk + mt * 2 * (Ly::vtok * 128)) / 16;
                                uint64_t pd = pd0 + (pb * Ly::parts * Ly::ptile + ch * (Ly::vtok / 16) * 2048) / 16;
#pragma unroll 1
                                for (int j = 0; j < Ly::vtok / 16; j += 2) {
#pragma unroll
                                    for (int k = 0; k < 2; k++) {
#pragma unroll
                                        for (int part = 0; part < Ly::parts; part++) {
                                            tc::mma_f16(tb + Ly::tO + mt * Ly::NP, vd + k * 2048 / 16, pd + (part * Ly::ptile + k * 2048) / 16, idpv,
                                                        (uint32_t) (!fresh || ch > 0 || j + k > 0 || part > 0));
                                        }
                                    }
                                    vd += 4096 / 16;
                                    pd += 4096 / 16;
                                }
                            }
                            tc::commit(&vempty[sl]);
                        }
                        tc::commit(&pvdone[g & 1]);
                    }
                    __syncwarp();
                }
                gi += n;
            }
        } else {
            // ---------------- Q: 16-byte pieces of 8 dims in K's order, 128-byte swizzle; rows that are none as zeros ----------------
            constexpr int all = N * (D / 8), per = kQW * 32, UN = PREC ? 1 : 2;
            const int     u0 = tid - (kSm + 1) * 32;
            uint32_t      items = 0;
            for (; active; active = walk_next<N, kTile>(a, w)) {
                if (w.sp.nkv == 0) continue;
                const int rb = w.rt * N, rows = min(N, w.n * a.G - rb);
#pragma unroll 1
                for (int u = u0; u < all; u += UN * per) {
                    uint2 x[UN][4];
#pragma unroll
                    for (int k = 0; k < UN; k++) {
                        const int v = u + k * per, row = v / (D / 8), pc = v % (D / 8), odd = (pc >> 2) & 1, word = pc & 3;
#pragma unroll
                        for (int e = 0; e < 4; e++) x[k][e] = make_uint2(0u, 0u);
                        if (v < all && row < rows) {
                            const int       tok = a.byG.div(rb + row), h = w.h * a.G + (rb + row - tok * a.G);
                            const uint8_t * src = a.q + (int64_t) (w.r0 + tok) * a.qnb1 + (int64_t) h * a.qnb2;
#pragma unroll
                            for (int e = 0; e < 4; e++) {  // pairs of neighbouring dims: bytes 0, 1 and 2, 3, low and high halves
                                const int d = (pc >> 2) * 32 + q4::byte_of(odd, word, 2 * (e & 1)) + 16 * (e >> 1);
                                if constexpr (PREC) {
                                    x[k][e] = *reinterpret_cast<const uint2 *>(src + 4 * d);
                                } else {
                                    x[k][e].x = *reinterpret_cast<const uint32_t *>(src + 2 * d);
                                }
                            }
                        }
                    }
                    if (u == u0 && items > 0) wait_bar(qempty, (items - 1) & 1, a.status, bad);
#pragma unroll
                    for (int k = 0; k < UN; k++) {
                        const int v = u + k * per, row = v / (D / 8), pc = v % (D / 8);
                        if (v >= all) break;
                        uint8_t * to = sm + Ly::q + (pc >> 3) * (N * 128) + row * 128 + (((pc & 7) ^ (row & 7)) << 4);
                        uint32_t  hw[4], lw[4];
#pragma unroll
                        for (int e = 0; e < 2; e++) {  // low halves, high halves
                            const uint2 A = x[k][2 * e], B = x[k][2 * e + 1];
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
                }
                items++;
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(qfull);
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Ly::ru));
        // ---------------- unpacking: K into tensor memory, V into swizzled rows ----------------
        const int      wq = warp & 3;
        const bool     isk = warp < kSm + 1 + kQW + 4;
        const Pool4 &  pool = isk ? kp : vp;
        uint8_t *      raw = sm + Ly::raw + (isk ? wq : 4 + wq) * (ST * Ly::stage);
        const uint32_t raw0 = smem_u32(raw);
        // copies: the tile and stage that come next
        uint64_t * rf = rawfull + (isk ? wq : 4 + wq) * ST;
        Walk       pw = w;
        int        pn = w.sp.nkv ? w.take : 0, pi = 0, ph = 0;
        bool       pact = active;
        // lane j: page of the (j / 2)-th tile from i0 on, tokens 16 (j & 1) .. of this warp's 32. Sixteen tiles' at a time: a table
        // entry asked for tile by tile held the warp up for its 700 cycles, half of the tile's time
        int        ent = -1, i0 = 0;
        auto       look = [&]() {
            bool fresh = pi - i0 == 16;
            while (pact && pi >= pn) {
                pact = walk_next<N, kTile>(a, pw);
                pn   = pact && pw.sp.nkv ? pw.take : 0;
                pi   = 0;
                fresh = true;
            }
            if (pact && fresh) {
                i0            = pi;
                const int ti  = pi + (lane >> 1);
                ent           = -1;
                if (ti < pn) {
                    const int tok = pw.tile(ti) * kTile + 32 * wq + 16 * (lane & 1);
                    if (tok < pw.sp.hi && tok + 16 > pw.sp.lo) {
                        ent = reinterpret_cast<const int32_t *>(a.table + (int64_t) pw.s * a.tstride)[a.byPage.div(tok)];
                        if (ent < 0 || ent >= a.n_pages) {  // no page: reads as zeros
                            atomicExch(a.status, kErrPage);
                            ent = a.n_pages;
                        }
                    }
                }
            }
        };
        auto issue = [&](int st) {
            if (!pact) return;
            const uint32_t to = raw0 + st * Ly::stage;
            const int      t0 = pw.tile(pi) * kTile + 32 * wq;
            const int      p0 = __shfl_sync(0xffffffffu, ent, 2 * (pi - i0)), p1 = __shfl_sync(0xffffffffu, ent, 2 * (pi - i0) + 1);  // -1: not seen
            const int      y0 = t0 - a.byPage.div(t0) * a.page, y1 = t0 + 16 - a.byPage.div(t0 + 16) * a.page;
            if (a.box) {
                // boxes of 16 tokens, or of 32 where pages hold them; one that no row sees is left out
                const int  x = (pw.h * (D / 16 * 9) + ph * Ly::rowb) & ~15;
                const bool one = a.box == 32, b0 = p0 >= 0 || (one && p1 >= 0), b1 = !one && p1 >= 0;
                if (elect_one()) {
                    mbar_arrive_expect_tx(&rf[st], (b0 + b1) * a.box * Ly::RS);
                    if (b0) tma_rows(to, isk ? &mk : &mv, x, y0, one ? max(p0, p1) : p0, &rf[st]);
                    if (b1) tma_rows(to + 16 * Ly::RS, isk ? &mk : &mv, x, y1, p1, &rf[st]);
                }
                __syncwarp();
            } else {
                const int64_t o0 = p0 < 0 || p0 >= a.n_pages ? -1 : p0 * pool.nb3 + y0 * pool.nb1 + pw.h * pool.nb2 + ph * Ly::rowb;
                const int64_t o1 = p1 < 0 || p1 >= a.n_pages ? -1 : p1 * pool.nb3 + y1 * pool.nb1 + pw.h * pool.nb2 + ph * Ly::rowb;
#pragma unroll 1
                for (int k = 0; k < 9; k++) {
                    const int     idx = 32 * k + lane, tk = idx / 9, pc = idx - 9 * tk;
                    const int64_t s = tk < 16 ? o0 : o1;
                    q4::copy_async<Ly::CB>(to + tk * Ly::RS + pc * Ly::CB, pool.p + (s < 0 ? 0 : s + (tk & 15) * pool.nb1 + pc * Ly::CB), s < 0 ? 0 : Ly::CB);
                }
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&rf[st])) : "memory");
            }
            if (++ph == Ly::SPT) {
                ph = 0;
                pi++;
                look();
            }
        };
        i0 = -16;
        look();
        for (int s = 0; s < ST; s++) issue(s);
        uint32_t gi = 0, use = 0;
        int      st = 0;
        for (; active; active = walk_next<N, kTile>(a, w)) {
            const int n = w.sp.nkv ? w.take : 0;
            for (int i = 0; i < n; i++, gi++) {
                const uint32_t kb = gi % KB, c = gi * CH + (CH == 2 ? wq >> 1 : 0), sl = c % VS;
                const int      tok = w.tile(i) * kTile + 32 * wq + lane;
                const bool     none = tok < w.sp.lo || tok >= w.sp.hi;  // no row sees it: its V row is zeros, as 0 * NaN is NaN
#pragma unroll 1
                for (int h = 0; h < Ly::SPT; h++) {
                    wait_bar(&rf[st], use & 1, a.status, bad);
                    __syncwarp();
                    const uint8_t * row  = raw + st * Ly::stage + lane * Ly::RS;
                    const int       lead = a.box ? (w.h * (D / 16 * 9) + h * Ly::rowb) & 15 : 0;
                    uint32_t        W[9];  // of a pair of blocks
                    [[maybe_unused]] uint32_t X[20];
                    if constexpr (Ly::HD == 128) {  // the whole row: rows of 80 bytes give 16-byte loads without bank conflicts
#pragma unroll
                        for (int e = 0; e < 5; e++) {
                            const uint4 x = *reinterpret_cast<const uint4 *>(row + 16 * e);
                            X[4 * e] = x.x; X[4 * e + 1] = x.y; X[4 * e + 2] = x.z; X[4 * e + 3] = x.w;
                        }
                    }
                    auto words = [&](int k) {
#pragma unroll
                        for (int e = 0; e < 9; e++) {
                            if constexpr (Ly::HD == 128) {
                                W[e] = lead ? X[9 * k + e + 2] : X[9 * k + e];
                            } else {
                                W[e] = *reinterpret_cast<const uint32_t *>(row + lead + 4 * e);
                            }
                        }
                    };
                    if (isk) {
                        if (h == 0 && gi >= KB) {
                            wait_bar(&kempty[kb], (gi / KB - 1) & 1, a.status, bad);
                            tc::fence_after();
                        }
                        __syncwarp();
#pragma unroll
                        for (int k = 0; k < Ly::HD / 64; k++) {
                            words(k);
                            uint32_t       v[16];
                            const uint32_t at = tc::taddr(tb + Ly::tK + kb * (D / 2) + h * (Ly::HD / 2) + 32 * k, wq, 0);
                            q4::unpack<false>(W, v);
                            tc::st16(at, v);
                            q4::unpack<true>(W, v);
                            tc::st16(at + 16, v);
                        }
                    } else {
                        if (h == 0 && c >= VS) wait_bar(&vempty[sl], (c / VS - 1) & 1, a.status, bad);
                        uint8_t * to = sm + Ly::ring + sl * Ly::chunk + ((32 * wq) % Ly::vtok + lane) * 128;
#pragma unroll
                        for (int k = 0; k < Ly::HD / 64; k++) {
                            words(k);
                            if (none) {
#pragma unroll
                                for (int e = 0; e < 9; e++) W[e] = 0;
                            }
                            uint8_t * pl = to + (h * (Ly::HD / 64) + k) * (Ly::vtok * 128);
                            uint32_t  v[16];
                            auto      put = [&](int c0) {
#pragma unroll
                                for (int e = 0; e < 4; e++) {
                                    *reinterpret_cast<uint4 *>(pl + (((c0 + e) ^ (lane & 7)) << 4)) = make_uint4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
                                }
                            };
                            q4::unpack<false>(W, v);
                            put(0);
                            q4::unpack<true>(W, v);
                            put(4);
                        }
                    }
                    __syncwarp();
                    issue(st);
                    if (++st == ST) {
                        st = 0;
                        use++;
                    }
                }
                if (isk) {
                    tc::wait_st();
                    tc::fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&kfull[kb]);
                } else {
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&vfull[sl]);
                }
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        // a wait that gave up: the loads in flight land before this CTA's shared memory goes
        if (bad && a.box) {
            for (int s = 0; s < ST; s++) mbar_wait(&rf[s], (use + (s < st)) & 1);
        }
    }
    __syncwarp();
    tc::fence_before();
    __syncthreads();
    if (warp == kSm) tc::tmem_free(tb, 512);
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
                        : launch_t<D, 128, false>(ctx, a, mk, mv, k, v, stream);
}

}  // namespace

int fap::q4_rows(int T, int S, int G, bool f32) {
    const int64_t R = (int64_t) T * G;
    if (R <= (int64_t) S * 8) return 8;
    if (R <= (int64_t) S * 16) return 16;
    if (f32 || R <= (int64_t) S * 64) return 64;
    return 128;
}

int fap::q4_parts(int rows, int D) { return rows == 8 ? (D == 256 ? 8 : 16) : 1; }

int fap::q4_run(srhpm_ctx * ctx, PArgs & a, const PagedCache & c, int rows, bool f32, cudaStream_t stream) {
    const Pool4 k{ c.k, c.knb1, c.knb2, c.knb3 }, v{ c.v, c.vnb1, c.vnb2, c.vnb3 };
    CUtensorMap maps[2] = {}, &mk = maps[0], &mv = maps[1];
    // the few-row kernel takes whole rows of 256 values, this file's half a row at a time
    const int box = rows == 8 && c.D == 256 ? 144 : row_stride(c.D);
    // TMA takes the rows where a token's heads stand side by side and tokens and pages start on 16 bytes; other layouts come in
    // pieces by cp.async
    const int rowb = c.D / 16 * 9;
    auto      fits = [&](const Pool4 & p) {
        return (p.nb2 == rowb || c.Hkv == 1) && c.Hkv * rowb >= box && p.nb1 % 16 == 0 && p.nb3 % 16 == 0 &&
               reinterpret_cast<uintptr_t>(p.p) % 16 == 0 && p.nb1 >= (int64_t) c.Hkv * rowb;
    };
    a.box = 0;
    if (fits(k) && fits(v)) {
        a.box = c.page % 32 || (rows == 8 && c.D == 256) ? 16 : 32;  // a step of the few-row kernel has 16 tokens of 256 values
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
