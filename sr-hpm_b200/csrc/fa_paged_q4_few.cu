// Attention of a batch's new tokens over a paged cache of q4_0 rows, for the few rows per KV head of decoding steps
// (srhpm_flash_attn_paged; fa_paged_q4.cu has the rest).
//
// A row tile (8 rows of a sequence and KV head, packed token by token) fills a sixteenth of a 5th-generation tensor product, and
// what its unpacked operands and its tiles' hand-overs between warps cost is paid for every cached token. Here the numbers
// become f16 in registers and stay there, and no warp waits for another within an item: a warp multiplies 16 tokens x 16 dims by
// the 8 rows (mma.sync m16n8k16, f32 sums), with K as the left operand of S^T = K Q^T and V as that of O^T = V^T P^T.
//   operand order  A product's inner index may run in any order that both sides share, so no value moves between lanes: lane
//                  4 g + t takes, of the 36 bytes of a pair of blocks, word t of either block (K: tokens g and g + 8; V: word g of
//                  tokens 2 t, 2 t + 1, 2 t + 8, 2 t + 9), and Q is laid out once per item in the order in which K's lanes hold their dims
//   P^T            comes out of S^T with the rows along the columns; two 8 x 8 transpositions (movmatrix) per 16 tokens make
//                  it the right operand of the second product
//   softmax        the running maximum is raised only when a score exceeds it by 2^8, sums in f32; p is kept times 2^7 as f16.
//                  f32 rows (PREC): Q and P as sums of two f16 parts; a step's part of O is summed up apart and then added, as
//                  the tensor cores' sums are truncated (a shrink of 2^-25 per product, measured: 2e-5 after 400)
//
// Measured: 32 sequences of 500 to 8192 tokens decoding, 32 / 8 heads of 128: 69 us with the join, 2.6 TB/s: the schedulers issue in 63 %
// of their cycles, 1150 instructions per step of 32 tokens, 560 of them unpacking. One row over 30000 tokens, 24 / 4 heads of 256: 30 us,
// over 131000 68. One warp per 16 rows and whole CTAs on a part (tiles unpacked in shared memory) 91 us; heads that come to a token at
// different times 91.
//
// Work: the line of all items' units of TS tokens is cut into equal parts, one per warp: every warp is by itself from the plan on, with
// a ring that TMA fills (row boxes of 16-byte multiples, so that a row may start up to 12 bytes into its place; layouts that TMA
// does not take come by cp.async, 9 pieces of D / 16 bytes a row) and records of its own. Rows of 48, 80 and 144 bytes make
// every load from the ring free of bank conflicts.
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

#include "fa_paged.cuh"
#include "fastdiv.cuh"
#include "internal.h"
#include "launch.cuh"
#include "ptx.cuh"
#include "q4.cuh"
#include "ring.h"

namespace srhpm {
using namespace fap;
using namespace q4;
namespace {

template <int D, bool PREC> struct LayF {
    static constexpr int BM    = 8;                    // rows of a tile
    static constexpr int TS    = D == 256 ? 16 : 32;   // tokens of a step
    static constexpr int W     = D == 256 ? 8 : 16;    // warps: O takes D / 4 registers of a lane
    static constexpr int rowb  = D / 16 * 9;
    static constexpr int CB    = D / 16;               // bytes of a copy
    static constexpr int RS    = row_stride(D);
    static constexpr int stage = 2 * TS * RS;          // K rows, V rows
    static constexpr int parts = PREC ? 2 : 1;
    static constexpr int qset  = parts * (D / 32) * 512;              // of a warp: [parts][D / 32][32] uint4
    static constexpr int bar   = 0;
    static constexpr int misc  = W * 4 * 8;
    static constexpr int q     = (misc + 16 + 127) / 128 * 128;
    static constexpr int ring  = q + W * qset;
    static constexpr int room  = 232448 - ring;
    static constexpr int ST    = room / (W * stage) < 4 ? room / (W * stage) : 4;
    static constexpr int total = ring + ST * W * stage;
    static_assert(ST >= 2 && ring % 128 == 0 && ST * W * stage >= kMaxSeqs * 8, "shared memory");
};

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

// an item's steps in this warp: steps t0 + TS u, u = rot, rot + 1 .. n - 1, 0 .. rot - 1
struct Run {
    int t0, n, rot;
};
// Heads of one sequence stand side by side in the cache, a row of 36 to 144 bytes each, and memory gives 64 bytes at least: what one head
// leaves of them another should find in L2. So a warp begins its part where its step's number is a multiple of the parts'
// length, and all heads come to a token at about the same time.
template <int TS> __device__ __forceinline__ Run run_of(const Walk & w, int period) {
    Run r{ 0, 0, 0 };
    if (w.sp.nkv) {
        r.t0 = (w.sp.kt0 + w.off) * TS;
        r.n  = w.take;
        r.rot = (period - w.off % period) % period;
        if (r.rot >= r.n) r.rot = 0;
    }
    return r;
}

template <int D, bool PREC>
__global__ void __launch_bounds__(LayF<D, PREC>::W * 32, 1)
    fa_paged_q4_few_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv, const __grid_constant__ PArgs a,
                           const __grid_constant__ Pool4 kp, const __grid_constant__ Pool4 vp) {
    using Ly           = LayF<D, PREC>;  // a.box <= TS
    constexpr int BM   = Ly::BM;
    constexpr int TS   = Ly::TS;
    constexpr int W    = Ly::W;
    constexpr int ST   = Ly::ST;
    constexpr int MT   = TS / 16;
    constexpr int NG   = D / 64;
    constexpr int CB   = Ly::CB;
    constexpr int RS   = Ly::RS;
    constexpr int GP   = TS / 16;  // 16-token groups of a step
    constexpr int rowb = Ly::rowb;
    extern __shared__ __align__(128) uint8_t sm[];

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3, part = blockIdx.x * W + warp;
    uint64_t * full = reinterpret_cast<uint64_t *>(sm + Ly::bar) + warp * 4;
    if (lane == 0) {
        for (int i = 0; i < ST; i++) mbar_init(&full[i], a.box ? 1 : 32);
        fence_mbar_init();
    }
    if (tid == 0 && a.box) {
        prefetch_tmap(&mk);
        prefetch_tmap(&mv);
    }
    pdl_launch_dependents();
    pdl_wait();
    int * tot = reinterpret_cast<int *>(sm + Ly::ring);
    plan_sums<BM, TS, true>(a, tot, reinterpret_cast<int *>(sm + Ly::misc));
    const Part pt = plan_find<BM, TS>(a, tot, part, gridDim.x * W);
    __syncthreads();  // the ring is free; no warp waits for another from here on
    if (lane == 0) a.desc[2 * part] = make_int4(0, 0, 0, 0);
    if (pt.s < 0) return;
    const int period = (int) min((pt.all + pt.parts - 1) / pt.parts, (int64_t) 1 << 30);
    Walk w;
    w.s   = pt.s;
    w.h   = pt.h;
    w.rt  = pt.rt;
    w.off = pt.off;
    w.rem = w.part = pt.b1 - pt.b0;
    walk_load<BM>(a, w);
    walk_item<BM, TS>(a, w);

    // ---- this warp's copies, up to ST steps ahead of its products, across items ----
    Walk pw   = w;
    Run  prun = run_of<TS>(pw, period);
    int  pst  = 0;   // step of the item
    int  idle = -1;  // how often a load was asked for since there were no more (negative: there are more)
    // lane j: page of the 16-token group j % GP of the (j / GP)-th step from i0 on: asked for step by step, an entry's 700 cycles held
    // the warp up each time
    auto step_at = [](const Run & r, int i) { return r.t0 + (i + r.rot < r.n ? i + r.rot : i + r.rot - r.n) * TS; };
    int            ent = -1, i0 = 0;
    const uint32_t ring0 = smem_u32(sm + Ly::ring + warp * (ST * Ly::stage));
    auto           look  = [&](bool fresh) {
        fresh |= pst - i0 >= 32 / GP;
        while (idle < 0 && pst >= prun.n) {
            if (walk_next<BM, TS>(a, pw)) {
                prun  = run_of<TS>(pw, period);
                pst   = 0;
                fresh = true;
            } else {
                idle = 0;
            }
        }
        if (idle < 0 && fresh) {
            i0            = pst;
            ent           = -1;
            const int tok = step_at(prun, pst + lane / GP) + 16 * (lane % GP);
            if (pst + lane / GP < prun.n && tok < pw.sp.hi && tok + 16 > pw.sp.lo) {
                ent = reinterpret_cast<const int32_t *>(a.table + (int64_t) pw.s * a.tstride)[a.byPage.div(tok)];
                if (ent < 0 || ent >= a.n_pages) {  // no page: reads as zeros
                    atomicExch(a.status, kErrPage);
                    ent = a.n_pages;
                }
            }
        }
    };
    auto issue = [&](int stage) {
        if (idle >= 0) {
            idle++;
            return;
        }
        const uint32_t to = ring0 + stage * Ly::stage;
        const int      t0 = step_at(prun, pst), at = (pst - i0) * GP;
        int            p[GP], y[GP];  // page (-1: no row sees the group) and place
#pragma unroll
        for (int k = 0; k < GP; k++) {
            p[k] = __shfl_sync(0xffffffffu, ent, at + k);
            y[k] = t0 + 16 * k - a.byPage.div(t0 + 16 * k) * a.page;
        }
        if (a.box) {
            // boxes of 16 tokens, or of 32 where pages hold them; one that no row sees is left out
            const bool one = GP == 2 && a.box == 32;
            const bool b0 = p[0] >= 0 || (one && p[GP - 1] >= 0), b1 = GP == 2 && !one && p[GP - 1] >= 0;
            if (elect_one()) {
                const int x = (pw.h * rowb) & ~15;
                mbar_arrive_expect_tx(&full[stage], (b0 + b1) * a.box * RS * 2);
                if (b0) {
                    const int z = one ? max(p[0], p[GP - 1]) : p[0];
                    tma_rows(to, &mk, x, y[0], z, &full[stage]);
                    tma_rows(to + TS * RS, &mv, x, y[0], z, &full[stage]);
                }
                if (b1) {
                    tma_rows(to + 16 * RS, &mk, x, y[GP - 1], p[GP - 1], &full[stage]);
                    tma_rows(to + (TS + 16) * RS, &mv, x, y[GP - 1], p[GP - 1], &full[stage]);
                }
            }
            __syncwarp();
        } else {
#pragma unroll 1
            for (int k = 0; k < TS * 9; k += 32) {
                const int idx = k + lane, tk = idx / 9, ch = idx - 9 * tk;
                if (idx < TS * 9) {
                    const int     pg = tk < 16 ? p[0] : p[GP - 1], yy = (tk < 16 ? y[0] : y[GP - 1]) + (tk & 15);
                    const bool    ok = pg >= 0 && pg < a.n_pages;
                    const int64_t ko = ok ? pg * kp.nb3 + yy * kp.nb1 + pw.h * kp.nb2 + ch * CB : 0, vo = ok ? pg * vp.nb3 + yy * vp.nb1 + pw.h * vp.nb2 + ch * CB : 0;
                    q4::copy_async<CB>(to + tk * RS + ch * CB, kp.p + ko, ok ? CB : 0);
                    q4::copy_async<CB>(to + (TS + tk) * RS + ch * CB, vp.p + vo, ok ? CB : 0);
                }
            }
            asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&full[stage])) : "memory");
        }
        pst++;
        look(false);
    };
    look(true);
    for (int s = 0; s < ST; s++) issue(s);

    const uint32_t selv = g == 3 ? 0x1076u : 0x3210u, selk = t == 3 ? 0x1076u : 0x3210u, seld = g < 4 ? 0x5410u : 0x7632u;
    int            stage = 0, use = 0;
    for (bool active = true; active;) {
        const int n  = w.n * a.G, rb = w.rt * BM, rows = min(BM, n - rb);
        const Run run = run_of<TS>(w, period);
        // ---- Q, in the order of K's lanes; rows that are none as zeros ----
        uint4 * qb = reinterpret_cast<uint4 *>(sm + Ly::q + warp * Ly::qset);
#pragma unroll 2
        for (int blk = 0; blk < D / 32; blk++) {
            const int u = 32 * blk + lane, row = g, tt = t;
            float     x[8];
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = 0.0f;
            if (row < rows) {
                const int       tok = a.byG.div(rb + row), h = w.h * a.G + (rb + row - tok * a.G);
                const uint8_t * src = a.q + (int64_t) (w.r0 + tok) * a.qnb1 + (int64_t) h * a.qnb2;
#pragma unroll
                for (int e = 0; e < 8; e++) {  // pairs (0, 2), (1, 3) of the low, then of the high halves
                    const int b = (e & 1) * 2 + ((e >> 1) & 1), d = 32 * blk + q4::byte_of(blk & 1, tt, b) + 16 * (e >> 2);
                    x[e] = PREC ? reinterpret_cast<const float *>(src)[d] : __half2float(reinterpret_cast<const __half *>(src)[d]);
                }
            }
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const __half2 h2 = __floats2half2_rn(x[2 * e], x[2 * e + 1]);
                const __half2 l2 = __floats2half2_rn(x[2 * e] - __low2float(h2), x[2 * e + 1] - __high2float(h2));
                hi[e] = *reinterpret_cast<const uint32_t *>(&h2);
                lo[e] = *reinterpret_cast<const uint32_t *>(&l2);
            }
            qb[u] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            if constexpr (PREC) qb[(D / 32) * 32 + u] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
        // ---- what this lane's rows see ----
        int   vlo[2], vhi[2];
        float m[2], l[2];
        float o[NG][4][4];
        int   alo = 0, ahi = INT32_MAX;  // seen by every row
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const int  row = 2 * t + k;
            const bool is  = row < rows;
            const int  pos = w.kv - w.n + a.byG.div(rb + (is ? row : 0));
            vhi[k]         = is ? min(pos + 1, w.sp.hi) : 0;
            vlo[k]         = a.window > 0 ? max(w.sp.lo, (int) max((int64_t) INT32_MIN, (int64_t) pos - a.window + 1)) : w.sp.lo;
            if (is) {
                alo = max(alo, vlo[k]);
                ahi = min(ahi, vhi[k]);
            }
            m[k] = -INFINITY;
            l[k] = 0.0f;
        }
        alo = __reduce_max_sync(0xffffffffu, alo);
        ahi = __reduce_min_sync(0xffffffffu, ahi);
#pragma unroll
        for (int i = 0; i < NG; i++) {
#pragma unroll
            for (int b = 0; b < 4; b++) {
#pragma unroll
                for (int e = 0; e < 4; e++) o[i][b][e] = 0.0f;
            }
        }
        __syncwarp();
        const uint4 * ql   = qb + lane;
        const int     lead = a.box ? (w.h * rowb) & 15 : 0;
        for (int st = 0; st < run.n; st++) {
            uint32_t i = 0;
            while (i < kProbes && !mbar_try_wait(&full[stage], use & 1)) i++;
            if (__any_sync(0xffffffffu, i == kProbes)) {
                // The warp gives up as one and asks for nothing more; its results are void. Its loads in flight land before the
                // CTA's shared memory goes.
                if (lane == 0) atomicExch(a.status, kErrWaitFull);
                const uint32_t done = use * ST + stage, issued = ring_issued(done, ST, idle);
                for (uint32_t c = done; c < issued; c++) mbar_wait(&full[ring_slot(c, ST)], ring_parity(c, ST));
                return;
            }
            const uint8_t * kr = sm + Ly::ring + warp * (ST * Ly::stage) + stage * Ly::stage + lead;
            const uint8_t * vr = kr + TS * RS;
            const int       tb   = step_at(run, st);
            const bool      mask = tb < alo || tb + TS > ahi;
            float           s[MT][4];
#pragma unroll
            for (int i = 0; i < MT; i++) {
#pragma unroll
                for (int e = 0; e < 4; e++) s[i][e] = 0.0f;
            }
#pragma unroll
            for (int bp = 0; bp < NG; bp++) {
#pragma unroll
                for (int i = 0; i < MT; i++) {
                    uint32_t p[2][2][4];  // token, block, pairs
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        const uint32_t * row = reinterpret_cast<const uint32_t *>(kr + (16 * i + g + 8 * k) * RS + 36 * bp);
                        const uint32_t   y0 = row[0], y1 = row[4], z = row[5 + t];
                        const uint32_t   x = q4::prmt(row[1 + t], y0, selk);
                        const uint32_t   d0 = q4::prmt(y0, y0, 0x1010u), d1 = q4::prmt(y1, y1, 0x3232u);
                        p[k][0][0] = q4::low4(x, d0);
                        p[k][0][1] = q4::low4(x >> 8, d0);
                        p[k][0][2] = q4::high4(x, d0);
                        p[k][0][3] = q4::high4(x >> 8, d0);
                        p[k][1][0] = q4::low4(z, d1);
                        p[k][1][1] = q4::low4(z >> 8, d1);
                        p[k][1][2] = q4::high4(z, d1);
                        p[k][1][3] = q4::high4(z >> 8, d1);
                    }
#pragma unroll
                    for (int b = 0; b < 2; b++) {
#pragma unroll
                        for (int pr = 0; pr < Ly::parts; pr++) {
                            const uint4 qv = ql[(pr * (D / 32) + 2 * bp + b) * 32];
                            mma16816(s[i], p[0][b][0], p[1][b][0], p[0][b][1], p[1][b][1], qv.x, qv.y);
                            mma16816(s[i], p[0][b][2], p[1][b][2], p[0][b][3], p[1][b][3], qv.z, qv.w);
                        }
                    }
                }
            }
            // ---- softmax: this lane has tokens g, g + 8 of every 16 and rows 2 t, 2 t + 1 ----
            float mx[2] = { -INFINITY, -INFINITY };
#pragma unroll
            for (int i = 0; i < MT; i++) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float x = s[i][e] * a.qscale;
                    if (a.softcap_l2 != 0.0f) x = a.softcap_l2 * tanhf(x);
                    if (mask) {
                        const int pos = tb + 16 * i + g + (e >> 1) * 8;
                        x             = pos >= vlo[e & 1] && pos < vhi[e & 1] ? x : -INFINITY;
                    }
                    s[i][e]   = x;
                    mx[e & 1] = fmaxf(mx[e & 1], x);
                }
            }
            if (__any_sync(0xffffffffu, mx[0] > m[0] + kLazy || mx[1] > m[1] + kLazy)) {
                float f[2];
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    float x = mx[k];
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
                    f[k] = 1.0f;
                    if (x > m[k] + kLazy) {
                        f[k] = exp2a(m[k] - x);
                        m[k] = x;
                    }
                    l[k] *= f[k];
                }
#pragma unroll
                for (int i = 0; i < NG; i++) {
#pragma unroll
                    for (int b = 0; b < 4; b++) {
#pragma unroll
                        for (int e = 0; e < 4; e++) o[i][b][e] *= f[e & 1];
                    }
                }
            }
            uint32_t ph[MT][2];
            [[maybe_unused]] uint32_t pl[MT][2];
            const float o0 = (m[0] == -INFINITY ? 0.0f : m[0]) - kShift, o1 = (m[1] == -INFINITY ? 0.0f : m[1]) - kShift;
#pragma unroll
            for (int i = 0; i < MT; i++) {
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const float x0 = exp2a(s[i][2 * k] - o0), x1 = exp2a(s[i][2 * k + 1] - o1);
                    l[0] += x0;
                    l[1] += x1;
                    const __half2 h2 = __floats2half2_rn(x0, x1);
                    ph[i][k]         = transpose8(*reinterpret_cast<const uint32_t *>(&h2));
                    if constexpr (PREC) {
                        const __half2 r2 = __floats2half2_rn(x0 - __low2float(h2), x1 - __high2float(h2));
                        pl[i][k]         = transpose8(*reinterpret_cast<const uint32_t *>(&r2));
                    }
                }
            }
            // tokens of the step that no row sees hold anything; 0 * NaN is NaN, so their V rows become zeros
            const bool edge = tb < w.sp.lo || tb + TS > w.sp.hi;
#pragma unroll
            for (int gq = 0; gq < NG; gq++) {
                [[maybe_unused]] float part_o[4][4];
                if constexpr (PREC) {
#pragma unroll
                    for (int b = 0; b < 4; b++) part_o[b][0] = part_o[b][1] = part_o[b][2] = part_o[b][3] = 0.0f;
                }
#pragma unroll
                for (int i = 0; i < MT; i++) {
                    uint32_t v[4], y[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const int        tk  = 16 * i + 2 * t + (k & 1) + 8 * (k >> 1);
                        const uint32_t * row = reinterpret_cast<const uint32_t *>(vr + tk * RS + 36 * gq);
                        y[k]                 = row[g < 4 ? 0 : 4];
                        v[k]                 = q4::prmt(row[1 + g], y[k], selv);
                    }
                    if (edge) {
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const int tok = tb + 16 * i + 2 * t + (k & 1) + 8 * (k >> 1);
                            if (tok < w.sp.lo || tok >= w.sp.hi) y[k] = v[k] = 0;
                        }
                    }
                    const uint32_t d0 = q4::prmt(y[0], y[1], seld), d1 = q4::prmt(y[2], y[3], seld);
#pragma unroll
                    for (int b = 0; b < 4; b++) {
                        const uint32_t sel = 0x4400u + 0x1111u * b, x0 = q4::prmt(v[0], v[1], sel), x1 = q4::prmt(v[2], v[3], sel);
                        const uint32_t a0 = q4::low4(x0, d0), a1 = q4::high4(x0, d0), a2 = q4::low4(x1, d1), a3 = q4::high4(x1, d1);
                        if constexpr (PREC) {
                            mma16816(part_o[b], a0, a1, a2, a3, ph[i][0], ph[i][1]);
                            mma16816(part_o[b], a0, a1, a2, a3, pl[i][0], pl[i][1]);
                        } else {
                            mma16816(o[gq][b], a0, a1, a2, a3, ph[i][0], ph[i][1]);
                        }
                    }
                }
                if constexpr (PREC) {
#pragma unroll
                    for (int b = 0; b < 4; b++) {
#pragma unroll
                        for (int e = 0; e < 4; e++) o[gq][b][e] += part_o[b][e];
                    }
                }
            }
            __syncwarp();
            issue(stage);
            if (++stage == ST) {
                stage = 0;
                use++;
            }
        }
        // ---- the item's end: a lane has rows 2 t, 2 t + 1, of each pair of blocks the numbers of its word ----
        const bool whole = w.off == 0 && w.take == w.sp.units;
        const int  slot  = 2 * part + (w.off == 0 ? 1 : 0);
#pragma unroll
        for (int k = 0; k < 2; k++) {
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) l[k] += __shfl_xor_sync(0xffffffffu, l[k], d);
            const int row = 2 * t + k;
            if (row >= rows) continue;
            const int tok = a.byG.div(rb + row), h = w.h * a.G + (rb + row - tok * a.G);
            float     f   = 1.0f;
            if (whole) {
                float L = l[k];
                if (a.sinks) {  // relative to the larger of the two maxima
                    const float sk = a.sinks[h] * kLog2e;
                    if (sk > m[k]) {
                        f = m[k] == -INFINITY ? 0.0f : exp2a(m[k] - sk);
                        L = L * f + exp2f(kShift);
                    } else if (sk > -INFINITY) {
                        L += exp2a(sk - m[k] + kShift);
                    }
                }
                f = L == 0.0f ? 0.0f : f / L;  // a NaN stays one
            } else if (g == 0) {
                a.part_ms[(int64_t) slot * a.prow + row] = make_float2(m[k], l[k]);
            }
            uint8_t * dst = a.dst + (int64_t) h * a.dnb1 + (int64_t) (w.r0 + tok) * a.dnb2;
            float *   acc = a.part_acc + ((int64_t) slot * a.prow + row) * D;
#pragma unroll
            for (int gq = 0; gq < NG; gq++) {
#pragma unroll
                for (int b = 0; b < 4; b += 2) {
#pragma unroll
                    for (int hi = 0; hi < 2; hi++) {
                        const int d = 64 * gq + 32 * (g >> 2) + q4::byte_of(g >= 4, g & 3, b) + 16 * hi;
                        float2    x = make_float2(o[gq][b][2 * hi + k], o[gq][b + 1][2 * hi + k]);
                        if (!whole) {
                            *reinterpret_cast<float2 *>(acc + d) = x;
                            continue;
                        }
                        x = f != 0.0f ? make_float2(x.x * f, x.y * f) : make_float2(0.0f, 0.0f);
                        if constexpr (PREC) {
                            *reinterpret_cast<float2 *>(dst + 4 * d) = x;
                        } else {
                            *reinterpret_cast<__half2 *>(dst + 2 * d) = __floats2half2_rn(x.x, x.y);
                        }
                    }
                }
            }
        }
        if (lane == 0 && !whole && w.off == 0) {
            // this warp opens an item that others go on with: parts of it, for the join
            const int64_t end = pt.b0 + (pt.b1 - pt.b0 - w.rem) + w.sp.units;
            const int     e   = part_of_end(pt.all, pt.parts, end, part);
            a.desc[2 * part + 1] = make_int4(rb, rows, 0, 0);
            a.desc[2 * part]     = make_int4(e - part + 1, w.h, w.r0, 0);
        }
        __syncwarp();  // Q is read
        active = walk_next<BM, TS>(a, w);
    }
}

template <int D, bool PREC>
int launch_few(srhpm_ctx * ctx, const PArgs & a, const CUtensorMap & mk, const CUtensorMap & mv, const Pool4 & k, const Pool4 & v,
               cudaStream_t stream) {
    using Ly = LayF<D, PREC>;
    auto                         kern = fa_paged_q4_few_kernel<D, PREC>;
    static std::atomic<unsigned> done{ 0 };
    const unsigned               bit = 1u << (ctx->device & 31);
    if (!(done.load() & bit)) {
        const int st = cuda_status(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Ly::total));
        if (st != SRHPM_OK) return st;
        done.fetch_or(bit);
    }
    const int st = cuda_status(launch_k_pdl(kern, dim3(ctx->num_sms), dim3(Ly::W * 32), Ly::total, stream, mk, mv, a, k, v));
    ctx->launches.fetch_add(1);
    if (st != SRHPM_OK) return st;
    return merge_launch(ctx, a, D, PREC, std::min(8, a.prow), stream, Ly::W);
}

}  // namespace

int fap::q4_few_run(srhpm_ctx * ctx, const PArgs & a, const void * maps, const PagedCache & c, bool f32, cudaStream_t stream) {
    const Pool4 k{ c.k, c.knb1, c.knb2, c.knb3 }, v{ c.v, c.vnb1, c.vnb2, c.vnb3 };
    const CUtensorMap & mk = static_cast<const CUtensorMap *>(maps)[0], & mv = static_cast<const CUtensorMap *>(maps)[1];
    if (c.D == 64) return f32 ? launch_few<64, true>(ctx, a, mk, mv, k, v, stream) : launch_few<64, false>(ctx, a, mk, mv, k, v, stream);
    if (c.D == 128) return f32 ? launch_few<128, true>(ctx, a, mk, mv, k, v, stream) : launch_few<128, false>(ctx, a, mk, mv, k, v, stream);
    return f32 ? launch_few<256, true>(ctx, a, mk, mv, k, v, stream) : launch_few<256, false>(ctx, a, mk, mv, k, v, stream);
}

}  // namespace srhpm
