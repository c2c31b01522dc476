// Attention of a batch's new tokens over a paged cache of q4_0 rows, for the few rows per KV head of decoding steps
// (srhpm_flash_attn_paged).
//
// A row tile (8 NT rows of a sequence and KV head, packed token by token) fills an eighth or less of a 5th-generation tensor
// product, and 4-bit values would have to go through shared memory as f16 to reach one: four times the cache's bytes in
// writes and as much again in reads. Here the numbers become f16 in registers and stay there: a warp multiplies 16 tokens x
// 16 dims by 8 rows (mma.sync m16n8k16, f32 sums), with K as the left operand of S^T = K Q^T and V as that of O^T = V^T P^T.
//   operand order  A product's inner index may run in any order that both sides share, so no value moves between lanes: lane
//                  4 g + t takes, of the 36 bytes of a pair of blocks, word t of either block (K: token g; V: token 4 t + i,
//                  word g), and Q is laid out once per item in the order in which K's lanes hold their dims
//   numbers        (w & 0x000f000f) | 0x64006400 is the f16 pair 1024 + q; minus 1032 it is q - 8, exactly; the high halves
//                  of the bytes come as 1024 + 16 q and go through x / 16 - 72, exactly. Then one product with d, rounded: the
//                  cache's value
//   P^T            comes out of S^T with the rows along the columns; two 8 x 8 transpositions (movmatrix) per 16 tokens make
//                  it the right operand of the second product
//   softmax        the running maximum is raised only when a score exceeds it by 2^8, sums in f32; p is kept times 2^7 as f16
//
// Work: the line of all items' units is cut into equal parts, one per CTA (plan_part). The CTA's warps share an item's steps
// of TS tokens out, every W-th each, with rings of their own that cp.async fills (no barrier in the loop): 9 pieces of D / 16
// bytes make a row, whatever its strides are. At an item's end the warps' sums are joined in shared memory.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

#include "fa_paged.cuh"
#include "fastdiv.cuh"
#include "internal.h"
#include "launch.cuh"
#include "ptx.cuh"

namespace srhpm {
using namespace fap;
namespace {

constexpr int kUnit = 128;  // tokens of a unit of work

struct Pool4 {
    const uint8_t * p;
    int64_t         nb1, nb2, nb3;
};

template <int D, int NT, bool PREC> struct LayF {
    static constexpr int BM    = 8 * NT;               // rows of a tile
    static constexpr int TS    = D == 256 ? 16 : 32;   // tokens of a step
    static constexpr int W     = D * NT > 128 ? 8 : 16;  // warps: O takes D NT / 4 registers of a lane
    static constexpr int rowb  = D / 16 * 9;
    static constexpr int CB    = D / 16;               // bytes of a copy
    static constexpr int stage = 2 * TS * rowb;        // K rows, V rows
    static constexpr int parts = PREC ? 2 : 1;
    static constexpr int pad   = D + 4;
    static constexpr int q     = 0;                                   // [2][parts][D / 32][NT][32] uint4
    static constexpr int qset  = parts * (D / 32) * NT * 512;
    static constexpr int part  = q + 2 * qset;                        // f32 [W][BM][pad]
    static constexpr int ms    = part + W * BM * pad * 4;             // float2 [W][BM]
    static constexpr int misc  = ms + W * BM * 8;
    static constexpr int ring  = misc + 64;
    static constexpr int room  = 232448 - ring;
    static constexpr int ST    = room / (W * stage) < 4 ? room / (W * stage) : 4;
    static constexpr int total = ring + ST * W * stage;
    static_assert(ST >= 2 && ring % 16 == 0 && ST * W * stage >= kMaxSeqs * 8, "shared memory");
};

template <int N> __device__ __forceinline__ void copy_async(uint32_t dst, const uint8_t * src, uint32_t size) {
    if constexpr (N == 16) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(size) : "memory");
    } else {
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(size) : "memory");
    }
}

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
    uint32_t r;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
    return r;
}
template <uint32_t MASK> __device__ __forceinline__ uint32_t magic(uint32_t x) {  // (x & MASK) | 0x64006400
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(x), "n"(MASK), "r"(0x64006400u));
    return r;
}
__device__ __forceinline__ uint32_t low4(uint32_t x, uint32_t dd) {  // bits 0..3 of either half -> d (q - 8)
    const uint32_t m = magic<0x000f000fu>(x);
    __half2        h = __hsub2(*reinterpret_cast<const __half2 *>(&m), __floats2half2_rn(1032.0f, 1032.0f));
    h                = __hmul2(h, *reinterpret_cast<const __half2 *>(&dd));
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t high4(uint32_t x, uint32_t dd) {  // bits 4..7
    const uint32_t m = magic<0x00f000f0u>(x);
    __half2        h = __hfma2(*reinterpret_cast<const __half2 *>(&m), __floats2half2_rn(0.0625f, 0.0625f), __floats2half2_rn(-72.0f, -72.0f));
    h                = __hmul2(h, *reinterpret_cast<const __half2 *>(&dd));
    return *reinterpret_cast<const uint32_t *>(&h);
}

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
__device__ __forceinline__ float exp2a(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// byte of a block's 16 that byte b of word w is: word 3 of an even block is made of the bytes around its others (the first
// block of a pair starts 2 bytes off the words)
__device__ __forceinline__ int byte_of(bool odd, int w, int b) { return odd ? 4 * w + b : w < 3 ? 2 + 4 * w + b : b < 2 ? b : 12 + b; }

// an item's tokens in this CTA
struct Run {
    int t0, n;  // first token (a multiple of TS), steps
};
template <int TS> __device__ __forceinline__ Run run_of(const Walk & w) {
    Run r{ 0, 0 };
    if (w.sp.nkv) {
        const int b = (w.sp.kt0 + w.off) * kUnit;
        const int e = min(b + w.take * kUnit, w.sp.hi);
        r.t0        = max(b, w.sp.lo) & ~(TS - 1);
        r.n         = (e - r.t0 + TS - 1) / TS;
    }
    return r;
}

template <int D, int NT, bool PREC>
__global__ void __launch_bounds__(LayF<D, NT, PREC>::W * 32, 1)
    fa_paged_q4_few_kernel(const __grid_constant__ PArgs a, const __grid_constant__ Pool4 kp, const __grid_constant__ Pool4 vp) {
    using Ly           = LayF<D, NT, PREC>;
    constexpr int BM   = Ly::BM;
    constexpr int TS   = Ly::TS;
    constexpr int W    = Ly::W;
    constexpr int ST   = Ly::ST;
    constexpr int MT   = TS / 16;
    constexpr int NG   = D / 64;
    constexpr int CB   = Ly::CB;
    constexpr int NI   = (TS * 9 + 31) / 32;
    constexpr int rowb = Ly::rowb;
    extern __shared__ __align__(16) uint8_t sm[];
    float *   part  = reinterpret_cast<float *>(sm + Ly::part);
    float2 *  ms    = reinterpret_cast<float2 *>(sm + Ly::ms);
    int *     first = reinterpret_cast<int *>(sm + Ly::misc);
    int64_t * range = reinterpret_cast<int64_t *>(sm + Ly::misc + 16);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    if (tid == 0) first[0] = -1;
    pdl_launch_dependents();
    pdl_wait();
    plan_part<BM, kUnit>(a, reinterpret_cast<int *>(sm + Ly::ring), reinterpret_cast<int *>(sm + Ly::ms), first, range);
    __syncthreads();
    if (tid == 0) a.desc[2 * blockIdx.x] = make_int4(0, 0, 0, 0);
    Walk w;
    w.s = first[0];
    if (w.s < 0) return;
    w.h   = first[1];
    w.rt  = first[2];
    w.off = first[3];
    w.rem = w.part = range[1] - range[0];
    walk_load<BM>(a, w);
    walk_item<BM, kUnit>(a, w);

    // ---- this warp's copies, up to ST steps ahead of its products, across items ----
    Walk      pw   = w;
    Run       prun = run_of<TS>(pw);
    int       pst  = warp;
    bool      pact = true;
    int       pg = -1, pin = 0;  // lane = token of the step to come: its page (-1: nobody sees it) and place
    const uint32_t ring0 = smem_u32(sm + Ly::ring + warp * (ST * Ly::stage));
    auto           look  = [&]() {
        while (pact && pst >= prun.n) {
            pact = walk_next<BM, kUnit>(a, pw);
            if (pact) {
                prun = run_of<TS>(pw);
                pst  = warp;
            }
        }
        pg = -1;
        if (pact && lane < TS) {
            const int tok = prun.t0 + pst * TS + lane;
            if (tok >= pw.sp.lo && tok < pw.sp.hi) {
                const int pi = a.byPage.div(tok);
                pin          = tok - pi * a.page;
                pg           = reinterpret_cast<const int32_t *>(a.table + (int64_t) pw.s * a.tstride)[pi];
                if (pg < 0 || pg >= a.n_pages) {  // no page: reads as zeros
                    atomicExch(a.status, kErrPage);
                    pg = -1;
                }
            }
        }
    };
    auto issue = [&](int stage) {
        if (pact) {
            const int64_t ko = pg < 0 ? -1 : pg * kp.nb3 + pin * kp.nb1 + pw.h * kp.nb2;
            const int64_t vo = pg < 0 ? -1 : pg * vp.nb3 + pin * vp.nb1 + pw.h * vp.nb2;
            const uint32_t to = ring0 + stage * Ly::stage;
#pragma unroll
            for (int i = 0; i < NI; i++) {
                const int     idx = i * 32 + lane, tk = idx / 9, ch = idx - 9 * tk;
                const int64_t ks = __shfl_sync(0xffffffffu, ko, tk & (TS - 1)), vs = __shfl_sync(0xffffffffu, vo, tk & (TS - 1));
                if (idx < TS * 9) {
                    copy_async<CB>(to + idx * CB, kp.p + (ks < 0 ? 0 : ks + ch * CB), ks < 0 ? 0 : CB);
                    copy_async<CB>(to + TS * rowb + idx * CB, vp.p + (vs < 0 ? 0 : vs + ch * CB), vs < 0 ? 0 : CB);
                }
            }
            pst += W;
            look();
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    look();
    for (int s = 0; s < ST; s++) issue(s);

    const uint32_t selv = g == 3 ? 0x1076u : 0x3210u, selk = t == 3 ? 0x1076u : 0x3210u, seld = g < 4 ? 0x5410u : 0x7632u;
    const uint32_t tmask = 4 * (g >> 1) + (g & 1);  // token of this lane's first score of 16; the second is 2 behind it
    int            stage = 0, par = 0;
    for (bool active = true; active; par ^= 1) {
        const int n  = w.n * a.G, rb = w.rt * BM, rows = min(BM, n - rb);
        const Run run = run_of<TS>(w);
        // ---- Q, in the order of K's lanes; rows that are none as zeros ----
        uint4 * qb = reinterpret_cast<uint4 *>(sm + Ly::q + par * Ly::qset);
        for (int u = tid; u < (D / 32) * NT * 32; u += W * 32) {
            const int ln = u & 31, nt = (u >> 5) % NT, blk = (u >> 5) / NT, row = 8 * nt + (ln >> 2), tt = ln & 3;
            float     x[8];
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = 0.0f;
            if (row < rows) {
                const int       tok = a.byG.div(rb + row), h = w.h * a.G + (rb + row - tok * a.G);
                const uint8_t * src = a.q + (int64_t) (w.r0 + tok) * a.qnb1 + (int64_t) h * a.qnb2;
#pragma unroll
                for (int e = 0; e < 8; e++) {  // pairs (0, 2), (1, 3) of the low, then of the high halves
                    const int b = (e & 1) * 2 + ((e >> 1) & 1), d = 32 * blk + byte_of(blk & 1, tt, b) + 16 * (e >> 2);
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
            if constexpr (PREC) qb[(D / 32) * NT * 32 + u] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
        // ---- what this lane's rows see ----
        int   vlo[NT][2], vhi[NT][2];
        float m[NT][2], l[NT][2];
        float o[NG][4][NT][4];
        int   alo = 0, ahi = INT32_MAX;  // seen by every row
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const int  row = 8 * nt + 2 * t + k;
                const bool is  = row < rows;
                const int  pos = w.kv - w.n + a.byG.div(rb + (is ? row : 0));
                vhi[nt][k]     = is ? min(pos + 1, w.sp.hi) : 0;
                vlo[nt][k]     = a.window > 0 ? max(w.sp.lo, (int) max((int64_t) INT32_MIN, (int64_t) pos - a.window + 1)) : w.sp.lo;
                if (is) {
                    alo = max(alo, vlo[nt][k]);
                    ahi = min(ahi, vhi[nt][k]);
                }
                m[nt][k]       = -INFINITY;
                l[nt][k]       = 0.0f;
            }
        }
        alo = __reduce_max_sync(0xffffffffu, alo);
        ahi = __reduce_min_sync(0xffffffffu, ahi);
#pragma unroll
        for (int i = 0; i < NG; i++) {
#pragma unroll
            for (int b = 0; b < 4; b++) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                    for (int e = 0; e < 4; e++) o[i][b][nt][e] = 0.0f;
                }
            }
        }
        __syncthreads();
        const uint4 * ql = qb + lane;
        for (int st = warp; st < run.n; st += W) {
            asm volatile("cp.async.wait_group %0;" ::"n"(ST - 1) : "memory");
            __syncwarp();
            const uint8_t * kr = sm + Ly::ring + warp * (ST * Ly::stage) + stage * Ly::stage;
            const uint8_t * vr = kr + TS * rowb;
            float           s[MT][NT][4];
#pragma unroll
            for (int i = 0; i < MT; i++) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                    for (int e = 0; e < 4; e++) s[i][nt][e] = 0.0f;
                }
            }
#pragma unroll
            for (int bp = 0; bp < NG; bp++) {
#pragma unroll
                for (int i = 0; i < MT; i++) {
                    uint32_t p[2][2][4];  // token, block, pairs
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        const uint32_t * row = reinterpret_cast<const uint32_t *>(kr + (16 * i + tmask + 2 * k) * rowb + 36 * bp);
                        const uint32_t   y0 = row[0], y1 = row[4], z = row[5 + t];
                        const uint32_t   x = prmt(row[1 + t], y0, selk);
                        const uint32_t   d0 = prmt(y0, y0, 0x1010u), d1 = prmt(y1, y1, 0x3232u);
                        p[k][0][0] = low4(x, d0);
                        p[k][0][1] = low4(x >> 8, d0);
                        p[k][0][2] = high4(x, d0);
                        p[k][0][3] = high4(x >> 8, d0);
                        p[k][1][0] = low4(z, d1);
                        p[k][1][1] = low4(z >> 8, d1);
                        p[k][1][2] = high4(z, d1);
                        p[k][1][3] = high4(z >> 8, d1);
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                        for (int b = 0; b < 2; b++) {
#pragma unroll
                            for (int pr = 0; pr < Ly::parts; pr++) {
                                const uint4 qv = ql[((pr * (D / 32) + 2 * bp + b) * NT + nt) * 32];
                                mma16816(s[i][nt], p[0][b][0], p[1][b][0], p[0][b][1], p[1][b][1], qv.x, qv.y);
                                mma16816(s[i][nt], p[0][b][2], p[1][b][2], p[0][b][3], p[1][b][3], qv.z, qv.w);
                            }
                        }
                    }
                }
            }
            // ---- softmax: this lane has tokens tmask, tmask + 2 of every 16 and rows 2 t, 2 t + 1 of every 8 ----
            const int  tb   = run.t0 + st * TS;
            const bool mask = tb < alo || tb + TS > ahi;
            const float qs  = a.qscale;
            float      mx[NT][2];
            bool       up = false;
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                mx[nt][0] = mx[nt][1] = -INFINITY;
#pragma unroll
                for (int i = 0; i < MT; i++) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        float x = s[i][nt][e] * qs;
                        if (a.softcap_l2 != 0.0f) x = a.softcap_l2 * tanhf(x);
                        if (mask) {
                            const int pos = tb + 16 * i + (int) tmask + (e >> 1) * 2;
                            x             = pos >= vlo[nt][e & 1] && pos < vhi[nt][e & 1] ? x : -INFINITY;
                        }
                        s[i][nt][e]   = x;
                        mx[nt][e & 1] = fmaxf(mx[nt][e & 1], x);
                    }
                }
                up |= mx[nt][0] > m[nt][0] + kLazy || mx[nt][1] > m[nt][1] + kLazy;
            }
            if (__any_sync(0xffffffffu, up)) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    float f[2];
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        float x = mx[nt][k];
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
                        f[k] = 1.0f;
                        if (x > m[nt][k] + kLazy) {
                            f[k]     = exp2a(m[nt][k] - x);
                            m[nt][k] = x;
                        }
                        l[nt][k] *= f[k];
                    }
#pragma unroll
                    for (int i = 0; i < NG; i++) {
#pragma unroll
                        for (int b = 0; b < 4; b++) {
#pragma unroll
                            for (int e = 0; e < 4; e++) o[i][b][nt][e] *= f[e & 1];
                        }
                    }
                }
            }
            uint32_t ph[MT][NT][2];
            [[maybe_unused]] uint32_t pl[MT][NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                const float o0 = (m[nt][0] == -INFINITY ? 0.0f : m[nt][0]) - kShift, o1 = (m[nt][1] == -INFINITY ? 0.0f : m[nt][1]) - kShift;
#pragma unroll
                for (int i = 0; i < MT; i++) {
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        const float x0 = exp2a(s[i][nt][2 * k] - o0), x1 = exp2a(s[i][nt][2 * k + 1] - o1);
                        l[nt][0] += x0;
                        l[nt][1] += x1;
                        const __half2 h2 = __floats2half2_rn(x0, x1);
                        ph[i][nt][k]     = transpose8(*reinterpret_cast<const uint32_t *>(&h2));
                        if constexpr (PREC) {
                            const __half2 r2 = __floats2half2_rn(x0 - __low2float(h2), x1 - __high2float(h2));
                            pl[i][nt][k]     = transpose8(*reinterpret_cast<const uint32_t *>(&r2));
                        }
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < MT; i++) {
#pragma unroll
                for (int gq = 0; gq < NG; gq++) {
                    uint32_t v[4], y[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const uint32_t * row = reinterpret_cast<const uint32_t *>(vr + (16 * i + 4 * t + k) * rowb + 36 * gq);
                        y[k]                 = row[g < 4 ? 0 : 4];
                        v[k]                 = prmt(row[1 + g], y[k], selv);
                    }
                    const uint32_t d0 = prmt(y[0], y[1], seld), d1 = prmt(y[2], y[3], seld);
#pragma unroll
                    for (int b = 0; b < 4; b++) {
                        const uint32_t sel = 0x4400u + 0x1111u * b, x0 = prmt(v[0], v[1], sel), x1 = prmt(v[2], v[3], sel);
                        const uint32_t a0 = low4(x0, d0), a1 = high4(x0, d0), a2 = low4(x1, d1), a3 = high4(x1, d1);
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            mma16816(o[gq][b][nt], a0, a1, a2, a3, ph[i][nt][0], ph[i][nt][1]);
                            if constexpr (PREC) mma16816(o[gq][b][nt], a0, a1, a2, a3, pl[i][nt][0], pl[i][nt][1]);
                        }
                    }
                }
            }
            __syncwarp();
            issue(stage);
            stage = stage + 1 == ST ? 0 : stage + 1;
        }
        // ---- the item's end: the warps' sums side by side ----
        const bool some = warp < run.n;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
            for (int k = 0; k < 2; k++) {
                float x = l[nt][k];
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
                if (g == 0) ms[warp * BM + 8 * nt + 2 * t + k] = make_float2(m[nt][k], x);
                if (some) {
                    float * to = part + (warp * BM + 8 * nt + 2 * t + k) * Ly::pad;
#pragma unroll
                    for (int gq = 0; gq < NG; gq++) {
#pragma unroll
                        for (int b = 0; b < 4; b++) {
                            const int d = 64 * gq + 32 * (g >> 2) + byte_of(g >= 4, g & 3, b);
                            to[d]       = o[gq][b][nt][k];
                            to[d + 16]  = o[gq][b][nt][2 + k];
                        }
                    }
                }
            }
        }
        __syncthreads();
        const bool whole = w.off == 0 && w.take == w.sp.units;
        const int  slot  = 2 * blockIdx.x + (w.off == 0 ? 1 : 0);
        for (int u = tid; u < rows * D; u += W * 32) {
            const int row = u / D, d = u % D;
            float     M = -INFINITY, L = 0.0f, x = 0.0f;
#pragma unroll
            for (int k = 0; k < W; k++) M = fmaxf(M, ms[k * BM + row].x);
#pragma unroll
            for (int k = 0; k < W; k++) {
                const float2 r = ms[k * BM + row];
                if (!(r.y == 0.0f)) {  // a warp without weight may have left anything; a NaN stays one
                    const float wt = exp2a(r.x == -INFINITY && M == -INFINITY ? 0.0f : r.x - M);
                    L += wt * r.y;
                    x += wt * part[(k * BM + row) * Ly::pad + d];
                }
            }
            if (!whole) {
                a.part_acc[((int64_t) slot * a.prow + row) * D + d] = x;
                if (d == 0) a.part_ms[(int64_t) slot * a.prow + row] = make_float2(M, L);
                continue;
            }
            const int tok = a.byG.div(rb + row), h = w.h * a.G + (rb + row - tok * a.G);
            float     f = 1.0f;
            if (a.sinks) {  // relative to the larger of the two maxima
                const float sk = a.sinks[h] * kLog2e;
                if (sk > M) {
                    f = M == -INFINITY ? 0.0f : exp2a(M - sk);
                    L = L * f + exp2f(kShift);
                } else if (sk > -INFINITY) {
                    L += exp2a(sk - M + kShift);
                }
            }
            f = L == 0.0f ? 0.0f : f / L;
            x = f != 0.0f ? x * f : 0.0f;
            uint8_t * dst = a.dst + (int64_t) h * a.dnb1 + (int64_t) (w.r0 + tok) * a.dnb2;
            if constexpr (PREC) {
                reinterpret_cast<float *>(dst)[d] = x;
            } else {
                reinterpret_cast<__half *>(dst)[d] = __float2half_rn(x);
            }
        }
        if (tid == 0 && !whole && w.off == 0) {
            // this CTA opens an item that others go on with: parts of it, for the join
            const int64_t end = range[0] + (range[1] - range[0] - w.rem) + w.sp.units;
            int           e   = blockIdx.x;
            while (range[2] * (e + 1) / range[3] < end) e++;
            a.desc[2 * blockIdx.x + 1] = make_int4(rb, rows, 0, 0);
            a.desc[2 * blockIdx.x]     = make_int4(e - (int) blockIdx.x + 1, w.h, w.r0, 0);
        }
        active = walk_next<BM, kUnit>(a, w);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

template <int D, int NT, bool PREC>
int launch_few(srhpm_ctx * ctx, const PArgs & a, const Pool4 & k, const Pool4 & v, cudaStream_t stream) {
    using Ly = LayF<D, NT, PREC>;
    auto                         kern = fa_paged_q4_few_kernel<D, NT, PREC>;
    static std::atomic<unsigned> done{ 0 };
    const unsigned               bit = 1u << (ctx->device & 31);
    if (!(done.load() & bit)) {
        const int st = cuda_status(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Ly::total));
        if (st != SRHPM_OK) return st;
        done.fetch_or(bit);
    }
    const int st = cuda_status(launch_k_pdl(kern, dim3(ctx->num_sms), dim3(Ly::W * 32), Ly::total, stream, a, k, v));
    ctx->launches.fetch_add(1);
    if (st != SRHPM_OK) return st;
    return merge_launch(ctx, a, D, PREC, std::min(32, a.prow), stream);
}

}  // namespace

int fap::q4_few_rows(int) { return 8; }

int fap::q4_few_run(srhpm_ctx * ctx, const PArgs & a, const PagedCache & c, bool f32, cudaStream_t stream) {
    const Pool4 k{ c.k, c.knb1, c.knb2, c.knb3 }, v{ c.v, c.vnb1, c.vnb2, c.vnb3 };
    if (c.D == 64) return f32 ? launch_few<64, 1, true>(ctx, a, k, v, stream) : launch_few<64, 1, false>(ctx, a, k, v, stream);
    if (c.D == 128) return f32 ? launch_few<128, 1, true>(ctx, a, k, v, stream) : launch_few<128, 1, false>(ctx, a, k, v, stream);
    return f32 ? launch_few<256, 1, true>(ctx, a, k, v, stream) : launch_few<256, 1, false>(ctx, a, k, v, stream);
}

}  // namespace srhpm
