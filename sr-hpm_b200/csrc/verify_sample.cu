// Acceptance of drafted tokens that keeps the target's distribution (srhpm_verify_sample).
//
// With e_rj = exp((l_rj - m_r) / t) and Z_r their sum over the vocabulary, row r's drafted token x is accepted when
// u q(x) < e_rx / Z_r; the first row that does not accept emits the first j whose inclusive sum of weights is above
// u' times their total, the weights being max(e_j / Z - q_j, 0), or e_j without x (a drafter without distributions), or
// e_j (the last row).
//
// Two launches:
//   sample_part_kernel   every row's logits once (bandwidth bound): per 512 to 4096 tokens the maximum, its first place
//                        and the sum of exponentials in f32.
//   sample_pick_kernel   a cluster of CTAs per sequence: joins the rows' records, accepts, and draws from the one row
//                        that emits. An accepted token is a comparison of two numbers, f32 exponentials (2^-22) do; a drawn
//                        token is a place in a sum over the whole vocabulary: with V tokens and sums off by d, the place
//                        moves in 2 V d of all draws, so 10^5 tokens want d well below 2^-30. Weights of that row and
//                        their sums are taken in 64 bits. The row is split over the cluster in blocks of 512 tokens or
//                        more, in order; block sums, CTA sums and the sums inside one block find the place.
//
// Measured with 151936 tokens: 9 rows of one sequence 16.4 us (latencies: 6 the parts, 3.5 acceptance, 4 the weights, 2 the
// place); 64 sequences of 3 to 9 rows with the drafter's distributions 75: 35 the parts at the copy rate, 40 the pick, whose
// 64-bit instructions and conversions take 67 cycles per 32 tokens and scheduler (two CTAs on 108 SMs, one on the others).
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "internal.h"
#include "launch.cuh"
#include "ptx.cuh"

namespace srhpm {
namespace {

constexpr int   kPartThreads = 256;
constexpr int   kPartVec     = 4;                // 16-byte loads of a lane in flight
constexpr int   kTurn        = kPartVec * 128;   // tokens of a warp's turn
constexpr int   kMaxTurns    = 8;                // of a record
constexpr int   kPickThreads = 512;
constexpr int   kPickWarps   = kPickThreads / 32;
constexpr int   kMaxBlocks   = 1024;                           // blocks of a CTA's share
constexpr float kLog2e       = 1.4426950408889634f;

struct SampleArgs {
    SampleView v;
    int        seg, nseg;  // tokens of a record, records of a row
    int4 *     part;  // [T][nseg]: maximum, sum (bits), first place of the maximum
};

__device__ __forceinline__ float clean(float x) { return x == x ? x : -INFINITY; }

__device__ __forceinline__ float fast_ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// tokens j .. j + 3 of a row (NaN and places behind the vocabulary: `none`)
__device__ __forceinline__ void load4(const float * row, bool vec, int j, int V, float none, float (&x)[4]) {
    if (vec && j + 4 <= V) {
        const float4 f = __ldcs(reinterpret_cast<const float4 *>(row + j));
        x[0] = f.x; x[1] = f.y; x[2] = f.z; x[3] = f.w;
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = x[e] == x[e] ? x[e] : none;
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float f = j + e < V ? __ldcs(row + j + e) : none;
            x[e]          = f == f ? f : none;
        }
    }
}

// the sequence of row t, by a 32-way search of the row starts (one warp); -1 behind the last one
__device__ __forceinline__ int seq_of_row(const SampleView & v, int t) {
    const int lane = threadIdx.x & 31;
    int       lo = 0, n = v.S;  // start[lo] <= t is taken for granted, the sequence is in [lo, lo + n)
    if (t < v.q_start[0] || t >= v.q_start[v.S]) return -1;
    while (n > 1) {
        const int      step = (n + 31) / 32, at = lo + lane * step;
        const uint32_t in   = 1u | __ballot_sync(0xffffffffu, at < lo + n && v.q_start[at] <= t);
        const int      k    = 31 - __clz(in);  // the last start at or before t (starts rise)
        const int      end  = lo + n;
        lo += k * step;
        n = min(step, end - lo);
    }
    return lo;
}

// A warp takes whole records of 1 to 8 turns, 512 tokens a turn, the next turn's loads in flight (over the border of a record too); every
// lane keeps its own maximum, sum and place, joined across the lanes at a record's end: no barrier, 148 SMs x 32 warps each
// with 2 KB on the way.
__global__ void __launch_bounds__(kPartThreads, 4) sample_part_kernel(const SampleArgs a) {
    const SampleView & v = a.v;
    pdl_launch_dependents();
    pdl_wait();
    const int     lane = threadIdx.x & 31;
    const int64_t jobs = (int64_t) v.T * a.nseg, step = (int64_t) gridDim.x * (kPartThreads / 32);
    int64_t       job = (int64_t) blockIdx.x * (kPartThreads / 32) + (threadIdx.x >> 5);
    if (job >= jobs) return;
    int   t = (int) (job / a.nseg), at = (int) (job % a.nseg) * a.seg;  // row, first token of the turn
    int   end = min(v.V, at + a.seg);
    float nx[kPartVec][4];
    auto  fetch = [&](int row_t, int from, int to) {
        const float * row = reinterpret_cast<const float *>(v.logits + (int64_t) row_t * v.ldb);
        const int     j   = from + lane * 4;
        if ((reinterpret_cast<uintptr_t>(row) & 15) == 0 && from + kTurn <= to) {
#pragma unroll
            for (int k = 0; k < kPartVec; k++) {
                const float4 f = __ldcs(reinterpret_cast<const float4 *>(row + j) + 32 * k);
                nx[k][0] = f.x; nx[k][1] = f.y; nx[k][2] = f.z; nx[k][3] = f.w;
            }
        } else {
#pragma unroll
            for (int k = 0; k < kPartVec; k++) {
#pragma unroll
                for (int e = 0; e < 4; e++) nx[k][e] = j + 128 * k + e < to ? __ldcs(row + j + 128 * k + e) : -INFINITY;
            }
        }
    };
    fetch(t, at, end);
    float c = kLog2e, m = -INFINITY, sum = 0.0f;
    int   top = INT32_MAX, known = -1;
    for (;;) {
        float x[kPartVec][4];
#pragma unroll
        for (int k = 0; k < kPartVec; k++) {
#pragma unroll
            for (int e = 0; e < 4; e++) x[k][e] = nx[k][e];
        }
        // the next turn
        const bool    last = at + kTurn >= end;
        const int64_t nj   = last ? job + step : job;
        int           nt = t, na = at + kTurn, ne = end;
        if (last && nj < jobs) {
            nt = (int) (nj / a.nseg);
            na = (int) (nj - (int64_t) nt * a.nseg) * a.seg;
            ne = min(v.V, na + a.seg);
        }
        if (nj < jobs) fetch(nt, na, ne);
        if (v.temp && t != known) {  // with the loads in flight
            const int s = seq_of_row(v, t);
            c           = s >= 0 ? fminf(kLog2e / v.temp[s], FLT_MAX) : kLog2e;  // finite: 0 c is 0
            known       = t;
        }
        float mt = m;
#pragma unroll
        for (int k = 0; k < kPartVec; k++) mt = fmaxf(mt, fmaxf(fmaxf(x[k][0], x[k][1]), fmaxf(x[k][2], x[k][3])));  // NaN: left out
        if (mt > m) {  // its first place; seldom after the first turns
            sum *= m == -INFINITY ? 0.0f : fast_ex2(fmaxf((m - mt) * c, -200.0f));
            m = mt;
#pragma unroll
            for (int k = kPartVec - 1; k >= 0; k--) {
#pragma unroll
                for (int e = 3; e >= 0; e--) {
                    if (x[k][e] == m) top = at + lane * 4 + 128 * k + e;
                }
            }
        }
        // differences first: a rounded product m * c would count into every term. fmaxf: a NaN becomes nothing (2^-200)
#pragma unroll
        for (int k = 0; k < kPartVec; k++) {
            float p[4];
#pragma unroll
            for (int e = 0; e < 4; e++) p[e] = fast_ex2(fmaxf((x[k][e] - m) * c, -200.0f));
            sum += (p[0] + p[1]) + (p[2] + p[3]);
        }
        if (m == INFINITY) {  // the weight stands on the infinities alone
#pragma unroll
            for (int k = 0; k < kPartVec; k++) {
#pragma unroll
                for (int e = 0; e < 4; e++) sum += x[k][e] == m ? 1.0f : 0.0f;
            }
        }
        if (last) {
            if (m == -INFINITY) {
                sum = 0.0f;
                top = INT32_MAX;
            }
            float mw = m;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) mw = fmaxf(mw, __shfl_xor_sync(0xffffffffu, mw, o));
            sum = m == mw ? sum : m == -INFINITY ? 0.0f : sum * fast_ex2(fmaxf((m - mw) * c, -200.0f));
            if (m != mw) top = INT32_MAX;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            top = __reduce_min_sync(0xffffffffu, top);
            if (lane == 0) {
                a.part[(int64_t) t * a.nseg + at / a.seg] = make_int4(__float_as_int(mw), __float_as_int(sum), top, 0);
            }
            m   = -INFINITY;
            sum = 0.0f;
            top = INT32_MAX;
            if (nj >= jobs) break;
        }
        job = nj;
        t   = nt;
        at  = na;
        end = ne;
    }
}

// exp((x - m) / t) in 64 bits, x <= m, as 2^y, y = x (log2 e / t) - m (log2 e / t) = k + f with |f| <= 1/2: 2^f by the
// polynomial that meets it in the 9 Chebyshev points of [-1/2, 1/2] (off by 2^-39.8 at most; the series of exp needs
// two powers more for the same), k added to the exponent. 13 instructions of 64
// bits, no table and no branches: these are what a drawn token costs. Weights below e^-690 of the row's largest are 0.
__constant__ double kPow2[8] = { 0.6931471805459335,    0.2402265069581299,     0.05550410941205933,    0.009618129159402558,
                                 0.0013333450568000645, 0.00015403455852453838, 1.5310079402249296e-05, 1.3255224878668817e-06 };
struct Exp64 {
    double a, b;   // y = a x + b
    float  least;  // x below it (and NaN): weight 0
    float  mf;
    // 0: as above; 1: all weight on the places of the maximum (+inf, or a temperature so low that the next smaller f32 has
    // none: y would be the rounding of m (log2 e / t) there); 2: all weight on `top`
    int    top, mode;
    __device__ __forceinline__ void set(float m, int t, float temp) {
        mf   = m;
        top  = t;
        // low temperatures: a step of an f32 is many times t; beyond 708 t the exponent would leave the doubles' range
        least = fmaxf(m - 690.0f * temp, -FLT_MAX);
        if (m - least > 700.0f * temp) least = nextafterf(least, INFINITY);
        mode = m == -INFINITY ? 0 : !(temp > 0.0f) ? 2 : m == INFINITY || least == m ? 1 : 0;
        if (mode != 0) least = -INFINITY;
        if (m == -INFINITY) least = INFINITY;  // a row of -inf and NaN: no token has weight
        a = mode == 0 ? 1.4426950408889634 / (double) temp : 0.0;
        b = mode == 0 && m > -INFINITY ? -(double) m * a : 0.0;
    }
    // without ZERO anything stands for a weight of 0: sums take it under the condition x >= least
    template <bool ZERO> __device__ __forceinline__ double of(float x) const {
        const double y = fma((double) fmaxf(x, least), a, b);
        const double t = y + 6755399441055744.0;  // rounds to a whole number
        const double f = y - (t - 6755399441055744.0);
        double       p = kPow2[7];
#pragma unroll
        for (int i = 6; i >= 0; i--) p = fma(p, f, kPow2[i]);
        p = fma(p, f, 1.0);
        p = __hiloint2double(__double2hiint(p) + (__double2loint(t) << 20), __double2loint(p));
        return !ZERO || x >= least ? p : 0.0;
    }
    // weights of tokens j .. j + 3; mode is the same for the whole row
    template <bool ZERO> __device__ __forceinline__ void four(const float (&x)[4], int j, double (&w)[4]) const {
        if (mode == 0) {
#pragma unroll
            for (int e = 0; e < 4; e++) w[e] = of<ZERO>(x[e]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) w[e] = (mode == 1 ? x[e] == mf : j + e == top) ? 1.0 : 0.0;
        }
    }
};

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

__device__ __forceinline__ double ld_dsmem_f64(uint32_t addr) {
    double v;
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(addr) : "memory");
    return v;
}

template <int kCluster> __global__ void __launch_bounds__(kPickThreads, 2) sample_pick_kernel(const SampleArgs a) {
    const SampleView & v = a.v;
    __shared__ double  bsum[kMaxBlocks], qsum[kMaxBlocks], share[3], wred[kPickWarps];
    __shared__ float   row_m[kPickWarps];
    __shared__ double  row_z[kPickWarps];
    __shared__ int     row_top[kPickWarps], row_ok[kPickWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rank = blockIdx.x % kCluster, s = blockIdx.x / kCluster;
    pdl_launch_dependents();
    pdl_wait();
    __syncthreads();
    const int r0 = min(max(v.q_start[s], 0), v.T), r1 = min(max(v.q_start[s + 1], r0), v.T);
    if (r0 == r1) {  // the whole cluster
        if (rank == 0 && threadIdx.x == 0) v.out_n[s] = 0;
        return;
    }
    const float  tf    = v.temp ? v.temp[s] : 1.0f;
    const float  c     = tf > 0.0f ? fminf(kLog2e / tf, FLT_MAX) : 0.0f;

    // ---- acceptance: a warp per row, kPickWarps rows at a time; every CTA of the cluster decides for itself
    Exp64 ex;
    int    pick = -1;  // the row that emits
    float  pm = 0.0f;
    int    ptop = 0;
    double pz = 0.0;  // its sum from the f32 records
    for (int b = r0; b < r1; b += kPickWarps) {
        const int r = b + warp;
        if (r < r1) {
            float  m = -INFINITY;
            int    top = INT32_MAX;
            double z = 0.0;
            for (int g0_ = 0; g0_ < a.nseg; g0_ += 128) {  // four records per lane in flight
                int4 p[4];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const int g = g0_ + 32 * k + lane;
                    p[k] = g < a.nseg ? __ldcg(a.part + (int64_t) r * a.nseg + g) : make_int4(__float_as_int(-INFINITY), 0, INT32_MAX, 0);
                }
                float mn = m;
#pragma unroll
                for (int k = 0; k < 4; k++) mn = fmaxf(mn, __int_as_float(p[k].x));
                if (mn > m) {
                    z  = m == -INFINITY ? 0.0 : z * (double) exp2f(fmaxf((m - mn) * c, -200.0f));
                    m  = mn;
                    top = INT32_MAX;
                }
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const float pm_ = __int_as_float(p[k].x);
                    if (pm_ == m) top = min(top, p[k].z);
                    if (pm_ > -INFINITY) z += (pm_ == m ? 1.0 : (double) exp2f(fmaxf((pm_ - m) * c, -200.0f))) * (double) __int_as_float(p[k].y);
                }
            }
            {
                float mw = m;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) mw = fmaxf(mw, __shfl_xor_sync(0xffffffffu, mw, o));
                if (m != mw) {
                    z   = m == -INFINITY ? 0.0 : z * (double) exp2f(fmaxf((m - mw) * c, -200.0f));
                    top = INT32_MAX;
                }
                m   = mw;
                top = __reduce_min_sync(0xffffffffu, top);
            }
            z = tf > 0.0f ? warp_sum(z) : 1.0;
            if (m == -INFINITY) top = 0;
            ex.set(m, top, tf);
            const bool last = r == r1 - 1;
            const int  x    = last ? -1 : v.ids[r + 1];
            double     p = 0.0, q = 0.0;
            if (x >= 0 && x < v.V) {
                const float l = clean(reinterpret_cast<const float *>(v.logits + (int64_t) r * v.ldb)[x]);
                if (m > -INFINITY) {
                    const float l4[4] = { l, l, l, l };
                    double      w4[4];
                    ex.four<true>(l4, x, w4);
                    p = w4[0] / z;
                }
                q = v.dprobs ? (double) reinterpret_cast<const float *>(v.dprobs + (int64_t) r * v.dldb)[x] : 1.0;
            }
            if (lane == 0) {
                row_m[warp]   = m;
                row_top[warp] = top;
                row_z[warp]   = z;
                row_ok[warp]  = !last && (double) v.u[r] * q < p;
                if (rank == 0 && v.p_draft) v.p_draft[r] = (float) p;
            }
        }
        __syncthreads();
        if (pick < 0) {
            for (int w = 0; w < kPickWarps && b + w < r1; w++) {
                if (!row_ok[w]) {
                    pick = b + w;
                    pm   = row_m[w];
                    ptop = row_top[w];
                    pz   = row_z[w];
                    break;
                }
            }
        }
        __syncthreads();
    }
    if (rank == 0) {
        for (int r = r0 + threadIdx.x; r < r1; r += kPickThreads) {
            if (r != pick) v.out_ids[r] = r < pick ? v.ids[r + 1] : -1;
        }
        if (threadIdx.x == 0) v.out_n[s] = pick - r0 + 1;
    }

    // ---- the emitted token: this CTA's share is blocks of `len` tokens, one warp each
    const bool    last = pick == r1 - 1;
    const int     x    = last ? -1 : v.ids[pick + 1];
    const float * row  = reinterpret_cast<const float *>(v.logits + (int64_t) pick * v.ldb);
    const float * qr   = !last && v.dprobs ? reinterpret_cast<const float *>(v.dprobs + (int64_t) pick * v.dldb) : nullptr;
    const bool    vec  = (reinterpret_cast<uintptr_t>(row) & 15) == 0, qvec = (reinterpret_cast<uintptr_t>(qr) & 15) == 0;
    // blocks of 512 tokens, 16 per lane, pay for the sums across the lanes and the loop; of 128 where a warp would have
    // no more than two of those (9 sequences of 32000 tokens 11.9 us, with 512 14.3; 16 of 151936 29.7 and 31.6; beyond: 64 of
    // 151936 69.0 with 512, with 128 72.0); longer ones where kMaxBlocks would not do
    const int     few = (int64_t) v.V <= (int64_t) kCluster * kPickWarps * 1024 ? 128 : 512;
    const int     len = few == 128 ? 128 : 512 * (int) (((int64_t) v.V + (int64_t) kCluster * kMaxBlocks * 512 - 1) / ((int64_t) kCluster * kMaxBlocks * 512));
    const int     nblk = (int) (((int64_t) v.V + len - 1) / len), per = (nblk + kCluster - 1) / kCluster;
    const int     g0 = min(nblk, rank * per), g1 = min(nblk, g0 + per);
    ex.set(pm, ptop, tf);
    double inv_z = 1.0;
    auto logits4 = [&](int j, float (&l)[4]) { load4(row, vec, j, v.V, -INFINITY, l); };
    auto drafts4 = [&](int j, float (&q)[4]) {
#pragma unroll
        for (int e = 0; e < 4; e++) q[e] = 0.0f;
        if (qr) load4(qr, qvec, j, v.V, 0.0f, q);
    };
    auto weights = [&](int j, const float (&l)[4], const float (&q)[4], double (&w)[4]) {  // tokens j .. j + 3
        ex.four<true>(l, j, w);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (qr) {
                w[e] = fmax(w[e] * inv_z - (double) q[e], 0.0);
            } else if (j + e == x) {
                w[e] = 0.0;
            }
        }
    };
    auto cluster_get = [&](int i, int r) { return ld_dsmem_f64(mapa_shared(smem_u32(&share[i]), r)); };
    // One pass over the share gives the row's sum Z, and per block the sums of e and of q over the tokens with e / Z > q,
    // told apart by the f32 records' Z: the block's weight is then (sum e) / Z - sum q. A block with a token whose e / Z is
    // nearer to q than 2^-19 (to 2^-18: 4 steps of the doubles' upper words) is done again with Z in 64 bits, and so are all
    // blocks where the records' Z turns out to be off by more than 2^-20 (it is mostly near 2^-22): every other token is on
    // its side. One token in 10^5 is that near where the drafter is 0.5 off in the logits, all are where it equals the
    // target. 64 sequences: 75 us; without 72, with a margin of 2^-16, which bounds the records' Z beforehand, 78.
    {
        double      sz = 0.0;
        auto block = [&](auto pieces, int at, double & se, double & sq, bool & near) {  // `pieces` times 128 tokens from `at`
            constexpr int P = decltype(pieces)::value;
            float         l[P][4], q[P][4];
            const int     j0 = at + lane * 4;
            if (vec && qvec && at + P * 128 <= v.V) {
#pragma unroll
                for (int k = 0; k < P; k++) {
                    const float4 f = __ldcs(reinterpret_cast<const float4 *>(row + j0) + 32 * k);
                    l[k][0] = f.x; l[k][1] = f.y; l[k][2] = f.z; l[k][3] = f.w;
                }
#pragma unroll
                for (int k = 0; k < P; k++) {
                    const float4 f = qr ? __ldcs(reinterpret_cast<const float4 *>(qr + j0) + 32 * k) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    q[k][0] = f.x; q[k][1] = f.y; q[k][2] = f.z; q[k][3] = f.w;
                }
            } else {
#pragma unroll
                for (int k = 0; k < P; k++) {
                    logits4(j0 + 128 * k, l[k]);
                    drafts4(j0 + 128 * k, q[k]);
                }
            }
            if (lane < 4 * P) {  // the warp's next block on its way to L2
                const int64_t next = min((int64_t) at + (int64_t) kPickWarps * len + 32 * lane, (int64_t) v.V - 1);
                asm volatile("prefetch.global.L2 [%0];" ::"l"(row + next));
                if (qr) asm volatile("prefetch.global.L2 [%0];" ::"l"(qr + next));
            }
            // sums of the tokens that have a weight (places behind the vocabulary are -inf): a sum of 0 means that none has
            // one, which a random number of 0 hangs on. Additions under the predicate cost nothing (batch of 64: 72.1 us,
            // 71.8 with e^-690 for a weight of 0)
#pragma unroll
            for (int k = 0; k < P; k++) {
                const int j = j0 + 128 * k;
                double    w[4];
                ex.four<false>(l[k], j, w);
                if (qr) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const double qe = q[k][e];
                        near |= (uint32_t) (__double2hiint(w[e]) - __double2hiint(qe * pz) + 4) <= 8u;
                        asm("{\n\t.reg .pred p, has;\n\tsetp.ge.f32 has, %6, %7;\n\tsetp.gt.and.f64 p, %3, %4, has;\n\t"
                            "@has add.f64 %2, %2, %3;\n\t@p add.f64 %0, %0, %3;\n\t@p add.f64 %1, %1, %5;\n\t}"
                            : "+d"(se), "+d"(sq), "+d"(sz)
                            : "d"(w[e]), "d"(qe * pz), "d"(qe), "f"(l[k][e]), "f"(ex.least));
                    }
                } else {
                    if (x >= j && x < j + 4) {
#pragma unroll
                        for (int e = 0; e < 4; e++) w[e] = j + e == x ? 0.0 : w[e];
                    }
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        asm("{\n\t.reg .pred has;\n\tsetp.ge.f32 has, %2, %3;\n\t@has add.f64 %0, %0, %1;\n\t}"
                            : "+d"(se)
                            : "d"(w[e]), "f"(l[k][e]), "f"(ex.least));
                    }
                }
            }
        };
        for (int g = g0 + warp; g < g1; g += kPickWarps) {
            double se = 0.0, sq = 0.0;
            bool   near = false;
            if (len == 128) {
                block(std::integral_constant<int, 1>{}, g * 128, se, sq, near);
            } else {
                for (int k = 0; k < len; k += 512) block(std::integral_constant<int, 4>{}, g * len + k, se, sq, near);
            }
            se = warp_sum(se);
            if (qr) sq = warp_sum(sq);
            near = __any_sync(0xffffffffu, near && ex.mode == 0);  // the other modes' sums are whole numbers
            if (lane == 0) {
                bsum[g - g0] = se;
                qsum[g - g0] = near ? -1.0 : sq;
            }
        }
        if (qr) {
            sz = warp_sum(sz);
            if (lane == 0) wred[warp] = sz;
            __syncthreads();
            if (threadIdx.x == 0) {
                double t = 0.0;
                for (int w = 0; w < kPickWarps; w++) t += wred[w];
                share[0] = t;
            }
            cluster_sync_all();
            sz = 0.0;
            for (int r = 0; r < kCluster; r++) sz += cluster_get(0, r);
            inv_z = sz > 0.0 ? 1.0 / sz : 0.0;
            const bool all = fabs(sz - pz) > sz * 0x1p-20;
            __syncwarp();
            for (int g = g0 + warp; g < g1; g += kPickWarps) {  // of this warp's blocks
                if (!all && qsum[g - g0] >= 0.0) continue;
                double sw = 0.0;
                auto   again = [&](auto pieces, int j0) {  // a piece's loads go out together
                    constexpr int P = decltype(pieces)::value;
                    float         l[P][4], q[P][4];
#pragma unroll
                    for (int k = 0; k < P; k++) {
                        logits4(j0 + 128 * k, l[k]);
                        drafts4(j0 + 128 * k, q[k]);
                    }
#pragma unroll
                    for (int k = 0; k < P; k++) {
                        double w[4];
                        weights(j0 + 128 * k, l[k], q[k], w);
                        sw += (w[0] + w[1]) + (w[2] + w[3]);
                    }
                };
                if (len == 128) {
                    again(std::integral_constant<int, 1>{}, g * 128 + lane * 4);
                } else {
                    for (int k = 0; k < len; k += 512) again(std::integral_constant<int, 4>{}, g * len + k + lane * 4);
                }
                sw = warp_sum(sw);
                __syncwarp();
                if (lane == 0) {
                    bsum[g - g0] = sw * sz;  // the scan below takes it times 1 / Z
                    qsum[g - g0] = 0.0;
                }
            }
        }
    }
    __syncthreads();
    if (warp == 0) {  // inclusive sums of the blocks
        double before = 0.0;
        for (int b = 0; b < g1 - g0; b += 32) {
            double t = b + lane < g1 - g0 ? (qr ? fmax(bsum[b + lane] * inv_z - qsum[b + lane], 0.0) : bsum[b + lane]) : 0.0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double u = __shfl_up_sync(0xffffffffu, t, o);
                if (lane >= o) t += u;
            }
            t += before;
            if (b + lane < g1 - g0) bsum[b + lane] = t;
            before = __shfl_sync(0xffffffffu, t, 31);
        }
        if (lane == 0) share[1] = before;
    }
    cluster_sync_all();
    if (warp == 0) {
        double t[kCluster], total = 0.0, before = 0.0;
        int    lastc = -1, owner = -1;
#pragma unroll
        for (int r = 0; r < kCluster; r++) t[r] = cluster_get(1, r);
#pragma unroll
        for (int r = 0; r < kCluster; r++) total += t[r];
        const double goal = (double) v.us[s] * total;
        double       run = 0.0;
#pragma unroll
        for (int r = 0; r < kCluster; r++) {
            if (t[r] > 0.0) lastc = r;
            if (owner < 0 && run + t[r] > goal) {
                owner  = r;
                before = run;
            }
            run += t[r];
        }
        const bool past = owner < 0;  // goal rounded up to the total: the last token with weight
        if (past) owner = lastc;
        if (!(total > 0.0)) {
            if (rank == 0 && lane == 0) v.out_ids[pick] = ptop;
        } else if (rank == owner) {
            // first block whose inclusive sum is above the goal (past: the last one that adds to the sum)
            int blk = -1;
            for (int b = 0; b < g1 - g0; b += 32) {
                const int  i  = b + lane;
                const bool in = i < g1 - g0;
                if (past) {
                    const uint32_t hit = __ballot_sync(0xffffffffu, in && bsum[i] > (i ? bsum[i - 1] : 0.0));
                    if (hit) blk = b + 31 - __clz(hit);
                } else {
                    const uint32_t hit = __ballot_sync(0xffffffffu, in && before + bsum[i] > goal);
                    if (hit) {
                        blk = b + __ffs(hit) - 1;
                        break;
                    }
                }
            }
            if (blk < 0) blk = g1 - g0 - 1;
            double start = before + (blk > 0 ? bsum[blk - 1] : 0.0);
            int    at = -1, lastw = -1;
            auto place = [&](auto pieces, int from) {  // 4 `pieces` tokens in a row per lane: one sum across the lanes
                constexpr int P = decltype(pieces)::value;
                float         l[P][4], q[P][4];
                double        w[P][4], t4 = 0.0;
                const int     j0 = from + lane * 4 * P;
#pragma unroll
                for (int i = 0; i < P; i++) {
                    logits4(j0 + 4 * i, l[i]);
                    drafts4(j0 + 4 * i, q[i]);
                }
#pragma unroll
                for (int i = 0; i < P; i++) {
                    weights(j0 + 4 * i, l[i], q[i], w[i]);
                    t4 += (w[i][0] + w[i][1]) + (w[i][2] + w[i][3]);
                }
                double inc = t4;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double u = __shfl_up_sync(0xffffffffu, inc, o);
                    if (lane >= o) inc += u;
                }
                double run4 = start + (inc - t4);
                int    mine = INT32_MAX, ml = -1;
#pragma unroll
                for (int i = 0; i < P; i++) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        run4 += w[i][e];
                        if (w[i][e] > 0.0) {
                            ml = j0 + 4 * i + e;
                            if (!past && run4 > goal && mine == INT32_MAX) mine = ml;
                        }
                    }
                }
                mine  = __reduce_min_sync(0xffffffffu, mine);
                lastw = max(lastw, __reduce_max_sync(0xffffffffu, ml));
                if (mine != INT32_MAX) at = mine;
                start += __shfl_sync(0xffffffffu, inc, 31);
            };
            const int from = (g0 + blk) * len;
            if (len == 128) {
                place(std::integral_constant<int, 1>{}, from);
            } else {
                for (int k = 0; k < len && at < 0; k += 512) place(std::integral_constant<int, 4>{}, from + k);
            }
            if (lane == 0) v.out_ids[pick] = at >= 0 ? at : lastw >= 0 ? lastw : ptop;
        }
    }
    cluster_sync_all();  // no CTA leaves while another reads its sums
}

template <int CL> int launch_pick(srhpm_ctx * ctx, const SampleArgs & a, cudaStream_t stream) {
    if (CL > 8) {
        static std::atomic<unsigned> done{ 0 };
        const unsigned               bit = 1u << (ctx->device & 31);
        if (!(done.load() & bit)) {
            const int st = cuda_status(cudaFuncSetAttribute(sample_pick_kernel<CL>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
            if (st != SRHPM_OK) return st;
            done.fetch_or(bit);
        }
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim            = dim3((unsigned) a.v.S * CL);
    cfg.blockDim           = dim3(kPickThreads);
    cfg.stream             = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id                                         = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id                                         = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x                           = CL;
    attr[1].val.clusterDim.y                           = 1;
    attr[1].val.clusterDim.z                           = 1;
    cfg.attrs                                          = attr;
    cfg.numAttrs                                       = 2;
    const int st = cuda_status(cudaLaunchKernelEx(&cfg, sample_pick_kernel<CL>, a));
    ctx->launches.fetch_add(1);
    return st;
}

}  // namespace

// tokens of a record: as many turns as leave every warp of the GPU a record (32 warps per SM), 8 at most
static int seg_tokens(const srhpm_ctx * ctx, int V, int T) {
    const int64_t turns = (int64_t) T * ((V + (int64_t) kTurn - 1) / kTurn), warps = 32 * (int64_t) ctx->num_sms;
    int           k = 2;  // one turn leaves too many records to join: 17.5 us instead of 16.4 for 9 rows of 151936
    while (k < kMaxTurns && turns >= 2 * k * warps) k *= 2;
    return k * kTurn;
}

size_t verify_sample_work_size(const srhpm_ctx * ctx, int V, int T, int) {
    const int seg = seg_tokens(ctx, V, T);
    return (size_t) T * ((V + (int64_t) seg - 1) / seg) * sizeof(int4) + 16;
}

int verify_sample_run(srhpm_ctx * ctx, const SampleView & v, void * wdata, size_t wsize, cudaStream_t stream) {
    if (wdata == nullptr || wsize < verify_sample_work_size(ctx, v.V, v.T, v.S)) return SRHPM_ERR_WORKSPACE;
    SampleArgs a;
    a.v    = v;
    a.seg  = seg_tokens(ctx, v.V, v.T);
    a.nseg = (int) ((v.V + (int64_t) a.seg - 1) / a.seg);
    a.part = reinterpret_cast<int4 *>((reinterpret_cast<uintptr_t>(wdata) + 15) & ~(uintptr_t) 15);
    if (v.V > 1 << 29) return SRHPM_UNSUPPORTED;
    const int64_t want = ((int64_t) v.T * a.nseg + kPartThreads / 32 - 1) / (kPartThreads / 32);
    const int     grid = (int) std::min<int64_t>(4 * (int64_t) ctx->num_sms, want);
    int st = cuda_status(launch_k_pdl(sample_part_kernel, dim3(grid), dim3(kPartThreads), 0, stream, a));
    ctx->launches.fetch_add(1);
    if (st != SRHPM_OK) return st;
    // as many CTAs per sequence as one wave of two per SM holds: a wave and a bit would take twice as long
    const int64_t slots = 2 * (int64_t) ctx->num_sms, S = v.S;
    if (S * 16 <= slots) return launch_pick<16>(ctx, a, stream);
    if (S * 8 <= slots) return launch_pick<8>(ctx, a, stream);
    if (S * 4 <= slots) return launch_pick<4>(ctx, a, stream);
    return launch_pick<2>(ctx, a, stream);
}

}  // namespace srhpm
