// Acceptance of drafted tokens that keeps the target's distribution (srhpm_verify_sample).
//
// With e_rj = exp((l_rj - m_r) / t) and Z_r their sum over the vocabulary, row r's drafted token x is accepted when
// u q(x) < e_rx / Z_r; the first row that does not accept emits the first j whose inclusive sum of weights is above
// u' times their total, the weights being max(e_j / Z - q_j, 0), or e_j without x (a drafter without distributions), or
// e_j (the last row).
//
// Two launches:
//   sample_part_kernel   every row's logits once (bandwidth bound): per 8192 tokens the maximum, its first place and the
//                        sum of exponentials in f32. A CTA holds its 32 KB in registers between the maximum and the sum.
//   sample_pick_kernel   a cluster of CTAs per sequence: joins the rows' records, accepts, and draws from the one row
//                        that emits. An accepted token is a comparison of two numbers, f32 exponentials (2^-22) do; a drawn
//                        token is a place in a sum over the whole vocabulary: with V tokens and sums off by d, the place
//                        moves in 2 V d of all draws, so 10^5 tokens want d well below 2^-30. Weights of that row and
//                        their sums are taken in 64 bits. The row is split over the cluster in blocks of 128 tokens or
//                        more, in order; block sums, CTA sums and the sums inside one block find the place.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "internal.h"
#include "launch.cuh"
#include "ptx.cuh"

namespace srhpm {
namespace {

constexpr int   kPartThreads = 256;
constexpr int   kPartVec     = 8;                              // 16-byte loads per thread
constexpr int   kSeg         = kPartThreads * kPartVec * 4;    // tokens per record
constexpr int   kPickThreads = 512;
constexpr int   kPickWarps   = kPickThreads / 32;
constexpr int   kCluster     = 8;
constexpr int   kMaxBlocks   = 1024;                           // blocks of a CTA's share
constexpr float kLog2e       = 1.4426950408889634f;

struct SampleArgs {
    SampleView v;
    int        nseg;
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

__global__ void __launch_bounds__(kPartThreads) sample_part_kernel(const SampleArgs a) {
    const SampleView & v = a.v;
    __shared__ float   sm[kPartThreads / 32], ss[kPartThreads / 32];
    __shared__ int     si[kPartThreads / 32];
    pdl_launch_dependents();
    pdl_wait();
    const int     t = blockIdx.x, seg = blockIdx.y, j0 = seg * kSeg, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float * row = reinterpret_cast<const float *>(v.logits + (int64_t) t * v.ldb);
    const bool    vec = (reinterpret_cast<uintptr_t>(row) & 15) == 0;
    float         x[kPartVec][4];
#pragma unroll
    for (int k = 0; k < kPartVec; k++) load4(row, vec, j0 + (k * kPartThreads + (int) threadIdx.x) * 4, v.V, -INFINITY, x[k]);
    float c = kLog2e;
    if (v.temp) {
        const int s = seq_of_row(v, t);  // while the loads are in flight
        if (s >= 0) c = kLog2e / v.temp[s];
    }
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < kPartVec; k++) m = fmaxf(m, fmaxf(fmaxf(x[k][0], x[k][1]), fmaxf(x[k][2], x[k][3])));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) sm[warp] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kPartThreads / 32; w++) m = fmaxf(m, sm[w]);
    // differences first: a rounded product m * c would count into every term
    float sum = 0.0f;
    int   top = INT32_MAX;
#pragma unroll
    for (int k = kPartVec - 1; k >= 0; k--) {
        float p[4];
#pragma unroll
        for (int e = 3; e >= 0; e--) {
            const bool is = x[k][e] == m;
            p[e]          = is ? 1.0f : fast_ex2((x[k][e] - m) * c);
            if (is) top = j0 + (k * kPartThreads + (int) threadIdx.x) * 4 + e;
        }
        sum += (p[0] + p[1]) + (p[2] + p[3]);
    }
    if (m == -INFINITY) sum = 0.0f;
    top = __reduce_min_sync(0xffffffffu, top);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) {
        ss[warp] = sum;
        si[warp] = top;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
        for (int w = 1; w < kPartThreads / 32; w++) {
            sum += ss[w];
            top = min(top, si[w]);
        }
        a.part[(int64_t) t * a.nseg + seg] = make_int4(__float_as_int(m), __float_as_int(sum), top, 0);
    }
}

// exp((x - m) / t) in 64 bits, x <= m: 2^(k/32) from a table of 32 values times a polynomial of degree 6 in
// |r| <= ln 2 / 64 (its rest: r^7 / 7! < 2^-57). Far cheaper than the full-range function and good to a few 2^-53.
struct Exp64 {
    double         m, inv_t;  // inv_t 0: all weight on `top`
    float          mf;
    int            top;
    const double * tab;
    __device__ __forceinline__ double operator()(float x, int j) const {
        if (inv_t == 0.0) return j == top ? 1.0 : 0.0;
        if (x == mf) return 1.0;
        const double d = ((double) x - m) * inv_t;
        if (!(d > -745.0)) return 0.0;  // below the smallest number (and -inf)
        const double kk = rint(d * 46.16624130844683);  // 32 / ln 2
        const int    k  = (int) kk;
        // ln 2 / 32 in two parts, the first of 36 bits: |kk| < 2^16 times it is exact
        double r = fma(kk, -0.021660849392446835, d);
        r        = fma(kk, -5.145609244655338e-14, r);
        double p = 1.0 / 720.0;
        p = fma(p, r, 1.0 / 120.0);
        p = fma(p, r, 1.0 / 24.0);
        p = fma(p, r, 1.0 / 6.0);
        p = fma(p, r, 0.5);
        p = fma(p, r, 1.0);
        p = fma(p, r, 1.0);
        const int    e = k >> 5;  // power of two, down to -1075
        const double s = tab[k & 31] * p;
        // in two steps below the normal range
        return e > -1022 ? s * __hiloint2double((1023 + e) << 20, 0)
                         : s * __hiloint2double((1023 + e + 600) << 20, 0) * __hiloint2double((1023 - 600) << 20, 0);
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

__global__ void __launch_bounds__(kPickThreads) sample_pick_kernel(const SampleArgs a) {
    const SampleView & v = a.v;
    __shared__ double  tab[32], bsum[kMaxBlocks], share[2], wred[kPickWarps];
    __shared__ float   row_m[kPickWarps];
    __shared__ int     row_top[kPickWarps], row_ok[kPickWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rank = blockIdx.x % kCluster, s = blockIdx.x / kCluster;
    if (threadIdx.x < 32) tab[threadIdx.x] = exp2((double) threadIdx.x / 32.0);
    pdl_launch_dependents();
    pdl_wait();
    __syncthreads();
    const int r0 = min(max(v.q_start[s], 0), v.T), r1 = min(max(v.q_start[s + 1], r0), v.T);
    if (r0 == r1) {  // the whole cluster
        if (rank == 0 && threadIdx.x == 0) v.out_n[s] = 0;
        return;
    }
    const float  tf    = v.temp ? v.temp[s] : 1.0f;
    const double inv_t = tf > 0.0f ? 1.0 / (double) tf : 0.0;
    const float  c     = tf > 0.0f ? kLog2e / tf : 0.0f;

    // ---- acceptance: a warp per row, kPickWarps rows at a time; every CTA of the cluster decides for itself
    Exp64 ex;
    ex.tab   = tab;
    ex.inv_t = inv_t;
    int    pick = -1;  // the row that emits
    float  pm = 0.0f;
    int    ptop = 0;
    for (int b = r0; b < r1; b += kPickWarps) {
        const int r = b + warp;
        if (r < r1) {
            float m = -INFINITY;
            int   top = INT32_MAX;
            for (int g = lane; g < a.nseg; g += 32) {
                const int4 p = __ldcg(a.part + (int64_t) r * a.nseg + g);
                const float pm_ = __int_as_float(p.x);
                if (pm_ > m) {
                    m   = pm_;
                    top = p.z;
                }
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const float om = __shfl_xor_sync(0xffffffffu, m, o);
                const int   ot = __shfl_xor_sync(0xffffffffu, top, o);
                if (om > m || (om == m && ot < top)) {
                    m   = om;
                    top = ot;
                }
            }
            double z = 0.0;
            for (int g = lane; g < a.nseg; g += 32) {
                const int4  p   = __ldcg(a.part + (int64_t) r * a.nseg + g);
                const float pm_ = __int_as_float(p.x);
                if (pm_ > -INFINITY) z += (pm_ == m ? 1.0 : (double) exp2f((pm_ - m) * c)) * (double) __int_as_float(p.y);
            }
            z = warp_sum(z);
            if (m == -INFINITY) top = 0;
            ex.m   = (double) m;
            ex.mf  = m;
            ex.top = top;
            const bool last = r == r1 - 1;
            const int  x    = last ? -1 : v.ids[r + 1];
            double     p = 0.0, q = 0.0;
            if (x >= 0 && x < v.V) {
                const float l = clean(reinterpret_cast<const float *>(v.logits + (int64_t) r * v.ldb)[x]);
                if (m > -INFINITY) p = inv_t == 0.0 ? (x == top ? 1.0 : 0.0) : ex(l, x) / z;
                q = v.dprobs ? (double) reinterpret_cast<const float *>(v.dprobs + (int64_t) r * v.dldb)[x] : 1.0;
            }
            if (lane == 0) {
                row_m[warp]   = m;
                row_top[warp] = top;
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
    const int     len  = 128 * (int) (((int64_t) v.V + (int64_t) kCluster * kMaxBlocks * 128 - 1) / ((int64_t) kCluster * kMaxBlocks * 128));
    const int     nblk = (int) (((int64_t) v.V + len - 1) / len), per = (nblk + kCluster - 1) / kCluster;
    const int     g0 = min(nblk, rank * per), g1 = min(nblk, g0 + per);
    const bool    none = pm == -INFINITY;
    ex.m   = (double) pm;
    ex.mf  = pm;
    ex.top = ptop;
    double inv_z = 1.0;
    auto weights = [&](int j, double (&w)[4]) {  // tokens j .. j + 3
        float l[4];
        load4(row, vec, j, v.V, -INFINITY, l);
        float q[4] = { 0.0f, 0.0f, 0.0f, 0.0f };
        if (qr) load4(qr, qvec, j, v.V, 0.0f, q);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            w[e] = none || j + e >= v.V ? 0.0 : ex(l[e], j + e);
            if (qr) {
                w[e] = fmax(w[e] * inv_z - (double) q[e], 0.0);
            } else if (j + e == x) {
                w[e] = 0.0;
            }
        }
    };
    auto cluster_get = [&](int i, int r) { return ld_dsmem_f64(mapa_shared(smem_u32(&share[i]), r)); };
    if (qr) {  // the row's sum in 64 bits: weights are differences of probabilities
        double z = 0.0;
        for (int g = g0 + warp; g < g1; g += kPickWarps) {
            for (int k = lane * 4; k < len; k += 128) {
                const int j = g * len + k;
                float     l[4];
                load4(row, vec, j, v.V, -INFINITY, l);
#pragma unroll
                for (int e = 0; e < 4; e++) z += none || j + e >= v.V ? 0.0 : ex(l[e], j + e);
            }
        }
        z = warp_sum(z);
        if (lane == 0) wred[warp] = z;
        __syncthreads();
        if (threadIdx.x == 0) {
            double t = 0.0;
            for (int w = 0; w < kPickWarps; w++) t += wred[w];
            share[0] = t;
        }
        cluster_sync_all();
        z = 0.0;
        for (int r = 0; r < kCluster; r++) z += cluster_get(0, r);
        inv_z = z > 0.0 ? 1.0 / z : 0.0;
    }
    for (int g = g0 + warp; g < g1; g += kPickWarps) {
        double t = 0.0;
        for (int k = lane * 4; k < len; k += 128) {
            double w[4];
            weights(g * len + k, w);
            t += (w[0] + w[1]) + (w[2] + w[3]);
        }
        t = warp_sum(t);
        if (lane == 0) bsum[g - g0] = t;
    }
    __syncthreads();
    if (warp == 0) {  // inclusive sums of the blocks
        double before = 0.0;
        for (int b = 0; b < g1 - g0; b += 32) {
            double t = b + lane < g1 - g0 ? bsum[b + lane] : 0.0;
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
            for (int k = 0; k < len && at < 0; k += 128) {
                const int j = (g0 + blk) * len + k + lane * 4;
                double    w[4];
                weights(j, w);
                double t4 = (w[0] + w[1]) + (w[2] + w[3]), inc = t4;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double u = __shfl_up_sync(0xffffffffu, inc, o);
                    if (lane >= o) inc += u;
                }
                double run4 = start + (inc - t4);
                int    mine = INT32_MAX, ml = -1;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    run4 += w[e];
                    if (w[e] > 0.0) {
                        ml = j + e;
                        if (!past && run4 > goal && mine == INT32_MAX) mine = j + e;
                    }
                }
                mine  = __reduce_min_sync(0xffffffffu, mine);
                lastw = max(lastw, __reduce_max_sync(0xffffffffu, ml));
                if (mine != INT32_MAX) at = mine;
                start += __shfl_sync(0xffffffffu, inc, 31);
            }
            if (lane == 0) v.out_ids[pick] = at >= 0 ? at : lastw;
        }
    }
    cluster_sync_all();  // no CTA leaves while another reads its sums
}

}  // namespace

size_t verify_sample_work_size(const srhpm_ctx *, int V, int T, int) {
    return (size_t) T * ((V + (int64_t) kSeg - 1) / kSeg) * sizeof(int4) + 16;
}

int verify_sample_run(srhpm_ctx * ctx, const SampleView & v, void * wdata, size_t wsize, cudaStream_t stream) {
    if (wdata == nullptr || wsize < verify_sample_work_size(ctx, v.V, v.T, v.S)) return SRHPM_ERR_WORKSPACE;
    SampleArgs a;
    a.v    = v;
    a.nseg = (int) ((v.V + (int64_t) kSeg - 1) / kSeg);
    a.part = reinterpret_cast<int4 *>((reinterpret_cast<uintptr_t>(wdata) + 15) & ~(uintptr_t) 15);
    if (a.nseg > 65535) return SRHPM_UNSUPPORTED;
    int st = cuda_status(launch_k_pdl(sample_part_kernel, dim3(v.T, a.nseg), dim3(kPartThreads), 0, stream, a));
    ctx->launches.fetch_add(1);
    if (st != SRHPM_OK) return st;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim            = dim3((unsigned) v.S * kCluster);
    cfg.blockDim           = dim3(kPickThreads);
    cfg.stream             = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id                                         = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id                                         = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x                           = kCluster;
    attr[1].val.clusterDim.y                           = 1;
    attr[1].val.clusterDim.z                           = 1;
    cfg.attrs                                          = attr;
    cfg.numAttrs                                       = 2;
    st = cuda_status(cudaLaunchKernelEx(&cfg, sample_pick_kernel, a));
    ctx->launches.fetch_add(1);
    return st;
}

}  // namespace srhpm
