// Acceptance of drafted tokens that keeps the target's distribution (srhpm_verify_sample): one CTA per sequence.
#include <cuda_runtime.h>

#include <cmath>

#include "internal.h"
#include "launch.cuh"
#include "ptx.cuh"

namespace srhpm {
namespace {

constexpr int kThreads = 1024;

__device__ double cta_sum(double v, double * sp) {
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sp[threadIdx.x >> 5] = v;
    __syncthreads();
    double s = 0.0;
    for (int w = 0; w < kThreads / 32; w++) s += sp[w];
    return s;
}

__device__ __forceinline__ float clean(float x) { return isnan(x) ? -INFINITY : x; }

__device__ __forceinline__ double weight(float x, int j, float m, int top, double inv_t) {
    if (inv_t == 0.0) return j == top ? 1.0 : 0.0;
    return x == m ? 1.0 : exp(((double) x - (double) m) / inv_t);
}

__global__ void __launch_bounds__(kThreads) verify_sample_kernel(const SampleView a) {
    __shared__ double sp[32];
    __shared__ float  sm[32];
    __shared__ int    si[32];
    pdl_launch_dependents();
    pdl_wait();
    const int s = blockIdx.x, r0 = min(max(a.q_start[s], 0), a.T), r1 = min(max(a.q_start[s + 1], r0), a.T);
    if (r0 == r1) {
        if (threadIdx.x == 0) a.out_n[s] = 0;
        return;
    }
    const double tmp  = a.temp ? (double) a.temp[s] : 1.0;
    const double t    = tmp > 0.0 ? tmp : 0.0;
    bool         open = true;
    for (int r = r0; r < r1; r++) {
        const float * x = reinterpret_cast<const float *>(a.logits + (int64_t) r * a.ldb);
        float         m = -INFINITY;
        int           top = INT32_MAX;
        for (int j = threadIdx.x; j < a.V; j += kThreads) {
            const float v = clean(x[j]);
            if (v > m || (v == m && j < top)) {
                m   = v;
                top = j;
            }
        }
        for (int o = 16; o > 0; o >>= 1) {
            const float v = __shfl_xor_sync(0xffffffffu, m, o);
            const int   i = __shfl_xor_sync(0xffffffffu, top, o);
            if (v > m || (v == m && i < top)) {
                m   = v;
                top = i;
            }
        }
        __syncthreads();
        if ((threadIdx.x & 31) == 0) {
            sm[threadIdx.x >> 5] = m;
            si[threadIdx.x >> 5] = top;
        }
        __syncthreads();
        for (int w = 0; w < kThreads / 32; w++) {
            if (sm[w] > m || (sm[w] == m && si[w] < top)) {
                m   = sm[w];
                top = si[w];
            }
        }
        const bool none = m == -INFINITY;
        if (none) top = 0;
        double z = 0.0;
        for (int j = threadIdx.x; j < a.V; j += kThreads) {
            if (!none) z += weight(clean(x[j]), j, m, top, t);
        }
        z                = cta_sum(z, sp);
        const bool  last = r == r1 - 1;
        const int   d    = last ? -1 : a.ids[r + 1];
        const float * q  = a.dprobs ? reinterpret_cast<const float *>(a.dprobs + (int64_t) r * a.dldb) : nullptr;
        const bool  in   = d >= 0 && d < a.V;
        const double p   = in && !none ? weight(clean(x[d]), d, m, top, t) / z : 0.0;
        const double b   = in ? (q ? (double) q[d] : 1.0) : 0.0;
        if (a.p_draft && threadIdx.x == 0) a.p_draft[r] = (float) p;
        if (!open) {
            if (threadIdx.x == 0) a.out_ids[r] = -1;
            continue;
        }
        if (!last && (double) a.u[r] * b < p) {
            if (threadIdx.x == 0) a.out_ids[r] = d;
            continue;
        }
        open = false;
        // the emitted token: contiguous segments per thread, inclusive sums over the threads
        auto w_of = [&](int j) -> double {
            if (none) return 0.0;
            const double e = weight(clean(x[j]), j, m, top, t);
            if (last) return e;
            if (q) return fmax(e / z - (double) q[j], 0.0);
            return j == d ? 0.0 : e;
        };
        const int seg = (a.V + kThreads - 1) / kThreads, j0 = min(a.V, (int) threadIdx.x * seg), j1 = min(a.V, j0 + seg);
        double    sum = 0.0;
        for (int j = j0; j < j1; j++) sum += w_of(j);
        __shared__ double ss[kThreads];
        __shared__ double tot;
        __shared__ int    pick, lastw;
        __syncthreads();
        ss[threadIdx.x] = sum;
        __syncthreads();
        if (threadIdx.x == 0) {
            double c = 0.0;
            for (int i = 0; i < kThreads; i++) {
                const double v = ss[i];
                ss[i]          = c;
                c += v;
            }
            tot   = c;
            pick  = INT32_MAX;
            lastw = -1;
        }
        __syncthreads();
        const double goal = (double) a.us[s] * tot;
        double       c    = ss[threadIdx.x];
        for (int j = j0; j < j1; j++) {
            const double w = w_of(j);
            c += w;
            if (w > 0.0) {
                atomicMax(&lastw, j);
                if (c > goal) {
                    atomicMin(&pick, j);
                    break;
                }
            }
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            a.out_ids[r] = tot > 0.0 ? (pick != INT32_MAX ? pick : lastw) : top;
            a.out_n[s]   = r - r0 + 1;
        }
        __syncthreads();
    }
}

}  // namespace

size_t verify_sample_work_size(const srhpm_ctx *, int, int, int) { return 0; }

int verify_sample_run(srhpm_ctx * ctx, const SampleView & v, void *, size_t, cudaStream_t stream) {
    const int st = cuda_status(launch_k_pdl(verify_sample_kernel, dim3(v.S), dim3(kThreads), 0, stream, v));
    ctx->launches.fetch_add(1);
    return st;
}

}  // namespace srhpm
