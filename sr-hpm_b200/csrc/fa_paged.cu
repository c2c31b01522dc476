// Attention of a batch's new tokens over a paged KV cache: one CTA per (row, head), a warp per cached token.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>

#include "internal.h"
#include "launch.cuh"
#include "ptx.cuh"

namespace srhpm {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float cache_value(const uint8_t * row, int d, int q8) {
    if (!q8) return __half2float(reinterpret_cast<const __half *>(row)[d]);
    const uint8_t * b = row + (d >> 5) * 34;
    const float     s = __half2float(*reinterpret_cast<const __half *>(b));
    return __half2float(__float2half_rn(s * (float) (int8_t) b[2 + (d & 31)]));
}

__global__ void __launch_bounds__(128) fa_paged_kernel(const FaPagedView a, int32_t * status) {
    const int t = blockIdx.x, h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_launch_dependents();
    pdl_wait();
    if (t >= a.q_start[a.S]) return;
    int lo = 0, hi = a.S;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.q_start[mid] <= t) {
            lo = mid;
        } else {
            hi = mid;
        }
    }
    const int D = a.c.D, e = D / 32, q8 = a.c.type == SRHPM_TYPE_Q8_0, g = h / (a.H / a.c.Hkv);
    const int n = a.q_start[lo + 1] - a.q_start[lo], p = a.kv_len[lo] - n + t - a.q_start[lo];
    float     q[8];
    for (int i = 0; i < e; i++) {
        const uint8_t * src = a.q + (int64_t) t * a.qnb1 + (int64_t) h * a.qnb2;
        q[i] = a.f32 ? reinterpret_cast<const float *>(src)[i * 32 + lane]
                     : __half2float(reinterpret_cast<const __half *>(src)[i * 32 + lane]);
    }
    float     m = -INFINITY, l = 0.0f, acc[8] = {};
    const int first = a.window > 0 ? max(0, p - a.window + 1) : 0;
    const int end   = (int) min((int64_t) p + 1, (int64_t) a.cols * a.c.page);
    for (int j = first + warp; j < end; j += 4) {
        const int page = reinterpret_cast<const int32_t *>(a.table + (int64_t) lo * a.tstride)[j / a.c.page];
        const bool ok  = page >= 0 && page < a.c.n_pages;
        if (!ok && lane == 0) atomicExch(status, kErrPage);
        const uint8_t * kr = a.c.k + (int64_t) page * a.c.knb3 + (int64_t) (j % a.c.page) * a.c.knb1 + (int64_t) g * a.c.knb2;
        const uint8_t * vr = a.c.v + (int64_t) page * a.c.vnb3 + (int64_t) (j % a.c.page) * a.c.vnb1 + (int64_t) g * a.c.vnb2;
        float           s  = 0.0f;
        for (int i = 0; i < e; i++) s = fmaf(q[i], ok ? cache_value(kr, i * 32 + lane, q8) : 0.0f, s);
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        s *= a.scale;
        if (a.softcap != 0.0f) s = a.softcap * tanhf(s / a.softcap);
        const float mn = fmaxf(m, s), al = expf(m - mn), w = expf(s - mn);
        l = l * al + w;
        for (int i = 0; i < e; i++) acc[i] = acc[i] * al + w * (ok ? cache_value(vr, i * 32 + lane, q8) : 0.0f);
        m = mn;
    }
    __shared__ float sm[4], sl[4], sa[4][256];
    if (lane == 0) {
        sm[warp] = m;
        sl[warp] = l;
    }
    for (int i = 0; i < e; i++) sa[warp][i * 32 + lane] = acc[i];
    __syncthreads();
    const float sink = a.sinks ? a.sinks[h] : -INFINITY;
    const float M    = fmaxf(fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3])), sink);
    float       L    = M > -INFINITY ? expf(sink - M) : 0.0f;
    for (int w = 0; w < 4; w++) L += sl[w] > 0.0f ? sl[w] * expf(sm[w] - M) : 0.0f;
    for (int d = threadIdx.x; d < D; d += 128) {
        float o = 0.0f;
        for (int w = 0; w < 4; w++) o += sl[w] > 0.0f ? sa[w][d] * expf(sm[w] - M) : 0.0f;
        o             = L > 0.0f ? o / L : 0.0f;
        uint8_t * dst = a.dst + (int64_t) h * a.dnb1 + (int64_t) t * a.dnb2;
        if (a.f32) {
            reinterpret_cast<float *>(dst)[d] = o;
        } else {
            reinterpret_cast<__half *>(dst)[d] = __float2half_rn(o);
        }
    }
}

}  // namespace

size_t fa_paged_work_size(const srhpm_ctx *, int, int, int, int, int) { return 0; }

int fa_paged_run(srhpm_ctx * ctx, const FaPagedView & v, void *, size_t, cudaStream_t stream) {
    const int st = cuda_status(launch_k_pdl(fa_paged_kernel, dim3(v.T, v.H), dim3(128), 0, stream, v, ctx->d_status));
    ctx->launches.fetch_add(1);
    return st;
}

}  // namespace srhpm
