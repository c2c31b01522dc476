// Rules on the logits of the rows that a step scores (srhpm_adjust_logits): biases of single tokens, penalties for tokens
// that the sequence has said already, and token masks.
//
// A row is a copy with a few changed places, so the copy is what costs: 8 bytes per logit (with out = logits only what a mask
// takes away is written). A CTA has one row's slice of kSlice tokens: it loads the slice into registers, counts the window's
// tokens that fall into the slice in shared memory meanwhile, writes the slice with the mask applied, and then goes through
// the window and the biases once more: the first visitor of a token takes its count and writes its value. No sort, no hash, and the same
// result whatever the order of the atomics: counts are whole numbers, and a token that is biased twice takes the later value.
#include <cuda_runtime.h>

#include <algorithm>

#include "internal.h"
#include "launch.cuh"
#include "ptx.cuh"

namespace srhpm {
namespace {

constexpr int kThreads = 512;
constexpr int kSlice   = 8192;
constexpr int kVec     = kSlice / kThreads / 4;  // groups of four of a thread

struct Args {
    LogitView v;
    int       slices;
};

template <bool VEC>
__global__ void __launch_bounds__(kThreads) adjust_logits_kernel(const __grid_constant__ Args a) {
    extern __shared__ uint32_t sh[];
    uint32_t * cnt = sh;           // [kSlice] times in the window
    uint32_t * bix = sh + kSlice;  // [kSlice] 1 + index of the token's bias
    const LogitView & v = a.v;
    const int         tid = threadIdx.x;
    const int         row = blockIdx.x / a.slices, x0 = (blockIdx.x - row * a.slices) * kSlice, nx = min(kSlice, v.V - x0);
    pdl_launch_dependents();
    pdl_wait();
    const int rows = v.q_start[v.S];
    if (row >= rows) return;  // padding
    const float * in  = reinterpret_cast<const float *>(v.logits + (int64_t) row * v.ldb) + x0;
    float *       out = reinterpret_cast<float *>(v.out + (int64_t) row * v.ldo) + x0;
    const bool    same = in == out;
    const uint32_t * mask = nullptr;
    if (v.mask) {
        const int mr = v.mask_row ? v.mask_row[row] : row;
        if (mr >= 0 && mr < v.n_masks) mask = reinterpret_cast<const uint32_t *>(v.mask + (int64_t) mr * v.ldm) + x0 / 32;
    }
    // the slice: group i of a thread has tokens 4 (i kThreads + tid) ..
    float4     x[kVec];
    const bool pass = !same || mask;
    if (pass) {
#pragma unroll
        for (int i = 0; i < kVec; i++) {
            const int at = 4 * (i * kThreads + tid);
            if constexpr (VEC) {
                if (at + 4 <= nx) {
                    x[i] = __ldcs(reinterpret_cast<const float4 *>(in + at));
                    continue;
                }
            }
            x[i].x = at < nx ? in[at] : 0.0f;
            x[i].y = at + 1 < nx ? in[at + 1] : 0.0f;
            x[i].z = at + 2 < nx ? in[at + 2] : 0.0f;
            x[i].w = at + 3 < nx ? in[at + 3] : 0.0f;
        }
    }
    // the row's sequence: starts at or before it
    int s = 0;
    for (int i0 = 0; i0 < v.S; i0 += kThreads) s += __syncthreads_count(i0 + tid < v.S && v.q_start[i0 + tid] <= row);
    s -= 1;
    const int first = s >= 0 ? max(v.q_start[s], 0) : 0;
    const int nh    = v.history && s >= 0 ? min(max(v.n_history[s], 0), v.cap) : 0;
    const int total = nh + row - first + 1;
    const int last  = v.last_n && s >= 0 ? v.last_n[s] : -1;
    const int begin = last < 0 ? 0 : max(total - last, 0);
    const bool pen  = s >= 0 && (v.repeat || v.frequency || v.presence) && begin < total;
    int b0 = 0, b1 = 0;
    if (v.n_bias && s >= 0) {
        b0 = min(max(v.bias_start[s], 0), v.n_bias);
        b1 = min(max(v.bias_start[s + 1], b0), v.n_bias);
    }
    const int32_t * said = v.history ? reinterpret_cast<const int32_t *>(v.history + (int64_t) max(s, 0) * v.ldh) : nullptr;
    auto token = [&](int j) { return j < nh ? said[j] : v.ids[first + j - nh]; };
    if (pen || b1 > b0) {
        uint4 * z = reinterpret_cast<uint4 *>(sh);
        for (int i = tid; i < 2 * kSlice / 4; i += kThreads) z[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        if (pen) {
            for (int j = begin + tid; j < total; j += kThreads) {
                const uint32_t k = (uint32_t) token(j) - (uint32_t) x0;
                if (k < (uint32_t) nx) atomicAdd(cnt + k, 1u);
            }
        }
        for (int j = b0 + tid; j < b1; j += kThreads) {
            const uint32_t k = (uint32_t) v.bias_ids[j] - (uint32_t) x0;
            if (k < (uint32_t) nx) atomicMax(bix + k, (uint32_t) j + 1u);
        }
    }
    if (pass) {
#pragma unroll
        for (int i = 0; i < kVec; i++) {
            const int at = 4 * (i * kThreads + tid);
            if (at >= nx) break;
            const uint32_t ok = mask ? mask[at >> 5] >> (at & 31) & 15u : 15u;
            if (same && ok == 15u) continue;
            if (!(ok & 1u)) x[i].x = -INFINITY;
            if (!(ok & 2u)) x[i].y = -INFINITY;
            if (!(ok & 4u)) x[i].z = -INFINITY;
            if (!(ok & 8u)) x[i].w = -INFINITY;
            if constexpr (VEC) {
                if (at + 4 <= nx) {
                    __stcs(reinterpret_cast<float4 *>(out + at), x[i]);
                    continue;
                }
            }
            out[at] = x[i].x;
            if (at + 1 < nx) out[at + 1] = x[i].y;
            if (at + 2 < nx) out[at + 2] = x[i].z;
            if (at + 3 < nx) out[at + 3] = x[i].w;
        }
    }
    if (!pen && b1 <= b0) return;
    __syncthreads();  // the slice is written, the counts are there
    const float rep = v.repeat ? v.repeat[s] : 1.0f, fr = v.frequency ? v.frequency[s] : 0.0f, pr = v.presence ? v.presence[s] : 0.0f;
    auto put = [&](uint32_t k, uint32_t times, uint32_t bi) {
        if (mask && !(mask[k >> 5] >> (k & 31) & 1u)) return;
        float l = in[k];
        if (bi) l += v.bias[bi - 1];
        if (times) {
            l = l > 0.0f ? __fdiv_rn(l, rep) : l * rep;
            l -= (float) times * fr + pr;
        }
        out[k] = l;
    };
    if (pen) {
        for (int j = begin + tid; j < total; j += kThreads) {
            const uint32_t k = (uint32_t) token(j) - (uint32_t) x0;
            if (k < (uint32_t) nx && cnt[k]) {
                const uint32_t times = atomicExch(cnt + k, 0u);
                if (times) put(k, times, atomicExch(bix + k, 0u));
            }
        }
        __syncthreads();  // biases of tokens in the window are done
    }
    for (int j = b0 + tid; j < b1; j += kThreads) {
        const uint32_t k = (uint32_t) v.bias_ids[j] - (uint32_t) x0;
        if (k < (uint32_t) nx) {
            const uint32_t bi = atomicExch(bix + k, 0u);
            if (bi) put(k, 0u, bi);
        }
    }
}

}  // namespace

int adjust_logits_run(srhpm_ctx * ctx, const LogitView & v, cudaStream_t stream) {
    Args a;
    a.v      = v;
    a.slices = (v.V + kSlice - 1) / kSlice;
    const int64_t grid = (int64_t) a.slices * v.T;
    if (grid > INT32_MAX) return SRHPM_UNSUPPORTED;
    const bool vec = ((reinterpret_cast<uintptr_t>(v.logits) | reinterpret_cast<uintptr_t>(v.out) | v.ldb | v.ldo) & 15) == 0;
    auto       kern = vec ? adjust_logits_kernel<true> : adjust_logits_kernel<false>;
    constexpr int smem = 2 * kSlice * 4;
    int st = cuda_status(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    if (st != SRHPM_OK) return st;
    st = cuda_status(launch_k_pdl(kern, dim3((unsigned) grid), dim3(kThreads), smem, stream, a));
    ctx->launches.fetch_add(1);
    return st;
}

}  // namespace srhpm
