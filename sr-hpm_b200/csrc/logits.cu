// Rules on the logits of the rows that a step scores (srhpm_adjust_logits): biases of single tokens, penalties for tokens
// that the sequence has said already, and token masks.
//
// A row is a copy with a few changed places, so the copy is what costs: 8 bytes per logit (with out = logits a row without a mask is
// touched only where a rule changes it). A CTA has a slice of kSlice tokens, of all rows of a sequence one after another where there are sequences enough,
// else of one row. The window's tokens that fall into the slice are counted in shared memory once per CTA; a warp has the same 512
// tokens of every row, lists those with a rule once, and from then on waits for no other: a row comes in, goes through the warp's
// shared memory, where 32 listed tokens at a time take their values, and out with the mask applied. From one row to the next the window
// moves by a token. 64 sequences of 2 to 8 rows of 151936, windows of 4096: 100 us, 4.6 TB/s of what has to move. (Four CTAs per SM,
// whose 64 registers spill, 121; sequences one after another in the grid 109, the last ones alone at its end; each row's window
// counted anew in each of its slices 201; listed tokens fetched and written behind the copy 154; barriers of the CTA around the
// listed tokens 142; rules applied by the lane that holds the token 180.)
// The result does not hang on the order of the atomics: counts are whole numbers, and a token that is biased twice takes the
// later value.
#include <cuda_runtime.h>

#include <algorithm>

#include "internal.h"
#include "launch.cuh"
#include "ptx.cuh"

namespace srhpm {
namespace {

constexpr int kThreads = 256;
constexpr int kSlice   = 4096;
constexpr int kVec     = kSlice / kThreads / 4;  // groups of four of a thread
constexpr int kWarpTok = 128 * kVec;             // tokens of a warp
constexpr uint32_t kListed = 1u << 31;           // beside a token's count
constexpr uint32_t kNoBias = 1u << 31;           // -0, which no sum shows: x + 0 would make +0 of -0
constexpr int kSmem = kSlice * 14;

struct Args {
    LogitView v;
    int       slices, by_seq;
};

template <bool VEC>
__global__ void __launch_bounds__(kThreads, 3) adjust_logits_kernel(const __grid_constant__ Args a) {
    static_assert(kVec == 4, "a thread's 16 tokens");
    extern __shared__ __align__(16) uint32_t cnt[];               // [kSlice] times in the window, kListed
    uint32_t * bix  = cnt + kSlice;                               // [kSlice] 1 + index of the token's bias, then its value
    float *    xs   = reinterpret_cast<float *>(bix + kSlice);    // [kSlice] the row
    uint16_t * list = reinterpret_cast<uint16_t *>(xs + kSlice) + (threadIdx.x >> 5) * kWarpTok;
    const LogitView & v = a.v;
    const int         tid = threadIdx.x, lane = tid & 31, w0 = (tid >> 5) * kWarpTok;
    // slice by slice with all sequences of each, so that those with many rows are spread over the grid; row by row otherwise
    const int unit = a.by_seq ? blockIdx.x % v.S : blockIdx.x / a.slices;
    const int x0 = (a.by_seq ? blockIdx.x / v.S : blockIdx.x - unit * a.slices) * kSlice, nx = min(kSlice, v.V - x0);
    pdl_launch_dependents();
    pdl_wait();
    int s, r0, r1, first;
    if (a.by_seq) {
        s     = unit;
        first = max(v.q_start[s], 0);
        r0    = first;
        r1    = min(v.q_start[s + 1], v.T);
    } else {
        r0 = unit;
        r1 = r0 + 1;
        if (r0 >= v.q_start[v.S]) return;  // padding
        s = -1;
        for (int i0 = 0; i0 < v.S; i0 += kThreads) s += __syncthreads_count(i0 + tid < v.S && v.q_start[i0 + tid] <= r0);
        if (s < 0) return;
        first = max(v.q_start[s], 0);
    }
    if (r0 >= r1) return;
    const bool same = v.logits == v.out;
    float4     x[kVec];  // group i of a lane has tokens w0 + 4 (32 i + lane) ..
    auto       in_row  = [&](int r) { return reinterpret_cast<const float *>(v.logits + (int64_t) r * v.ldb) + x0; };
    uint32_t   mw[kVec];  // their words of the mask
    auto       mask_row = [&](int r) { return v.mask && r < r1 ? v.mask_row ? v.mask_row[r] : r : -1; };
    auto       mask_of  = [&](int m) -> const uint32_t * {
        return m >= 0 && m < v.n_masks ? reinterpret_cast<const uint32_t *>(v.mask + (int64_t) m * v.ldm) + x0 / 32 : nullptr;
    };
    auto load = [&](const float * in, const uint32_t * mk) {
#pragma unroll
        for (int i = 0; i < kVec; i++) {
            const int at = w0 + 4 * (32 * i + lane);
            mw[i]        = mk && at < nx ? mk[at >> 5] : ~0u;
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
    };
    const uint32_t * mask = mask_of(mask_row(r0));
    if (!same || mask) load(in_row(r0), mask);
    int m_next = mask_row(r0 + 1);
    const int nh    = v.history ? min(max(v.n_history[s], 0), v.cap) : 0;
    const int last  = v.last_n ? v.last_n[s] : -1;
    int       total = nh + r0 - first + 1;
    int       begin = last < 0 ? 0 : max(total - last, 0);
    const bool pen  = (v.repeat || v.frequency || v.presence) && last != 0;
    int b0 = 0, b1 = 0;
    if (v.n_bias) {
        b0 = min(max(v.bias_start[s], 0), v.n_bias);
        b1 = min(max(v.bias_start[s + 1], b0), v.n_bias);
    }
    const int32_t * said = v.history ? reinterpret_cast<const int32_t *>(v.history + (int64_t) s * v.ldh) : nullptr;
    // place in the slice of the j-th token ahead of a row; those elsewhere are not below nx
    auto token = [&](int j) { return (uint32_t) *(j < nh ? said + j : v.ids + first + (j - nh)) - (uint32_t) x0; };
    const bool rules = pen || b1 > b0;
    int        n_list = 0;  // of the warp's tokens: those with a rule
    float      rep = 1.0f, fr = 0.0f, pr = 0.0f;
    if (rules) {
        uint4 * z = reinterpret_cast<uint4 *>(cnt);
        for (int i = tid; i < kSlice / 4; i += kThreads) z[i] = make_uint4(0, 0, 0, 0);
        z = reinterpret_cast<uint4 *>(bix);
        for (int i = tid; b1 > b0 && i < kSlice / 4; i += kThreads) z[i] = make_uint4(0, 0, 0, 0);
        if (v.repeat) rep = v.repeat[s];
        if (v.frequency) fr = v.frequency[s];
        if (v.presence) pr = v.presence[s];
        __syncthreads();
        if (pen) {
            constexpr int U = 8;  // tokens of a thread in flight
            for (int j0 = begin; j0 < total; j0 += U * kThreads) {
                uint32_t k[U];
#pragma unroll
                for (int u = 0; u < U; u++) {  // one load each, whichever list it is from, so that all are on their way at once
                    const int j = min(j0 + u * kThreads + tid, total - 1);
                    k[u]        = token(j);
                }
#pragma unroll
                for (int u = 0; u < U; u++) {
                    if (k[u] < (uint32_t) nx && j0 + u * kThreads + tid < total) atomicAdd(cnt + k[u], 1u);
                }
            }
        }
        for (int j = b0 + tid; j < b1; j += kThreads) {
            const uint32_t k = (uint32_t) v.bias_ids[j] - (uint32_t) x0;
            if (k < (uint32_t) nx) atomicMax(bix + k, (uint32_t) j + 1u);
        }
        __syncthreads();
        uint32_t hit = 0;  // of this lane's 16 tokens
#pragma unroll
        for (int i = 0; i < kVec; i++) {
            const int   at = w0 + 4 * (32 * i + lane);
            const uint4 c = *reinterpret_cast<const uint4 *>(cnt + at), b = b1 > b0 ? *reinterpret_cast<const uint4 *>(bix + at) : make_uint4(0, 0, 0, 0);
            hit |= ((c.x | b.x) != 0) << (4 * i) | ((c.y | b.y) != 0) << (4 * i + 1) | ((c.z | b.z) != 0) << (4 * i + 2) | ((c.w | b.w) != 0) << (4 * i + 3);
        }
        int to = __popc(hit);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, to, o);
            if (lane >= o) to += u;
        }
        n_list = __shfl_sync(0xffffffffu, to, 31);
        to -= __popc(hit);
        for (; hit; hit &= hit - 1) {
            const int e = __ffs(hit) - 1, k = w0 + 4 * (32 * (e >> 2) + lane) + (e & 3);
            cnt[k] |= kListed;
            list[to++] = (uint16_t) k;
        }
        __syncwarp();
        if (b1 > b0) {
            for (int i = lane; i < n_list; i += 32) {
                const uint32_t k = list[i], bi = bix[k];
                bix[k] = bi ? __float_as_uint(v.bias[bi - 1]) : kNoBias;
            }
        }
    }
    auto rule = [&](float l, uint32_t k) {
        if (b1 > b0) l += __uint_as_float(bix[k]);
        const uint32_t times = cnt[k] & ~kListed;
        if (times) {
            l = l > 0.0f ? __fdiv_rn(l, rep) : __fmul_rn(l, rep);  // each operation rounded by itself: no fused one
            l = __fsub_rn(l, __fadd_rn(__fmul_rn((float) times, fr), pr));
        }
        return l;
    };
    for (int r = r0; r < r1; r++) {
        const float * in   = in_row(r);
        float *       out  = reinterpret_cast<float *>(v.out + (int64_t) r * v.ldo) + x0;
        const bool    pass = !same || mask;  // the whole row goes through; else only the listed tokens
        uint32_t      add = ~0u, drop = ~0u;
        if (pen && r + 1 < r1) {
            add = token(total);
            if (last >= 0 && total + 1 - last > begin) drop = token(begin);
        }
        uint32_t ok = 0;
        if (pass) {
#pragma unroll
            for (int i = 0; i < kVec; i++) {
                const int at = w0 + 4 * (32 * i + lane);
                ok |= (mw[i] >> (at & 31) & 15u) << (4 * i);
                *reinterpret_cast<float4 *>(xs + at) = x[i];
            }
        }
        if (r + 1 < r1) {
            mask = mask_of(m_next);
            if (!same || mask) load(in_row(r + 1), mask);
            m_next = mask_row(r + 2);
        }
        __syncwarp();
        for (int i = lane; i < n_list; i += 32) {
            const uint32_t k = list[i];
            if (pass) {
                xs[k] = rule(xs[k], k);
            } else {
                out[k] = rule(in[k], k);
            }
        }
        __syncwarp();
        if (pass) {
#pragma unroll
            for (int i = 0; i < kVec; i++) {
                const int at = w0 + 4 * (32 * i + lane);
                if (at >= nx) break;
                float4         y = *reinterpret_cast<const float4 *>(xs + at);
                const uint32_t o = ok >> (4 * i);
                if (!(o & 1u)) y.x = -INFINITY;
                if (!(o & 2u)) y.y = -INFINITY;
                if (!(o & 4u)) y.z = -INFINITY;
                if (!(o & 8u)) y.w = -INFINITY;
                if constexpr (VEC) {
                    if (at + 4 <= nx) {
                        __stcs(reinterpret_cast<float4 *>(out + at), y);
                        continue;
                    }
                }
                out[at] = y.x;
                if (at + 1 < nx) out[at + 1] = y.y;
                if (at + 2 < nx) out[at + 2] = y.z;
                if (at + 3 < nx) out[at + 3] = y.w;
            }
        }
        if (r + 1 < r1 && pen) {  // the window of the next row: a token's count is its warp's own by now
            total++;
            if (last >= 0) begin = max(total - last, 0);
            if (add - (uint32_t) w0 < (uint32_t) kWarpTok && add < (uint32_t) nx) {
                const uint32_t old = cnt[add];
                __syncwarp();
                if (lane == 0) {
                    cnt[add] = (old | kListed) + 1;
                    if (!(old & kListed)) {
                        list[n_list] = (uint16_t) add;
                        bix[add]     = kNoBias;
                    }
                }
                if (!(old & kListed)) n_list++;
                __syncwarp();
            }
            if (drop - (uint32_t) w0 < (uint32_t) kWarpTok && drop < (uint32_t) nx && lane == 0) cnt[drop]--;
            __syncwarp();
        }
    }
}

}  // namespace

int adjust_logits_run(srhpm_ctx * ctx, const LogitView & v, cudaStream_t stream) {
    Args a;
    a.v      = v;
    a.slices = (v.V + kSlice - 1) / kSlice;
    // all rows of a sequence in one CTA where that leaves some CTAs for each SM
    a.by_seq           = (int64_t) v.S * a.slices >= 4 * (int64_t) ctx->num_sms;
    if ((int64_t) a.slices * std::max(v.S, v.T) > INT32_MAX) return SRHPM_UNSUPPORTED;
    const int64_t grid = (int64_t) a.slices * (a.by_seq ? v.S : v.T);
    const bool vec = ((reinterpret_cast<uintptr_t>(v.logits) | reinterpret_cast<uintptr_t>(v.out) | v.ldb | v.ldo) & 15) == 0;
    auto       kern = vec ? adjust_logits_kernel<true> : adjust_logits_kernel<false>;
    int        st   = cuda_status(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
    if (st != SRHPM_OK) return st;
    st = cuda_status(launch_k_pdl(kern, dim3((unsigned) grid), dim3(kThreads), kSmem, stream, a));
    ctx->launches.fetch_add(1);
    return st;
}

}  // namespace srhpm
