// The operators that keep a paged KV cache for a batch of sequences:
//   page_plan      block table entries, row starts, cache lengths, positions and slots of a step, from the sequences'
//                  lengths on the device (no host round trip, so a captured step replays with new lengths)
//   rope_kv_paged  NeoX rotary embedding of a fused QKV row; the turned queries go to the attention's input, the turned
//                  keys and the values into the cache rows that the slots name
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "fastdiv.cuh"
#include "internal.h"
#include "launch.cuh"
#include "ptx.cuh"

namespace srhpm {
namespace {

// ---- page plan ---------------------------------------------------------------------------------------------------
// With P slots per page, have_s = max(ceil(past_s / P), held_s) and want_s = ceil((past_s + new_s) / P): rows start at the
// exclusive sum of new, and sequence s takes max(want_s - have_s, 0) pages behind those of the sequences before it. Both sums run over
// all sequences, and every row needs its sequence's part of them. A step moves a few bytes per sequence and 12 per row,
// so launches and round trips to memory are what it costs: there is ONE launch, in which every CTA takes both sums
// itself (S <= 8192 lengths from L2, kept in shared memory) and then fills its share of rows and table entries, instead
// of a scan kernel with a fill kernel behind it. 8 sequences 4.9 us on the GPU (as a launch of its own 6.2), 1024 with 249886
// rows 16.4, 8192 152: the sums 2.5, 2.8 and 18, the rows 3, and in CTA 0 the walk for n_taken 0.7, 11 and 140.
constexpr int kPlanThreads = 1024;

struct PlanArgs {
    const int32_t * past;
    const int32_t * fresh;
    const int32_t * held;  // or null: ceil(past / P)
    int             S, P;
    uint8_t *       table;
    int64_t         tstride;  // bytes
    int             cols;
    const int32_t * free_pages;
    int             n_free;
    const int32_t * free_head;  // or null (0)
    int             n_rows;
    int32_t *       q_start;
    int32_t *       kv_len;
    int32_t *       pos;
    int64_t *       slots;
    int32_t *       status;
    int32_t *       n_taken;
};

__device__ __forceinline__ int64_t warp_incl(int64_t v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    return v;
}

// inclusive sum over the CTA's threads; sp: 32 words of shared memory. Ends with every thread past its reads of sp.
__device__ __forceinline__ int64_t cta_incl(int64_t v, int64_t * sp, int64_t * total) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
    v              = warp_incl(v);
    if (lane == 31) sp[warp] = v;
    __syncthreads();
    if (warp == 0) {
        const int64_t u = warp_incl(lane < nw ? sp[lane] : 0);
        sp[lane]        = u;
    }
    __syncthreads();
    const int64_t r = v + (warp ? sp[warp - 1] : 0);
    *total          = sp[nw - 1];
    __syncthreads();
    return r;
}

// pages that the table row of sequence s names, and those that it wants beside them
__device__ __forceinline__ int64_t held_of(const PlanArgs & a, int s, int64_t past) {
    const int64_t full = (past + a.P - 1) / a.P;
    return a.held ? max(full, (int64_t) a.held[s]) : full;
}
__device__ __forceinline__ int64_t need_of(const PlanArgs & a, int64_t past, int64_t fresh, int64_t have) {
    return max((past + fresh + a.P - 1) / a.P - have, (int64_t) 0);
}

__global__ void __launch_bounds__(kPlanThreads) page_plan_kernel(const PlanArgs a) {
    extern __shared__ int32_t sh[];
    int32_t *          start = sh;              // [S + 1] first row of each sequence (saturated)
    int32_t *          first = sh + a.S + 1;    // [S] index of its first new page in the free list (0: needs none), -1: refused
    __shared__ int64_t sp[32];
    pdl_launch_dependents();
    pdl_wait();
    const int64_t head = a.free_head ? (int64_t) *a.free_head : 0;
    int64_t       rows0 = 0, need0 = 0;
    for (int s0 = 0; s0 < a.S; s0 += blockDim.x) {
        const int     s   = s0 + threadIdx.x;
        const bool    in  = s < a.S;
        const int64_t pa  = in ? a.past[s] : 0, nw = in ? a.fresh[s] : 0;
        int64_t       all;
        const int64_t row_end = rows0 + cta_incl(nw > 0 ? nw : 0, sp, &all);
        rows0 += all;
        const int64_t have = in ? held_of(a, s, pa) : 0, want = (pa + nw + a.P - 1) / a.P;
        int           st   = SRHPM_PAGES_OK;
        if (pa < 0 || nw < 0) {
            st = SRHPM_PAGES_BAD_LENGTH;
        } else if (row_end > a.n_rows) {
            st = SRHPM_PAGES_NO_ROWS;
        } else if (want > a.cols || pa + nw > INT32_MAX) {
            st = SRHPM_PAGES_TABLE_FULL;
        }
        const int64_t need = st == SRHPM_PAGES_OK ? need_of(a, pa, nw, have) : 0;
        const int64_t end  = need0 + cta_incl(need, sp, &all);
        need0 += all;
        if (need > 0 && (head < 0 || head + end > a.n_free)) st = SRHPM_PAGES_NONE_FREE;
        // pages handed out: the end of the last sequence that got its own (ends rise, so it is their maximum)
        if (in) {
            start[s] = (int32_t) min(row_end - max(nw, (int64_t) 0), (int64_t) INT32_MAX);
            first[s] = st != SRHPM_PAGES_OK ? -1 : need > 0 ? (int32_t) (head + end - need) : 0;
            if (blockIdx.x == 0) {
                a.q_start[s] = start[s];
                a.kv_len[s]  = st == SRHPM_PAGES_OK ? (int32_t) (pa + nw) : 0;
                a.status[s]  = st;
            }
        }
    }
    if (threadIdx.x == 0) {
        start[a.S] = (int32_t) min(rows0, (int64_t) INT32_MAX);
        if (blockIdx.x == 0) a.q_start[a.S] = start[a.S];
    }
    __syncthreads();
    if (blockIdx.x == 0 && threadIdx.x < 32) {
        int32_t taken = 0;
        for (int s = threadIdx.x; s < a.S; s += 32) {
            if (first[s] >= 0) {
                const int64_t pa = a.past[s], nw = a.fresh[s];
                const int     need = (int) need_of(a, pa, nw, held_of(a, s, pa));
                if (need > 0) taken = max(taken, (int32_t) (first[s] - head + need));
            }
        }
        taken = __reduce_max_sync(0xffffffffu, taken);
        if (threadIdx.x == 0) *a.n_taken = taken;
    }
    // new table entries: a warp per sequence
    const int wid = (blockIdx.x * blockDim.x + threadIdx.x) >> 5, nwarp = (gridDim.x * blockDim.x) >> 5;
    for (int s = wid; s < a.S; s += nwarp) {
        if (first[s] < 0) continue;
        const int64_t pa = a.past[s], nw = a.fresh[s];
        const int     have = (int) held_of(a, s, pa), need = (int) need_of(a, pa, nw, have);
        int32_t *     row = reinterpret_cast<int32_t *>(a.table + (int64_t) s * a.tstride);
        for (int c = threadIdx.x & 31; c < need; c += 32) row[have + c] = a.free_pages[first[s] + c];
    }
    // rows: the sequence by bisection of the starts; a row in a page that was there reads the table, one in a new page
    // the free list (the entry may not be in the table yet: another CTA writes it)
    for (int64_t t = (int64_t) blockIdx.x * blockDim.x + threadIdx.x; t < a.n_rows; t += (int64_t) gridDim.x * blockDim.x) {
        int32_t pos  = 0;
        int64_t slot = -1;
        if (t < start[a.S]) {
            int lo = 0, hi = a.S;  // start[lo] <= t < start[hi]
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (start[mid] <= t) {
                    lo = mid;
                } else {
                    hi = mid;
                }
            }
            if (first[lo] >= 0) {
                const int32_t pa = a.past[lo];
                pos              = pa + (int32_t) (t - start[lo]);
                const int c = pos / a.P, have = (int) held_of(a, lo, pa);
                const int32_t page =
                    c < have ? reinterpret_cast<const int32_t *>(a.table + (int64_t) lo * a.tstride)[c]
                             : a.free_pages[first[lo] + c - have];
                slot = page < 0 ? -1 : (int64_t) page * a.P + pos % a.P;
            }
        }
        a.pos[t]   = pos;
        a.slots[t] = slot;
    }
}

// ---- RoPE and the paged store ------------------------------------------------------------------------------------
// Per token row of (H + 2 Hkv) heads: pairs (x_j, x_{j + D/2}) of the query and key heads turn by the angle
// pos * base^(-2j/D). At position 10^5 a 32-bit product of the two is off by 10^-2 of a turn, so the angle is taken in
// 64 bits (the frequencies once on the host, one product and one reduction to a fraction of a turn per angle) and only
// its fraction goes to the 32-bit sine and cosine. The D/2 angles of a token serve all its heads: they are computed by
// the first threads into shared memory while the row's loads are in flight. Bandwidth bound: a row is read once and
// every output written once. A thread holds 4 pairs (two 16-byte loads); a row's loads go out before its angles. 8192 rows
// of 32 + 2 * 8 heads of 128 into f16 pages: 49 us, 0.94 of the copy rate; 4001 rows of 24 + 2 * 4 of 256 into q8_0: 32.5,
// 0.89; 9 rows 4.2 (the launch). q4_0 pages: 62 us, and 4001 rows of 24 + 2 * 4 of 256 41 (q8_0 34): the numbers take a third of the
// instructions, 66 % of the issue slots are used, and half of the SM's threads wait at 64 registers with 52 bytes spilled. The rare
// rotation in 64 bits has registers of its own (in the loop 8 us more, capped at 3 CTAs per SM by them).
constexpr int kStoreThreads = 256;
constexpr int kMaxHalf      = 128;

struct StoreArgs {
    const uint8_t * qkv;
    int64_t         ldb;
    int             n, H, Hkv, D;
    FastDiv         by_units, by_page;
    const int32_t * pos;
    const int64_t * slots;
    uint8_t *       q;  // token stride qnb1, head stride qnb2
    int64_t         qnb1, qnb2;
    uint8_t *       kc;
    int64_t         knb1, knb2, knb3;
    uint8_t *       vc;
    int64_t         vnb1, vnb2, vnb3;
    int             page;
    int64_t         n_slots;
    int             q8mode;
    double          freq[kMaxHalf];  // base^(-2j/D) / (2 pi): turns per position
};

// 4 values as f32 or f16
template <bool F16> __device__ __forceinline__ void put4(uint8_t * dst, int j, float4 v) {
    if constexpr (F16) {
        const __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
        *reinterpret_cast<uint2 *>(dst + 2 * j) =
            make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
    } else {
        *reinterpret_cast<float4 *>(dst + 4 * j) = v;
    }
}

// 4 of the 32 values of a q8_0 block; the block's 8 threads are 8 consecutive lanes (mask: those lanes)
__device__ __forceinline__ void put4_q8(uint8_t * dst, int j, float4 v, int mode, uint32_t mask) {
    float amax = fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w)));
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(mask, amax, o));
    const float dd = __fdiv_rn(amax, 127.0f);
    int         q[4];
    const float x[4] = { v.x, v.y, v.z, v.w };
    if (mode == SRHPM_Q8_0_ACT_SIMD) {
        const float id = amax != 0.0f ? __fdiv_rn(127.0f, amax) : 0.0f;
#pragma unroll
        for (int e = 0; e < 4; e++) q[e] = __float2int_rn(__fmul_rn(x[e], id));
    } else {
        const float id = dd != 0.0f ? __fdiv_rn(1.0f, dd) : 0.0f;
#pragma unroll
        for (int e = 0; e < 4; e++) q[e] = (int) roundf(__fmul_rn(x[e], id));
    }
    uint8_t * b = dst + (j >> 5) * 34;
    if ((j & 31) == 0) *reinterpret_cast<__half *>(b) = __float2half_rn(dd);
    uint16_t * w = reinterpret_cast<uint16_t *>(b + 2 + (j & 31));
    w[0]         = (uint16_t) ((q[0] & 0xff) | (q[1] & 0xff) << 8);
    w[1]         = (uint16_t) ((q[2] & 0xff) | (q[3] & 0xff) << 8);
}

// what the 8 lanes of a q4_0 block need: -1/8 of its value of largest size (the first of equals; a NaN is never it) and the
// reciprocal
struct Step4 {
    float d, id;
};
__device__ __forceinline__ Step4 step_q4(float4 v, uint32_t mask) {
    const float x[4] = { v.x, v.y, v.z, v.w };
    float       m = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; e++) m = fabsf(x[e]) > fabsf(m) ? x[e] : m;
#pragma unroll
    for (int o = 1; o <= 4; o <<= 1) {
        const float w = __shfl_xor_sync(mask, m, o);
        if (fabsf(w) > fabsf(m) || (fabsf(w) == fabsf(m) && (threadIdx.x & o))) m = w;
    }
    const float d = m * -0.125f;
    return { d, d != 0.0f ? __frcp_rn(d) : 0.0f };
}
// The numbers of 4 values, a byte each: x / d + 8.5 rounded down, 0 to 15 (NaN: 0). Added to 256 rounding down, the sum's bits hold
// the number above 15 places of the fraction: the conversion instruction has an eighth of that rate. near: the rounding of a
// rotation may decide, as a value stands within 2^-15 of the border of two numbers, or within 2^-14 of the step's size at its other
// end (16.5), where it and not the step's might be the largest.
__device__ __forceinline__ uint32_t numbers_q4(float4 v, float id, bool & near) {
    const float x[4] = { v.x, v.y, v.z, v.w };
    float       top = 0.0f;
    uint32_t    n[4], low = 0x7fff;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const float y = __fadd_rn(__fmul_rn(x[e], id), 8.5f);
        top  = fmaxf(top, y);
        n[e] = __float_as_uint(__fadd_rd(fminf(fmaxf(y, 0.0f), 15.75f), 256.0f));
        low  = min(low, (n[e] + 1) & 0x7fffu);
    }
    near |= low < 2 || top > 16.5f - 0x1p-14f;
    return (n[0] >> 15 & 0xfu) | (n[1] >> 7 & 0xf00u) | (n[2] << 1 & 0xf0000u) | (n[3] << 9 & 0xf000000u);
}
// 4 of the 32 values of a q4_0 block: byte j holds number j in its low and number j + 16 in its high half
__device__ __forceinline__ void put4_q4(uint8_t * dst, int j, uint32_t q, float d, uint32_t mask) {
    const uint32_t up = __shfl_xor_sync(mask, q, 4);
    uint8_t *      b  = dst + (j >> 5) * 18;
    if ((j & 31) == 0) *reinterpret_cast<__half *>(b) = __float2half_rn(d);
    if ((j & 16) == 0) {
        const uint32_t w = q | up << 4;
        uint16_t *     p = reinterpret_cast<uint16_t *>(b + 2 + (j & 15));
        p[0]             = (uint16_t) w;
        p[1]             = (uint16_t) (w >> 16);
    }
}

// 4 pairs of a key's block and the one half a head further, turned in 64 bits (8 lanes, 32 pairs). Not inlined and from the row
// itself: the registers that it needs would cost the kernel a third of its warps.
__device__ __noinline__ void redo_q4(const float * x, int half, double pos, const double * freq, uint8_t * dst, int j, uint32_t mask) {
    float l[4] = {}, h[4] = {};
#pragma unroll 1
    for (int e = 0; e < 4; e++) {
        double turns = pos * freq[j + e], s, c;
        turns -= rint(turns);
        sincospi(2.0 * turns, &s, &c);
        const double a = x[j + e], b = x[half + j + e];
        const float  nl = (float) (a * c - b * s), nh = (float) (a * s + b * c);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            l[i] = i == e ? nl : l[i];
            h[i] = i == e ? nh : h[i];
        }
    }
    const float4 lo = make_float4(l[0], l[1], l[2], l[3]), hi = make_float4(h[0], h[1], h[2], h[3]);
    const Step4  sl = step_q4(lo, mask), sh = step_q4(hi, mask);
    bool         near = false;
    put4_q4(dst, j, numbers_q4(lo, sl.id, near), sl.d, mask);
    put4_q4(dst, half + j, numbers_q4(hi, sh.id, near), sh.d, mask);
}

template <bool QF16, int KV>
__global__ void __launch_bounds__(kStoreThreads, 4) rope_kv_paged_kernel(const __grid_constant__ StoreArgs a) {
    __shared__ __align__(16) float cs[2][kMaxHalf], sn[2][kMaxHalf];
    constexpr int NU = 3;  // units of a thread in flight: 48 heads of 128 or 32 of 256 in one turn
    pdl_launch_dependents();
    pdl_wait();
    const int half = a.D >> 1, units = half >> 2;  // 4-pair units per head
    const int total = (a.H + 2 * a.Hkv) * units;
    int       par = 0;
    for (int t = blockIdx.x; t < a.n; t += gridDim.x, par ^= 1) {
        const uint8_t * row  = a.qkv + (int64_t) t * a.ldb;
        const int64_t   slot = a.slots[t];
        const bool      keep = slot >= 0 && slot < a.n_slots;
        float4          lo[NU], hi[NU];
        // units is a multiple of 8, so 8 consecutive lanes hold 32 consecutive values of one head (a q8_0 block)
        auto load = [&](int u0) {
#pragma unroll
            for (int k = 0; k < NU; k++) {
                const int u = u0 + k * kStoreThreads;
                if (u < total) {
                    const int     hh = a.by_units.div(u), j = (u - hh * units) * 4;
                    const float * x  = reinterpret_cast<const float *>(row) + hh * a.D;
                    lo[k] = __ldcs(reinterpret_cast<const float4 *>(x + j));
                    hi[k] = __ldcs(reinterpret_cast<const float4 *>(x + half + j));
                }
            }
        };
        load(threadIdx.x);
        if (threadIdx.x < half) {
            double turns = (double) a.pos[t] * a.freq[threadIdx.x];
            turns -= rint(turns);
            float s, c;
            sincospif((float) (2.0 * turns), &s, &c);
            cs[par][threadIdx.x] = c;
            sn[par][threadIdx.x] = s;
        }
        const int64_t pg = !keep ? 0 : a.n_slots <= INT32_MAX ? a.by_page.div((int) slot) : slot / a.page, off = keep ? slot - pg * a.page : 0;
        uint8_t *     kd = a.kc + pg * a.knb3 + off * a.knb1;
        uint8_t *     vd = a.vc + pg * a.vnb3 + off * a.vnb1;
        uint8_t *     qd = a.q + (int64_t) t * a.qnb1;
        __syncthreads();  // one per token: the next one writes the other half of the angles
        for (int u0 = threadIdx.x; u0 < total; u0 += NU * kStoreThreads) {
            if (u0 != threadIdx.x) load(u0);
#pragma unroll
            for (int k = 0; k < NU; k++) {
                const int u = u0 + k * kStoreThreads;
                if (u >= total) break;
                const int hh = a.by_units.div(u), j = (u - hh * units) * 4;
                if (hh < a.H + a.Hkv) {
                    const float4 c = *reinterpret_cast<const float4 *>(cs[par] + j), s = *reinterpret_cast<const float4 *>(sn[par] + j);
                    const float4 l = lo[k], h = hi[k];
                    lo[k] = make_float4(l.x * c.x - h.x * s.x, l.y * c.y - h.y * s.y, l.z * c.z - h.z * s.z, l.w * c.w - h.w * s.w);
                    hi[k] = make_float4(l.x * s.x + h.x * c.x, l.y * s.y + h.y * c.y, l.z * s.z + h.z * c.z, l.w * s.w + h.w * c.w);
                }
                if (hh < a.H) {
                    uint8_t * d = qd + (int64_t) hh * a.qnb2;
                    put4<QF16>(d, j, lo[k]);
                    put4<QF16>(d, half + j, hi[k]);
                } else if (keep) {
                    const bool isk = hh < a.H + a.Hkv;
                    const int  g   = hh - a.H - (isk ? 0 : a.Hkv);
                    uint8_t *  d   = isk ? kd + (int64_t) g * a.knb2 : vd + (int64_t) g * a.vnb2;
                    [[maybe_unused]] const uint32_t oct = 0xffu << (threadIdx.x & 24);
                    if constexpr (KV == SRHPM_TYPE_Q4_0) {
                        const Step4 sl = step_q4(lo[k], oct), sh = step_q4(hi[k], oct);
                        bool           near = false;
                        const uint32_t ql = numbers_q4(lo[k], sl.id, near), qh = numbers_q4(hi[k], sh.id, near);
                        // a number hangs on the 32-bit rotation only where a value is next to a border: there the whole
                        // block's are taken in 64 bits (one block in 500)
                        if (isk && (__ballot_sync(oct, near) & oct)) {
                            redo_q4(reinterpret_cast<const float *>(row) + hh * a.D, half, (double) a.pos[t], a.freq, d, j, oct);
                        } else {
                            put4_q4(d, j, ql, sl.d, oct);
                            put4_q4(d, half + j, qh, sh.d, oct);
                        }
                    } else if constexpr (KV == SRHPM_TYPE_Q8_0) {
                        put4_q8(d, j, lo[k], a.q8mode, oct);
                        put4_q8(d, half + j, hi[k], a.q8mode, oct);
                    } else {
                        put4<true>(d, j, lo[k]);
                        put4<true>(d, half + j, hi[k]);
                    }
                }
            }
        }
    }
}

}  // namespace

int page_plan_run(srhpm_ctx * ctx, const int32_t * n_past, const int32_t * n_new, const int32_t * n_held, int S, int page, void * table,
                  int64_t tstride, int cols, const int32_t * free_pages, int n_free, const int32_t * free_head,
                  int n_rows, int32_t * q_start, int32_t * kv_len, int32_t * pos, int64_t * slots, int32_t * status,
                  int32_t * n_taken, cudaStream_t stream) {
    PlanArgs a;
    a.past       = n_past;
    a.fresh      = n_new;
    a.held       = n_held;
    a.S          = S;
    a.P          = page;
    a.table      = reinterpret_cast<uint8_t *>(table);
    a.tstride    = tstride;
    a.cols       = cols;
    a.free_pages = free_pages;
    a.n_free     = n_free;
    a.free_head  = free_head;
    a.n_rows     = n_rows;
    a.q_start    = q_start;
    a.kv_len     = kv_len;
    a.pos        = pos;
    a.slots      = slots;
    a.status     = status;
    a.n_taken    = n_taken;
    const size_t smem = (size_t) (2 * S + 1) * sizeof(int32_t);  // at most 64 KB
    if (smem > 48 * 1024) {
        const int st = cuda_status(cudaFuncSetAttribute(page_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                        (int) ((2 * kPlanMaxSeqs + 1) * sizeof(int32_t))));
        if (st != SRHPM_OK) return st;
    }
    const int64_t want = std::max<int64_t>(((int64_t) n_rows + kPlanThreads - 1) / kPlanThreads, (S + 31) / 32);
    const int     grid = (int) std::max<int64_t>(1, std::min<int64_t>(ctx->num_sms, want));
    const cudaError_t e = launch_k_pdl(page_plan_kernel, dim3(grid), dim3(kPlanThreads), smem, stream, a);
    ctx->launches.fetch_add(1);
    return cuda_status(e);
}

int rope_kv_paged_run(srhpm_ctx * ctx, const uint8_t * qkv, int64_t ldb, int n, int H, int Hkv, int D,
                      const int32_t * pos, const int64_t * slots, float theta_base, const srhpm_tensor * q_out,
                      const PagedCache & c, cudaStream_t stream) {
    StoreArgs a;
    a.qkv     = qkv;
    a.ldb     = ldb;
    a.n       = n;
    a.H       = H;
    a.Hkv     = Hkv;
    a.D       = D;
    a.by_units = FastDiv::of((uint32_t) (D / 8));
    a.pos     = pos;
    a.slots   = slots;
    a.q       = reinterpret_cast<uint8_t *>(q_out->data);
    a.qnb1    = (int64_t) q_out->nb[1];
    a.qnb2    = (int64_t) q_out->nb[2];
    a.kc      = const_cast<uint8_t *>(c.k);
    a.knb1    = c.knb1;
    a.knb2    = c.knb2;
    a.knb3    = c.knb3;
    a.vc      = const_cast<uint8_t *>(c.v);
    a.vnb1    = c.vnb1;
    a.vnb2    = c.vnb2;
    a.vnb3    = c.vnb3;
    a.page    = c.page;
    a.n_slots = c.n_pages * c.page;
    a.by_page = FastDiv::of((uint32_t) c.page);
    a.q8mode  = ctx->q8_0_act_mode;
    // the frequencies of a model stay the same from call to call: 128 powers took the host 5 us of a 9-row step
    {
        std::lock_guard<std::mutex> lk(ctx->rope_mu);  // threads that share the context
        if (ctx->rope_base != theta_base || ctx->rope_dim != D) {
            const double two_pi = 6.283185307179586476925286766559;
            for (int j = 0; j < D / 2; j++) ctx->rope_freq[j] = pow((double) theta_base, -2.0 * j / D) / two_pi;
            ctx->rope_base = theta_base;
            ctx->rope_dim  = D;
        }
        std::copy(ctx->rope_freq, ctx->rope_freq + D / 2, a.freq);
    }
    const int         grid = std::min(n, 8 * ctx->num_sms);
    const bool qf = q_out->type == SRHPM_TYPE_F16;
    auto       kern = c.type == SRHPM_TYPE_Q4_0   ? (qf ? rope_kv_paged_kernel<true, SRHPM_TYPE_Q4_0> : rope_kv_paged_kernel<false, SRHPM_TYPE_Q4_0>)
                      : c.type == SRHPM_TYPE_Q8_0 ? (qf ? rope_kv_paged_kernel<true, SRHPM_TYPE_Q8_0> : rope_kv_paged_kernel<false, SRHPM_TYPE_Q8_0>)
                                                  : (qf ? rope_kv_paged_kernel<true, SRHPM_TYPE_F16> : rope_kv_paged_kernel<false, SRHPM_TYPE_F16>);
    const cudaError_t e = launch_k_pdl(kern, dim3(grid), dim3(kStoreThreads), 0, stream, a);
    ctx->launches.fetch_add(1);
    return cuda_status(e);
}

}  // namespace srhpm
