// What the kernels of attention over pages share: arguments, work items, and the cut of all items' units into equal parts.
#pragma once
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "fastdiv.cuh"
#include "internal.h"
#include "ptx.cuh"

namespace srhpm {
namespace fap {

constexpr float kLog2e   = 1.4426950408889634f;
constexpr float kLazy    = 8.0f;  // raise the running maximum only beyond 2^8
constexpr float kShift   = 7.0f;  // p is kept times 2^7
constexpr int   kMaxSeqs = 8192;

struct PArgs {
    const uint8_t * q;
    int64_t         qnb1, qnb2;
    uint8_t *       dst;
    int64_t         dnb1, dnb2;
    int             wide;  // dst and its strides are multiples of 32 bytes
    const uint8_t * table;
    int64_t         tstride;
    int             cols, page, n_pages, box;  // box: tokens of a TMA box (divides the page)
    const int32_t * q_start;
    const int32_t * kv_len;
    int             S, T, H, Hkv, G, window;
    FastDiv         byG, byPage;
    float           qscale;      // scale * log2e, or scale / softcap
    float           softcap_l2;  // softcap * log2e, 0 = none
    const float *   sinks;
    float *         part_acc;    // [2 n_cta][prow][D]
    float2 *        part_ms;     // [2 n_cta][prow] (max in log2 units, sum * 2^kShift)
    int4 *          desc;        // [n_cta][2]: parts of the item that a CTA opens and leaves unfinished, and its rows
    int             prow;        // rows of a record
    int32_t *       status;
};

// ---- work items --------------------------------------------------------------------------------------------------
struct Span {
    int kt0, nkv;  // first tile, tiles (0: nothing visible)
    int lo, hi;    // visible tokens of any row
    int units;     // max(nkv, 1)
};

// q_start, clamped into the row buffer
__device__ __forceinline__ int row_at(const PArgs & a, int s) { return min(max(a.q_start[s], 0), a.T); }

template <int BMN, int BN> __device__ __forceinline__ Span span_of(const PArgs & a, int n, int kv, int rt) {
    const int     r0 = rt * BMN, r1 = min(n * a.G, r0 + BMN);  // T * G < 2^31 (checked)
    const int     t0 = a.byG.div(r0), t1 = a.byG.div(r1 - 1);
    const int     base = kv - n;
    const int64_t cap  = min((int64_t) a.cols * a.page, (int64_t) INT32_MAX - BN);
    Span          p;
    p.hi = (int) max((int64_t) 0, min((int64_t) base + t1 + 1, cap));
    p.lo = a.window > 0 ? (int) max((int64_t) 0, (int64_t) base + t0 - a.window + 1) : 0;
    if (p.hi <= p.lo) {
        p.kt0 = p.nkv = 0;
        p.lo = p.hi = 0;
    } else {
        p.kt0 = p.lo / BN;
        p.nkv = (p.hi + BN - 1) / BN - p.kt0;
    }
    p.units = max(p.nkv, 1);
    return p;
}
template <int BMN> __device__ __forceinline__ int tiles_of(const PArgs & a, int n) { return (n * a.G + BMN - 1) / BMN; }

// a CTA's walk over its part of the line; every role keeps its own
struct Walk {
    int     s, h, rt;   // item
    int     off;        // first unit of the item in this CTA
    int64_t rem;        // units left in this CTA
    int     r0, n, kv;  // the sequence's first row, rows and cache length
    Span    sp;
    int     take;       // units of the item done here
    int64_t part;       // units of this CTA in all
    int     tile0, lap; // first tile in this CTA's order; the turn at which the order goes back to the item's first tile
    __device__ __forceinline__ int tile(int i) const { return tile0 + i - (i >= lap ? sp.nkv : 0); }
};

template <int BMN> __device__ __forceinline__ void walk_load(const PArgs & a, Walk & w) {
    w.r0 = row_at(a, w.s);
    w.n  = row_at(a, w.s + 1) - w.r0;
    w.kv = max(a.kv_len[w.s], 0);
}
template <int BMN, int BN> __device__ __forceinline__ void walk_item(const PArgs & a, Walk & w) {
    w.sp   = span_of<BMN, BN>(a, w.n, w.kv, w.rt);
    w.take = (int) min((int64_t) (w.sp.units - w.off), w.rem);
    // A whole item's tiles may come in any order: a long one begins where CTAs that began together and took a tile per turn
    // would be by now, so that those of one KV head read the same tiles at the same time and find them in L2 (2048 rows over
    // 32768 tokens: 1.4 GB from memory instead of 5.2, 1.52 ms instead of 1.69). Short ones find theirs there anyhow (a mixed
    // batch of up to 4000 tokens took 136 us turned and 133 not).
    const bool turned = w.off == 0 && w.take == w.sp.nkv && w.sp.nkv >= 64;
    const int  turn   = turned ? (int) ((uint64_t) (w.part - w.rem) % (uint32_t) w.sp.nkv) : 0;
    w.tile0 = w.sp.kt0 + w.off + turn;
    w.lap   = w.sp.nkv - w.off - turn;
}
// to the next item; false at the end of the part
template <int BMN, int BN> __device__ __forceinline__ bool walk_next(const PArgs & a, Walk & w) {
    w.rem -= w.take;
    if (w.rem <= 0) return false;
    w.off = 0;
    if (++w.rt >= tiles_of<BMN>(a, w.n)) {
        w.rt = 0;
        if (++w.h >= a.Hkv) {
            w.h = 0;
            do {
                if (++w.s >= a.S) return false;
                walk_load<BMN>(a, w);
            } while (w.n <= 0);
        }
    }
    walk_item<BMN, BN>(a, w);
    return true;
}

// Units per KV head of each sequence into tot, by all of the CTA's threads. tot: 2 a.S words of scratch, nbg one, both in shared
// memory. Ends with a barrier. TMA: loads of it come to the place of the sums next.
template <int BMN, int BN, bool TMA> __device__ __forceinline__ void plan_sums(const PArgs & a, int * tot, int * nbg) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int * big = tot + a.S;  // sequences whose tiles a warp sums up
    if (tid == 0) *nbg = 0;
    __syncthreads();
    for (int s = tid; s < a.S; s += blockDim.x) {
        const int r0 = row_at(a, s), n = row_at(a, s + 1) - r0, nt = n > 0 ? tiles_of<BMN>(a, n) : 0;
        int       u = 0;
        if (nt <= 2) {
            const int kv = nt ? max(a.kv_len[s], 0) : 0;
            for (int rt = 0; rt < nt; rt++) u += span_of<BMN, BN>(a, n, kv, rt).units;
        } else {
            big[atomicAdd(nbg, 1)] = s;  // any order: each entry is worked out by itself
        }
        tot[s] = u;
    }
    __syncthreads();
    for (int b = warp; b < *nbg; b += blockDim.x / 32) {
        const int s = big[b], r0 = row_at(a, s), n = row_at(a, s + 1) - r0, nt = tiles_of<BMN>(a, n), kv = max(a.kv_len[s], 0);
        int       u = 0;
        for (int rt = lane; rt < nt; rt += 32) u += span_of<BMN, BN>(a, n, kv, rt).units;
        u = __reduce_add_sync(0xffffffffu, u);
        if (lane == 0) tot[s] = u;
    }
    if constexpr (TMA) fence_proxy_async_smem();
    __syncthreads();
}

// the part, from `part` on, in which unit `end` - 1 of all stands (a search part by part took 30 us of one sequence's 80, cut into 1184)
__device__ __forceinline__ int part_of_end(int64_t all, int64_t parts, int64_t end, int part) {
    return max(part, (int) ((end * parts + all - 1) / all) - 1);
}

// Part `part` of `parts` of the line of units, found by one warp: its first unit (s = -1: the part is empty), its place in the
// line, the units and the parts in all
struct Part {
    int     s, h, rt, off;
    int64_t b0, b1, all, parts;
};
template <int BMN, int BN> __device__ __forceinline__ Part plan_find(const PArgs & a, const int * tot, int part, int parts) {
    const int lane = threadIdx.x & 31;
    Part      p;
    p.s = -1;
    int64_t sum = 0;
    for (int s = lane; s < a.S; s += 32) sum += tot[s];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    // fewer units than parts: one each for the first W, so that an item's parts stand side by side
    const int64_t W = sum * a.Hkv, np = max((int64_t) 1, min((int64_t) parts, W)), c = min((int64_t) part, np);
    const int64_t b0 = W * c / np, b1 = W * min(c + 1, np) / np;
    p.b0    = b0;
    p.b1    = b1;
    p.all   = W;
    p.parts = np;
    if (b1 > b0) {
        int64_t before = 0;
        for (int s0 = 0; s0 < a.S; s0 += 32) {
            const int64_t v   = s0 + lane < a.S ? (int64_t) tot[s0 + lane] * a.Hkv : 0;
            int64_t       inc = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t x = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += x;
            }
            const int64_t  end = before + inc, beg = end - v;
            const uint32_t hit = __ballot_sync(0xffffffffu, b0 >= beg && b0 < end);
            if (hit) {
                const int     src = __ffs(hit) - 1, s = s0 + src;
                const int64_t in  = b0 - __shfl_sync(0xffffffffu, beg, src);
                const int     per = tot[s];
                const int     h   = (int) (in / per);
                int           off = (int) (in - (int64_t) h * per);
                const int     r0 = row_at(a, s), n = row_at(a, s + 1) - r0, nt = tiles_of<BMN>(a, n), kv = max(a.kv_len[s], 0);
                for (int t0 = 0; t0 < nt; t0 += 32) {
                    const int u  = t0 + lane < nt ? span_of<BMN, BN>(a, n, kv, t0 + lane).units : 0;
                    int       ic = u;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const int x = __shfl_up_sync(0xffffffffu, ic, o);
                        if (lane >= o) ic += x;
                    }
                    const uint32_t ht = __ballot_sync(0xffffffffu, off >= ic - u && off < ic);
                    if (ht) {
                        const int l = __ffs(ht) - 1;
                        off -= __shfl_sync(0xffffffffu, ic - u, l);
                        p.s   = s;
                        p.h   = h;
                        p.rt  = t0 + l;
                        p.off = off;
                        break;
                    }
                    off -= __shfl_sync(0xffffffffu, ic, 31);
                }
                break;
            }
            before = __shfl_sync(0xffffffffu, end, 31);
        }
    }
    return p;
}

// This CTA's part of the line, as one of gridDim.x: first = {s, h, rt, off} (s stays as it was, -1, for an empty part), range =
// {start, end, units in all, parts}, both in shared memory. Ends without a barrier.
template <int BMN, int BN, bool TMA>
__device__ __forceinline__ void plan_part(const PArgs & a, int * tot, int * nbg, int * first, int64_t * range) {
    plan_sums<BMN, BN, TMA>(a, tot, nbg);
    if (threadIdx.x < 32) {
        const Part p = plan_find<BMN, BN>(a, tot, blockIdx.x, gridDim.x);
        if (threadIdx.x == 0) {
            range[0] = p.b0;
            range[1] = p.b1;
            range[2] = p.all;
            range[3] = p.parts;
            if (p.s >= 0) {
                first[0] = p.s;
                first[1] = p.h;
                first[2] = p.rt;
                first[3] = p.off;
            }
        }
    }
}

// over q4_0 pages: rows of a tile, parts that the line is cut into on each SM (fa_paged_q4.cu)
int q4_rows(int T, int S, int G, bool f32);
int q4_parts(int rows, int D);
int q4_few_run(srhpm_ctx * ctx, const PArgs & a, const void * maps, const PagedCache & c, bool f32, cudaStream_t stream);  // fa_paged_q4_few.cu
int q4_run(srhpm_ctx * ctx, PArgs & a, const PagedCache & c, int rows, bool f32, cudaStream_t stream);

// every page that a row sees, as f16 [pages][page][Hkv][D] under its own number (unpack_q4.cu)
int unpack_q4_run(srhpm_ctx * ctx, const FaPagedView & v, void * ko, void * vo, cudaStream_t stream);

// tensor map of bytes [pages][tokens][width], boxes of `tokens_box` rows of `box` bytes (fa_paged.cu); false: not encoded
bool encode_rows(void * map, const void * p, uint64_t width, int tokens, int64_t pages, int64_t nb1, int64_t nb3, int box, int tokens_box);

// the records' join behind a kernel that cut items (fa_paged.cu)
int merge_launch(srhpm_ctx * ctx, const PArgs & a, int D, bool f32, int rows_y, cudaStream_t stream, int parts = 1);  // parts: of an SM

inline size_t align16(size_t n) { return (n + 15) / 16 * 16; }

}  // namespace fap
}  // namespace srhpm
