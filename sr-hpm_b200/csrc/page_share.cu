// Pages of a paged KV cache that change hands between steps:
//   page_fork     new sequences that begin with the tokens of others: whole pages are shared, a partly filled one is copied
//   page_copy     whole pages within the pools of all layers, in one launch
//   page_free     pages that sequences no longer hold, back onto the free list
//   page_compact  the pages in use moved to the lowest numbers (tables, references and free list; page_copy moves the bytes)
// All lengths, tables and lists are read on the device, so a captured step replays with new ones. Results do not hang on the
// order of atomics: references are counted in whole numbers, and lists are written in the order of page numbers.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

#include "fastdiv.cuh"
#include "internal.h"
#include "launch.cuh"
#include "ptx.cuh"

namespace cg = cooperative_groups;

namespace srhpm {
namespace {

__device__ __forceinline__ int warp_incl(int v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    return v;
}
// exclusive sum over the CTA's threads and their total; sp: 32 words of shared memory
__device__ __forceinline__ int cta_excl(int v, int * sp, int * total) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
    const int in   = warp_incl(v);
    if (lane == 31) sp[warp] = in;
    __syncthreads();
    if (warp == 0) sp[lane] = warp_incl(lane < nw ? sp[lane] : 0);
    __syncthreads();
    const int r = in - v + (warp ? sp[warp - 1] : 0);
    *total      = sp[nw - 1];
    __syncthreads();
    return r;
}

// ---- fork ----------------------------------------------------------------------------------------------------------
// Fork i takes a page when keep_i is no multiple of the page size: its place in the free list is an exclusive sum over the
// forks, which every CTA takes itself (n <= 8192 numbers from L2) before it copies its share of table entries.
constexpr int kForkThreads = 1024;
constexpr int kForkChunk   = 256;  // table entries of a warp's job

struct ForkArgs {
    const int32_t * parent;
    const int32_t * child;
    const int32_t * keep;
    int             n, P;
    uint8_t *       table;
    int64_t         tstride;
    int             cols, rows;
    int32_t *       refs;
    int             n_pages;
    const int32_t * free_pages;
    int             n_free;
    const int32_t * free_head;  // or null (0)
    int32_t *       src;
    int32_t *       dst;
    int32_t *       status;
    int32_t *       n_taken;
    int             chunks;  // of a table row
};

__global__ void __launch_bounds__(kForkThreads) page_fork_kernel(const ForkArgs a) {
    extern __shared__ int32_t spot[];  // [n] place of the fork's new page in the free list, -1: needs none, -2: refused
    __shared__ int            sp[32];
    __shared__ int            taken_s;
    if (threadIdx.x == 0) taken_s = 0;
    pdl_launch_dependents();
    pdl_wait();
    const int64_t head = a.free_head ? (int64_t) *a.free_head : 0;
    int           before = 0;  // at most n
    __syncthreads();
    for (int i0 = 0; i0 < a.n; i0 += blockDim.x) {
        const int  i  = i0 + threadIdx.x;
        const bool in = i < a.n;
        int        st = SRHPM_PAGES_OK, need = 0;
        if (in) {
            const int keep = a.keep[i], pa = a.parent[i], ch = a.child[i];
            if (keep < 0 || pa < 0 || pa >= a.rows || ch < 0 || ch >= a.rows || pa == ch) {
                st = SRHPM_PAGES_BAD_LENGTH;
            } else if ((int64_t) keep > (int64_t) a.cols * a.P) {
                st = SRHPM_PAGES_TABLE_FULL;
            } else {
                need = keep % a.P != 0;
            }
        }
        int       all;
        const int at = before + cta_excl(need, sp, &all);
        before += all;
        if (need && (head < 0 || head + at >= a.n_free)) st = SRHPM_PAGES_NONE_FREE;
        if (in) {
            spot[i] = st != SRHPM_PAGES_OK ? -2 : need ? (int) (head + at) : -1;
            if (need && st == SRHPM_PAGES_OK) atomicMax(&taken_s, at + 1);
            if (blockIdx.x == 0) a.status[i] = st;
        }
    }
    __syncthreads();
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.n_taken = taken_s;
    const int     lane = threadIdx.x & 31;
    const int64_t jobs = (int64_t) a.n * a.chunks, nwarp = (int64_t) gridDim.x * (blockDim.x / 32);
    for (int64_t j = (int64_t) blockIdx.x * (blockDim.x / 32) + (threadIdx.x >> 5); j < jobs; j += nwarp) {
        const int i = (int) (j / a.chunks), c0 = (int) (j - (int64_t) i * a.chunks) * kForkChunk;
        const int at = spot[i];
        if (at == -2) {
            if (c0 == 0 && lane == 0) a.src[i] = a.dst[i] = -1;
            continue;
        }
        const int       keep = a.keep[i], full = keep / a.P;
        const int32_t * from = reinterpret_cast<const int32_t *>(a.table + (int64_t) a.parent[i] * a.tstride);
        int32_t *       to   = reinterpret_cast<int32_t *>(a.table + (int64_t) a.child[i] * a.tstride);
        const int       end  = min(full, c0 + kForkChunk);
        int             p[kForkChunk / 32];
#pragma unroll
        for (int k = 0; k < kForkChunk / 32; k++) p[k] = c0 + 32 * k + lane < end ? from[c0 + 32 * k + lane] : -1;
#pragma unroll
        for (int k = 0; k < kForkChunk / 32; k++) {
            if (c0 + 32 * k + lane < end) {
                to[c0 + 32 * k + lane] = p[k];
                if (p[k] >= 0 && p[k] < a.n_pages) atomicAdd(a.refs + p[k], 1);
            }
        }
        if (c0 == 0 && lane == 0) {
            int s = -1, d = -1;
            if (at >= 0) {
                s        = from[full];
                d        = a.free_pages[at];
                to[full] = d;
                if (s < 0 || s >= a.n_pages) s = d = -1;
            }
            a.src[i] = s;
            a.dst[i] = d;
        }
    }
}

// ---- copy ----------------------------------------------------------------------------------------------------------
// Pure traffic: a job is a piece of one page of one pool, four loads in flight per thread.
constexpr int kCopyThreads = 256;
constexpr int kCopyLoads   = 4;
constexpr int kCopyPools   = 256;  // of a launch

struct CopyArgs {
    uint8_t *       pool[kCopyPools];
    int             n_pools, n, n_pages;
    const int32_t * src;
    const int32_t * dst;
    const int32_t * n_moves;  // or null (n)
    int64_t         nb3;
    int             units, pieces;  // of a page
    // a page: n2 x n1 runs of `run` units, s2 and s1 bytes apart
    FastDiv by_run, by_n1;
    int64_t s1, s2;
};

template <class U, bool DENSE>
__global__ void __launch_bounds__(kCopyThreads) page_copy_kernel(const __grid_constant__ CopyArgs a) {
    pdl_launch_dependents();
    pdl_wait();
    const int     n    = a.n_moves ? min(max(*a.n_moves, 0), a.n) : a.n;
    const int64_t per  = (int64_t) a.pieces * a.n_pools;  // jobs of a move
    const int64_t jobs = per * n;
    for (int64_t j = blockIdx.x; j < jobs; j += gridDim.x) {
        const int m = (int) (j / per), r = (int) (j - m * per), pool = r / a.pieces, piece = r - pool * a.pieces;
        const int s = a.src[m], d = a.dst[m];
        if (s < 0 || s >= a.n_pages || d < 0 || d >= a.n_pages || s == d) continue;
        const uint8_t * from = a.pool[pool] + s * a.nb3;
        uint8_t *       to   = a.pool[pool] + d * a.nb3;
        U               x[kCopyLoads];
        int64_t         off[kCopyLoads];
#pragma unroll
        for (int k = 0; k < kCopyLoads; k++) {
            const int u = (piece * kCopyLoads + k) * kCopyThreads + (int) threadIdx.x;
            if constexpr (DENSE) {
                off[k] = (int64_t) u * sizeof(U);
            } else {
                const int row = a.by_run.div(u), i2 = a.by_n1.div(row);
                off[k] = i2 * a.s2 + (row - i2 * (int) a.by_n1.d) * a.s1 + (int64_t) (u - row * (int) a.by_run.d) * sizeof(U);
            }
            if (u < a.units) x[k] = *reinterpret_cast<const U *>(from + off[k]);
        }
#pragma unroll
        for (int k = 0; k < kCopyLoads; k++) {
            const int u = (piece * kCopyLoads + k) * kCopyThreads + (int) threadIdx.x;
            if (u < a.units) *reinterpret_cast<U *>(to + off[k]) = x[k];
        }
    }
}

// ---- free and compact ----------------------------------------------------------------------------------------------
// One launch of one cluster: the page numbers are shared out among its CTAs, each of which keeps a bit per page in shared
// memory that all of them set. Lists in the order of page numbers then come from sums over the bits.
constexpr int kSetThreads = 1024;
constexpr int kSetCtas    = 8;

struct SetArgs {
    const int32_t * rows;   // free: table rows; compact: null (all)
    const int32_t * begin;  // or null (0)
    const int32_t * end;
    int             n, chunks;
    uint8_t *       table;
    int64_t         tstride;
    int             cols, trows;
    int32_t *       refs;
    int             n_pages, shift;  // pages of a CTA: 1 << shift
    int32_t *       free_pages;
    int             n_free;
    const int32_t * free_head;
    int32_t *       src;
    int32_t *       dst;
    int32_t *       out0;  // free: pages freed; compact: moves
    int32_t *       out1;  // compact: pages in use
    int32_t *       status;
};

// For each entry in range of this cluster's rows, kForkChunk at a time per warp: p = take(entry), then r = look(p) for those that
// are pages, then use(entry, p, r). Each of the three goes over a warp's 256 entries before the next, so that a round trip is waited
// for once and not eight times (48 of 1024 sequences freed, 12000 pages: 19 us, now 15.6).
template <class Take, class Look, class Use>
__device__ __forceinline__ void each_entry(const SetArgs & a, int rank, int ctas, Take take, Look look, Use use) {
    constexpr int K    = kForkChunk / 32;
    const int     lane = threadIdx.x & 31;
    const int64_t jobs = (int64_t) a.n * a.chunks, nwarp = (int64_t) ctas * (blockDim.x / 32);
    for (int64_t j = (int64_t) rank * (blockDim.x / 32) + (threadIdx.x >> 5); j < jobs; j += nwarp) {
        const int i = (int) (j / a.chunks), c0 = (int) (j - (int64_t) i * a.chunks) * kForkChunk + lane;
        const int row = a.rows ? a.rows[i] : i;
        const int lo = max(a.begin ? a.begin[i] : 0, 0), hi = min(a.end[i], a.cols);
        if (row < 0 || row >= a.trows) continue;
        int32_t * e = reinterpret_cast<int32_t *>(a.table + (int64_t) row * a.tstride) + c0;
        int       p[K], r[K];
#pragma unroll
        for (int k = 0; k < K; k++) p[k] = c0 + 32 * k >= lo && c0 + 32 * k < hi ? take(e + 32 * k) : -1;
#pragma unroll
        for (int k = 0; k < K; k++) r[k] = p[k] >= 0 && p[k] < a.n_pages ? look(p[k]) : 0;
#pragma unroll
        for (int k = 0; k < K; k++) {
            if (p[k] >= 0 && p[k] < a.n_pages) use(e + 32 * k, p[k], r[k]);
        }
    }
}

__global__ void __launch_bounds__(kSetThreads) page_free_kernel(const SetArgs a) {
    extern __shared__ uint32_t bits[];  // of this CTA's pages
    __shared__ int             sp[32];
    __shared__ int             count;
    cg::cluster_group cl = cg::this_cluster();
    const int rank = (int) cl.block_rank(), ctas = (int) cl.num_blocks();
    const int words = 1 << (a.shift - 5);
    pdl_launch_dependents();
    for (int i = threadIdx.x; i < words; i += blockDim.x) bits[i] = 0;
    pdl_wait();
    cl.sync();
    auto take = [](int32_t * e) { return atomicExch(e, -1); };  // an entry that is listed twice is freed once
    auto drop = [&](int p) { return atomicSub(a.refs + p, 1); };
    each_entry(a, rank, ctas, take, drop, [&](int32_t *, int p, int others) {
        if (others > 0) return;
        const int q = p & ((1 << a.shift) - 1);
        atomicOr(cl.map_shared_rank(bits, p >> a.shift) + (q >> 5), 1u << (q & 31));
    });
    cl.sync();
    // words of a thread stand side by side
    const int per = (words + blockDim.x - 1) / blockDim.x, w0 = min((int) threadIdx.x * per, words), w1 = min(w0 + per, words);
    int       mine = 0, all;
    for (int i = w0; i < w1; i++) mine += __popc(bits[i]);
    int at = cta_excl(mine, sp, &all);
    if (threadIdx.x == 0) count = all;
    cl.sync();
    int total = 0;
    for (int c = 0; c < ctas; c++) {
        const int v = *cl.map_shared_rank(&count, c);
        if (c < rank) at += v;
        total += v;
    }
    const int head = min(max(*a.free_head, 0), a.n_free);
    if (rank == 0 && threadIdx.x == 0) {
        *a.out0 = min(total, head);
        if (total > head) atomicExch(a.status, kErrPage);  // more pages than were ever taken
    }
    for (int i = w0; i < w1; i++) {
        for (uint32_t b = bits[i]; b; b &= b - 1) {
            const int p = (rank << a.shift) + 32 * i + __ffs(b) - 1, to = head - total + at++;
            a.refs[p] = 0;
            if (to >= 0) a.free_pages[to] = p;
        }
    }
    cl.sync();  // the others read this CTA's count
}

__global__ void __launch_bounds__(kSetThreads) page_compact_kernel(const SetArgs a) {
    extern __shared__ uint32_t bits[];  // of this CTA's pages; behind them the pages in use before each word
    __shared__ int             sp[32];
    __shared__ int             count, split;
    cg::cluster_group cl = cg::this_cluster();
    const int  rank = (int) cl.block_rank(), ctas = (int) cl.num_blocks();
    const int  words = 1 << (a.shift - 5);
    int32_t *  pre = reinterpret_cast<int32_t *>(bits + words);
    pdl_launch_dependents();
    for (int i = threadIdx.x; i < words; i += blockDim.x) bits[i] = 0;
    pdl_wait();
    cl.sync();
    auto read = [](int32_t * e) { return *e; };
    each_entry(a, rank, ctas, read, [](int) { return 0; }, [&](int32_t *, int p, int) {
        const int q = p & ((1 << a.shift) - 1);
        atomicOr(cl.map_shared_rank(bits, p >> a.shift) + (q >> 5), 1u << (q & 31));
    });
    cl.sync();
    const int per = (words + blockDim.x - 1) / blockDim.x, w0 = min((int) threadIdx.x * per, words), w1 = min(w0 + per, words);
    int       mine = 0, all;
    for (int i = w0; i < w1; i++) mine += __popc(bits[i]);
    int at = cta_excl(mine, sp, &all);
    if (threadIdx.x == 0) count = all;
    cl.sync();
    int used = 0;
    for (int c = 0; c < ctas; c++) {
        const int v = *cl.map_shared_rank(&count, c);
        if (c < rank) at += v;
        used += v;
    }
    for (int i = w0; i < w1; i++) {
        pre[i] = at;
        at += __popc(bits[i]);
    }
    __syncthreads();
    // pages in use among the first `used`: the rest of those stay free places for the others
    const int owner = min(used, a.n_pages - 1) >> a.shift;
    auto      before = [&](const uint32_t * b, const int32_t * pr, int p) {  // of CTA p >> shift
        const int q = p & ((1 << a.shift) - 1);
        return pr[q >> 5] + __popc(b[q >> 5] & ((1u << (q & 31)) - 1));
    };
    if (threadIdx.x == 0 && rank == owner) split = used < a.n_pages ? before(bits, pre, used) : used;
    cl.sync();
    const int low = *cl.map_shared_rank(&split, owner), moves = used - low;
    if (rank == 0 && threadIdx.x == 0) {
        *a.out0 = moves;
        *a.out1 = used;
    }
    if (moves > 0) {
        for (int i = w0; i < w1; i++) {
            const int p0 = (rank << a.shift) + 32 * i;
            if (p0 + 32 > used) {  // pages behind the border that are in use
                uint32_t b = bits[i];
                if (p0 < used) b &= ~0u << (used - p0);
                int k = pre[i] + __popc(bits[i] & ~b) - low;
                for (; b; b &= b - 1) a.src[k++] = p0 + __ffs(b) - 1;
            }
            if (p0 < used) {  // places before it that are not
                uint32_t b = ~bits[i];
                if (p0 + 32 > used) b &= (1u << (used - p0)) - 1;
                int k = p0 - pre[i];
                for (; b; b &= b - 1) a.dst[k++] = p0 + __ffs(b) - 1;
            }
        }
    }
    const int tid = rank * blockDim.x + threadIdx.x, nthr = ctas * blockDim.x;
    for (int p = used + tid; p < a.n_pages; p += nthr) a.free_pages[p] = p;
    __threadfence();
    cl.sync();
    if (moves > 0) {
        for (int k = tid; k < moves; k += nthr) {
            const int s = __ldcg(a.src + k), d = __ldcg(a.dst + k);
            a.refs[d] = a.refs[s];
            a.refs[s] = 0;
        }
        auto place = [&](int p) {
            const int o = p >> a.shift;
            return p < used ? p : __ldcg(a.dst + before(cl.map_shared_rank(bits, o), cl.map_shared_rank(pre, o), p) - low);
        };
        each_entry(a, rank, ctas, read, place, [](int32_t * e, int p, int to) {
            if (to != p) *e = to;
        });
    }
    cl.sync();
}

// WORD: bytes of shared memory per 32 pages of a CTA
template <void (*KERN)(SetArgs), int WORD> int set_launch(srhpm_ctx * ctx, SetArgs & a, cudaStream_t stream) {
    // The limit belongs to the kernel, not to the call: always that of the largest pool, as another thread's call over a smaller
    // one may come between this one's limit and its launch.
    static std::atomic<unsigned> done{ 0 };
    const unsigned               bit = 1u << (ctx->device & 31);
    if (!(done.load() & bit)) {
        const int st = cuda_status(cudaFuncSetAttribute(KERN, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxPages / kSetCtas / 32 * WORD));
        if (st != SRHPM_OK) return st;
        done.fetch_or(bit);
    }
    // pages of a CTA: all 8 share them out, 1024 at least
    a.shift = 10;
    while (((int64_t) kSetCtas << a.shift) < a.n_pages) a.shift++;
    // CTAs: those that have pages or entries to look at
    const int64_t jobs = (int64_t) a.n * a.chunks;
    int           ctas = 1;
    while (ctas < kSetCtas && (((int64_t) ctas << a.shift) < a.n_pages || ctas * 32 < jobs)) ctas *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim            = dim3(ctas);
    cfg.blockDim           = dim3(kSetThreads);
    cfg.dynamicSmemBytes   = (size_t) WORD << (a.shift - 5);
    cfg.stream             = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id                                         = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id                                         = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x                           = ctas;
    attr[1].val.clusterDim.y                           = 1;
    attr[1].val.clusterDim.z                           = 1;
    cfg.attrs    = attr;
    cfg.numAttrs = 2;
    const int st = cuda_status(cudaLaunchKernelEx(&cfg, KERN, a));
    ctx->launches.fetch_add(1);
    return st;
}

template <class U, bool DENSE> int copy_launch(srhpm_ctx * ctx, const CopyArgs & a, cudaStream_t stream) {
    const int64_t jobs = (int64_t) a.pieces * a.n_pools * a.n;
    const int     grid = (int) std::min<int64_t>(jobs, (int64_t) ctx->num_sms * 8);
    const int     st   = cuda_status(launch_k_pdl(page_copy_kernel<U, DENSE>, dim3(grid), dim3(kCopyThreads), 0, stream, a));
    ctx->launches.fetch_add(1);
    return st;
}

}  // namespace

int page_fork_run(srhpm_ctx * ctx, const PageTable & t, const int32_t * parent, const int32_t * child, const int32_t * keep, int n,
                  int page, int32_t * refs, int n_pages, const int32_t * free_pages, int n_free, const int32_t * free_head,
                  int32_t * src, int32_t * dst, int32_t * status, int32_t * n_taken, cudaStream_t stream) {
    ForkArgs a{ parent, child, keep, n, page, t.data, t.stride, t.cols, t.rows, refs, n_pages, free_pages, n_free, free_head,
                src, dst, status, n_taken, (t.cols + kForkChunk - 1) / kForkChunk };
    const int64_t jobs = (int64_t) n * a.chunks;
    const int     grid = (int) std::max<int64_t>(1, std::min<int64_t>(ctx->num_sms, (jobs + 31) / 32));
    const int     st = cuda_status(launch_k_pdl(page_fork_kernel, dim3(grid), dim3(kForkThreads), n * sizeof(int32_t), stream, a));
    ctx->launches.fetch_add(1);
    return st;
}

int page_free_run(srhpm_ctx * ctx, const PageTable & t, const int32_t * rows, const int32_t * begin, const int32_t * end, int n,
                  int32_t * refs, int n_pages, int32_t * free_pages, int n_free, const int32_t * free_head, int32_t * n_freed,
                  cudaStream_t stream) {
    SetArgs a{ rows, begin, end, n, (t.cols + kForkChunk - 1) / kForkChunk, t.data, t.stride, t.cols, t.rows, refs, n_pages, 0,
               free_pages, n_free, free_head, nullptr, nullptr, n_freed, nullptr, ctx->d_status };
    return set_launch<page_free_kernel, 4>(ctx, a, stream);
}

int page_compact_run(srhpm_ctx * ctx, const PageTable & t, const int32_t * held, int32_t * refs, int n_pages, int32_t * free_pages,
                     int32_t * src, int32_t * dst, int32_t * n_moves, int32_t * n_used, cudaStream_t stream) {
    SetArgs a{ nullptr, nullptr, held, t.rows, (t.cols + kForkChunk - 1) / kForkChunk, t.data, t.stride, t.cols, t.rows, refs, n_pages, 0,
               free_pages, n_pages, nullptr, src, dst, n_moves, n_used, ctx->d_status };
    return set_launch<page_compact_kernel, 8>(ctx, a, stream);
}

int page_copy_run(srhpm_ctx * ctx, const srhpm_tensor * caches, int n_caches, const int32_t * src, const int32_t * dst, int n,
                  const int32_t * n_moves, cudaStream_t stream) {
    const srhpm_tensor & c = caches[0];
    // runs of bytes that stand side by side, the two outer dimensions by their strides
    int64_t run = (int64_t) srhpm_row_size(c.type, c.ne[0]), n1 = c.ne[1], s1 = (int64_t) c.nb[1], n2 = c.ne[2], s2 = (int64_t) c.nb[2];
    if (n1 == 1 || (n2 > 1 && s2 < s1)) {
        std::swap(n1, n2);
        std::swap(s1, s2);
    }
    if (n1 == 1 || s1 == run) {
        run *= n1;
        n1 = n2;
        s1 = s2;
        n2 = 1;
        s2 = 0;
        if (n1 == 1 || s1 == run) {
            run *= n1;
            n1 = 1;
            s1 = 0;
        }
    }
    uint64_t all = (uint64_t) run | (n1 > 1 ? (uint64_t) s1 : 0) | (n2 > 1 ? (uint64_t) s2 : 0) | (c.ne[3] > 1 ? (uint64_t) c.nb[3] : 0);
    for (int i = 0; i < n_caches; i++) all |= reinterpret_cast<uintptr_t>(caches[i].data);
    const int U = all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : 2;
    CopyArgs  a;
    const int64_t units = run / U * n1 * n2;
    if (units > INT32_MAX / 2) return SRHPM_UNSUPPORTED;
    a.n       = n;
    a.n_pages = (int) c.ne[3];
    a.src     = src;
    a.dst     = dst;
    a.n_moves = n_moves;
    a.nb3     = (int64_t) c.nb[3];
    a.units   = (int) units;
    a.pieces  = (int) ((units + kCopyLoads * kCopyThreads - 1) / (kCopyLoads * kCopyThreads));
    a.by_run  = FastDiv::of((uint32_t) (run / U));
    a.by_n1   = FastDiv::of((uint32_t) n1);
    a.s1      = s1;
    a.s2      = s2;
    const bool dense = n1 == 1 && n2 == 1;
    for (int i0 = 0; i0 < n_caches; i0 += kCopyPools) {
        a.n_pools = std::min(kCopyPools, n_caches - i0);
        for (int i = 0; i < a.n_pools; i++) a.pool[i] = reinterpret_cast<uint8_t *>(caches[i0 + i].data);
        const int st = U == 16  ? (dense ? copy_launch<uint4, true>(ctx, a, stream) : copy_launch<uint4, false>(ctx, a, stream))
                       : U == 8 ? (dense ? copy_launch<uint2, true>(ctx, a, stream) : copy_launch<uint2, false>(ctx, a, stream))
                       : U == 4 ? (dense ? copy_launch<uint32_t, true>(ctx, a, stream) : copy_launch<uint32_t, false>(ctx, a, stream))
                                : (dense ? copy_launch<uint16_t, true>(ctx, a, stream) : copy_launch<uint16_t, false>(ctx, a, stream));
        if (st != SRHPM_OK) return st;
    }
    return SRHPM_OK;
}

}  // namespace srhpm
