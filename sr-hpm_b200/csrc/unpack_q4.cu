// The visible pages of prompts' sequences as f16, for attention over a q4_0 cache by the kernel of f16 caches (fa_paged.cu): the
// rows of a long prompt fill so many tiles that each cached token would be unpacked tens of times over, while once takes the time of
// the bytes (0.56 read and 2 written per value). 2048 rows over 32768 tokens, 24 / 4 heads of 256: 42 us (4.1 TB/s)
// and 1.67 ms in all, unpacked tile by tile 2.69.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "fa_paged.cuh"
#include "fastdiv.cuh"
#include "internal.h"
#include "launch.cuh"
#include "ptx.cuh"
#include "q4.cuh"

namespace srhpm {
using namespace fap;
namespace {

constexpr int kThreads = 256;
constexpr int kTokens  = 16;  // of a CTA's turn

struct Args {
    const uint8_t * k;
    int64_t         knb1, knb2, knb3;
    const uint8_t * v;
    int64_t         vnb1, vnb2, vnb3;
    const uint8_t * table;
    int64_t         tstride;
    int             cols, page, n_pages;
    const int32_t * q_start;
    const int32_t * kv_len;
    int             S, T, Hkv, D, window;
    int             turns;              // of a sequence
    FastDiv         by_words, by_page;  // words of a token's heads
    __half *        ko;
    __half *        vo;
};

// A thread has a word of four bytes, eight values: two runs of four dims. Pages that several sequences share are written by each, the
// same values.
__global__ void __launch_bounds__(kThreads) unpack_q4_kernel(const __grid_constant__ Args a) {
    pdl_launch_dependents();
    pdl_wait();
    const int words = a.by_words.d, per = a.D / 8;  // words of a token, of a head
    for (int64_t job = blockIdx.x; job < (int64_t) a.S * a.turns; job += gridDim.x) {
        const int s = (int) (job / a.turns), t0 = (int) (job - (int64_t) s * a.turns) * kTokens;
        const int r0 = min(max(a.q_start[s], 0), a.T), n = min(max(a.q_start[s + 1], 0), a.T) - r0, kv = max(a.kv_len[s], 0);
        if (n <= 0 || t0 >= kv) continue;
        if (a.window > 0 && (int64_t) t0 + kTokens <= (int64_t) kv - n - a.window + 1) continue;  // before every row's window
        const int e  = a.by_page.div(t0), y = t0 - e * a.page;
        const int pg = reinterpret_cast<const int32_t *>(a.table + (int64_t) s * a.tstride)[e];
        if (pg < 0 || pg >= a.n_pages) continue;  // the attention sees that it is no page
        const int64_t out0 = ((int64_t) pg * a.page + y) * a.Hkv * a.D;
        for (int u = threadIdx.x; u < kTokens * words; u += kThreads) {
            const int     tk = a.by_words.div(u), x = u - tk * words, h = x / per, w = x - h * per;
            const int64_t at = (w >> 2) * 18 + 2 + 4 * (w & 3);  // numbers j .. j + 3 and j + 16 .. of the block, j = 4 (w & 3)
            const int64_t ok = (int64_t) pg * a.knb3 + (int64_t) (y + tk) * a.knb1 + h * a.knb2, ov = (int64_t) pg * a.vnb3 + (int64_t) (y + tk) * a.vnb1 + h * a.vnb2;
            const int64_t out = out0 + (int64_t) tk * a.Hkv * a.D + h * a.D + 32 * (w >> 2) + 4 * (w & 3);
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const uint8_t * p = (i ? a.v + ov : a.k + ok);
                const uint32_t  q = *reinterpret_cast<const uint16_t *>(p + at) | (uint32_t) *reinterpret_cast<const uint16_t *>(p + at + 2) << 16;
                const uint32_t  d = *reinterpret_cast<const uint16_t *>(p + (w >> 2) * 18), dd = d | d << 16;
                const uint32_t  l0 = q4::low4(q, dd), l1 = q4::low4(q >> 8, dd), h0 = q4::high4(q, dd), h1 = q4::high4(q >> 8, dd);
                __half * o = (i ? a.vo : a.ko) + out;
                *reinterpret_cast<uint2 *>(o)      = make_uint2(q4::prmt(l0, l1, 0x5410u), q4::prmt(l0, l1, 0x7632u));
                *reinterpret_cast<uint2 *>(o + 16) = make_uint2(q4::prmt(h0, h1, 0x5410u), q4::prmt(h0, h1, 0x7632u));
            }
        }
    }
}

}  // namespace

int fap::unpack_q4_run(srhpm_ctx * ctx, const FaPagedView & v, void * ko, void * vo, cudaStream_t stream) {
    const int64_t turns = (std::min<int64_t>((int64_t) v.cols * v.c.page, INT32_MAX) + kTokens - 1) / kTokens;  // as far as kv_len counts
    Args a{ v.c.k, v.c.knb1, v.c.knb2, v.c.knb3, v.c.v, v.c.vnb1, v.c.vnb2, v.c.vnb3, v.table, v.tstride, v.cols, v.c.page, (int) v.c.n_pages,
            v.q_start, v.kv_len, v.S, v.T, v.c.Hkv, v.c.D, v.window, (int) turns, FastDiv::of((uint32_t) (v.c.Hkv * (v.c.D / 8))),
            FastDiv::of((uint32_t) v.c.page), static_cast<__half *>(ko), static_cast<__half *>(vo) };
    const int grid = (int) std::min<int64_t>((int64_t) v.S * turns, (int64_t) ctx->num_sms * 8);
    const int st   = cuda_status(launch_k_pdl(unpack_q4_kernel, dim3(grid), dim3(kThreads), 0, stream, a));
    ctx->launches.fetch_add(1);
    return st;
}

}  // namespace srhpm
