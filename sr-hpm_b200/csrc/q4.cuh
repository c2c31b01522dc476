// q4_0 blocks in registers. A pair of blocks is 36 bytes, nine words: W0 = d0 | numbers 0, 1 of block 0; W1 .. W3 = numbers 2 ..
// 13; W4 = 14, 15 | d1; W5 .. W8 = block 1. The numbers are taken by words, four bytes each, a byte holding the numbers j and j + 16:
// words 0 .. 3 of block 0 are W1, W2, W3 and the bytes that remain of W0 and W4, those of block 1 W5 .. W8. A word's eight
// values come as f16 pairs of bytes (0, 2) and (1, 3), low halves before high ones; whoever multiplies with them takes the other
// operand in the same order.
#pragma once
#include <cuda.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "ptx.cuh"

namespace srhpm {
namespace q4 {

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
    uint32_t r;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
    return r;
}
template <uint32_t MASK> __device__ __forceinline__ uint32_t magic(uint32_t x) {  // (x & MASK) | 0x64006400
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(x), "n"(MASK), "r"(0x64006400u));
    return r;
}
// bits 0 .. 3 of either half, as f16 1024 + q, minus 1032 is q - 8, exactly; one product with d, rounded, is the cache's value
__device__ __forceinline__ uint32_t low4(uint32_t x, uint32_t dd) {
    const uint32_t m = magic<0x000f000fu>(x);
    __half2        h = __hsub2(*reinterpret_cast<const __half2 *>(&m), __floats2half2_rn(1032.0f, 1032.0f));
    h                = __hmul2(h, *reinterpret_cast<const __half2 *>(&dd));
    return *reinterpret_cast<const uint32_t *>(&h);
}
// bits 4 .. 7: 1024 + 16 q, through x / 16 - 72, exactly
__device__ __forceinline__ uint32_t high4(uint32_t x, uint32_t dd) {
    const uint32_t m = magic<0x00f000f0u>(x);
    __half2        h = __hfma2(*reinterpret_cast<const __half2 *>(&m), __floats2half2_rn(0.0625f, 0.0625f), __floats2half2_rn(-72.0f, -72.0f));
    h                = __hmul2(h, *reinterpret_cast<const __half2 *>(&dd));
    return *reinterpret_cast<const uint32_t *>(&h);
}

// the block's number that byte b of its word w holds in its low half
__device__ __forceinline__ int byte_of(bool odd, int w, int b) { return odd ? 4 * w + b : w < 3 ? 2 + 4 * w + b : b < 2 ? b : 12 + b; }

// the place among a pair's 64 values of the one that stands at place k of their order here
__device__ __forceinline__ int value_at(int k) {
    const int  w = (k >> 3) & 3, p = (k >> 1) & 3, e = k & 1;
    const bool odd = k >= 32;
    return 32 * odd + byte_of(odd, w, (p & 1) + 2 * e) + 16 * (p >> 1);
}

// a block's 16 pairs; W: the nine words of its pair of blocks
template <bool ODD> __device__ __forceinline__ void unpack(const uint32_t * W, uint32_t (&v)[16]) {
    const uint32_t d = ODD ? prmt(W[4], W[4], 0x3232u) : prmt(W[0], W[0], 0x1010u);
#pragma unroll
    for (int w = 0; w < 4; w++) {
        const uint32_t x = ODD ? W[5 + w] : w < 3 ? W[1 + w] : prmt(W[0], W[4], 0x5432u);
        v[4 * w]     = low4(x, d);
        v[4 * w + 1] = low4(x >> 8, d);
        v[4 * w + 2] = high4(x, d);
        v[4 * w + 3] = high4(x >> 8, d);
    }
}

template <int N> __device__ __forceinline__ void copy_async(uint32_t dst, const uint8_t * src, uint32_t size) {
    if constexpr (N == 16) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(size) : "memory");
    } else {
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(size) : "memory");
    }
}


// ---- what both kernels of attention over q4_0 pages use ----
struct Pool4 {
    const uint8_t * p;
    int64_t         nb1, nb2, nb3;  // token, KV head, page
};
constexpr uint32_t kProbes = 1u << 19;  // of a wait before it gives up: about 2 s

// bytes of a raw row's place: TMA's boxes start on 16 bytes, the row up to 12 later
constexpr int row_stride(int D) { return D == 64 ? 48 : D == 128 ? 80 : 144; }

__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void tma_rows(uint32_t dst, const CUtensorMap * m, int x, int y, int z, uint64_t * bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(m), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}
__device__ __forceinline__ float exp2a(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

}  // namespace q4
}  // namespace srhpm
