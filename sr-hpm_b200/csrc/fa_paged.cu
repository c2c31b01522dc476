// Attention of a batch's new tokens over a paged KV cache (srhpm_flash_attn_paged), on the 5th-generation tensor cores.
//
// The R = G * n rows (G query heads per KV head, n new tokens) that a sequence has for one KV head are packed token by
// token into tiles of BR rows: a decode step's few rows and a prompt's thousands take the same path, and K/V is read once
// for all heads of a group. Per row tile and tile of BN cached tokens (128; f32 rows over q8_0: 64):
//   S = Q K^T      M = 128 rows (BR = 56: 64), N = BN tokens, f32 in tensor memory (both operands from shared memory)
//   softmax        one pass with the running maximum m and sum l of each row in registers; the maximum is raised only
//                  when a tile exceeds it by more than 2^8 (then O is rescaled in place), p = 2^(s - m + 7) <= 2^15 as
//                  f16 back into S's place in tensor memory: the 2^7 keeps probabilities down to 2^-21 of the row's
//                  largest out of f16's subnormals
//   O += P V       A = P from tensor memory, B = V as it lies in shared memory (N = head_dim)
// f32 rows (PREC): Q and P as sums of two f16 parts (2^-22), two products each. f16 rows: one product each, P rounded to
// f16 (2^-11 of each probability; the sums l stay f32).
//
// Work: an item is (sequence, KV head, row tile); its units are the BN-token tiles that the rows see. All items' units
// stand in one line that is cut into equal parts, one per CTA (one CTA per SM: any mix of lengths keeps every SM busy to
// the end, and one long row is spread over the whole GPU). An item cut between CTAs leaves (m, l, O) records, which
// fa_paged_merge_kernel joins in the order of the cuts (same bits every run). The plan is taken from the lengths on the
// device by every CTA itself, in its prologue (2.5 us): no planning launch. Cuts moved to the items' borders where one was
// near gained nothing (0 to 7 % slower).
//
// Roles: 8 softmax warps, 1 MMA warp, 3 producer warps (TMA boxes of at most 64 tokens x 64 dims, each within a page, into
// a ring of 128-byte-swizzled chunks), and for a q8_0 cache 16 converter warps (raw rows by TMA into a second ring, d * q
// rounded to f16 into the chunks). NT = 1: the 8 softmax warps halve the columns of one row tile and S has two buffers;
// NT = 2 (head_dim <= 128): two row tiles share K/V, each with its own 4 softmax warps and buffer.
//
// Measured (6.55 TB/s copy, 1632 TFLOP/s burst and 1321 sustained of a library product), both launches:
//   32 sequences of 500 to 8192 tokens decoding, 32 / 8 heads of 128, pages of 16: 119 us, 5.3 TB/s, back to back 125; four
//   times as long 6.5 TB/s: 8 us go to the plan and the first loads, 11 to the spread of the CTAs' ends, 7 to the join.
//   9 rows of f32 over 131072 tokens, 24 / 4 heads of 256: 109 us; back to back 129, the card at 1000 W and 1.6 GHz.
//   4 sequences of 2048 to 16384 tokens over q8_0, 2 to 9 f16 rows, same heads: 71 us, a quarter of memory's rate: 3.3 us per
//   tile and CTA (the conversion, a job of 32 tokens in 0.7 us, is under half of it) and 12 us until the first scores.
//   2048 rows over 32768 tokens, 24 / 4 heads of 256: 1.38 ms, 1155 TFLOP/s; 1.63 back to back at 1.45 GHz (of sustained
//   0.74). Shared memory's reads: QK takes 128 bytes a cycle for M = N = 128, PV 64, the tiles' arrival 64.
//   seven sequences, prompts to 1000 rows and decoding, window 1024, 32 / 8 heads of 128: 137 us: 22 tiles per CTA at 3.4 us, 3
//   to 4 for each item's end (a row per lane: its stores go at a sector per cycle; 2 to 11 items per CTA, so that the slowest
//   is 28 us behind the mean), 12 the join.
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "fa_paged.cuh"
#include "fastdiv.cuh"
#include "internal.h"
#include "launch.cuh"
#include "ptx.cuh"
#include "tc.cuh"

namespace srhpm {
using namespace fap;
namespace {

constexpr int   kBM      = 128;    // rows of a tile
constexpr int   kSmWarps = 8;      // softmax warps
constexpr int   kProd    = 3;      // producer warps (f16 cache)
constexpr int   kConv    = 16;     // converter warps (q8_0 cache): K's two groups of four, then V's
constexpr int   kFew     = 56;     // rows of a tile where sequences bring few (below)
constexpr uint32_t kProbes = 1u << 19;  // of a wait before it gives up: about 2 s (a probe sleeps up to 4 us)
constexpr int   kRawTok  = 32;     // tokens of a raw q8_0 slot
constexpr int   kRawB    = kRawTok * 272;

// ring order of the K and V tiles: the order in which the products take them
// NT = 1: K0 K1 V0 K2 V1 ... V(n-1);  NT = 2: K0 V0 K1 V1 ...
template <int NT> __device__ __forceinline__ int v_pos(int i, int n) {
    return NT == 2 ? 2 * i + 1 : (i == n - 1 ? 2 * n - 1 : 2 * i + 2);
}
template <int NT> __device__ __forceinline__ int k_pos(int i) { return NT == 2 ? 2 * i : (i == 0 ? 0 : 2 * i - 1); }
template <int NT> __device__ __forceinline__ void at_pos(int pos, int n, bool & isk, int & i) {
    if (NT == 2) {
        isk = (pos & 1) == 0;
        i   = pos >> 1;
    } else if (pos == 2 * n - 1) {
        isk = false;
        i   = n - 1;
    } else if (pos == 0 || (pos & 1)) {
        isk = true;
        i   = (pos + 1) >> 1;
    } else {
        isk = false;
        i   = (pos >> 1) - 1;
    }
}

// ---- shared memory -----------------------------------------------------------------------------------------------
template <int D, int NT, int BR, bool PREC, bool Q8> struct Lay {
    // Tokens of a tile. f32 rows over q8_0: 64, since their V ring has one chunk, which then is a whole tile (131072 tokens:
    // 141 us, with 128 162); f16 rows over q8_0: 128 (110 us, with 64 119: the softmax of 64 is mostly waiting).
    static constexpr int BN     = Q8 && PREC ? 64 : 128;
    static constexpr int CH     = BN * D > 128 * 128 ? BN * D / (128 * 128) : 1;  // chunks of a K or V tile, 32 KB at most
    static constexpr int vtok   = BN / CH;                     // tokens of a V chunk
    // tokens of a K chunk: all, with D / CH dims each; q8_0: 64 with all dims, as its V, so that the next tile's first half
    // is converted while the second half is multiplied
    static constexpr int ktok   = Q8 ? 64 : BN;
    static constexpr int kdim   = Q8 ? D : D / CH;
    static constexpr int chunk  = BN * D * 2 / CH;             // bytes of either
    static constexpr int qtile  = BR * D * 2;                  // one part (hi or lo) of one row tile
    static constexpr int qparts = PREC ? 2 : 1;
    static constexpr int q      = 0;                           // [NT][qparts][qtile]
    static constexpr int ring   = NT * qparts * qtile;
    // chunks in flight: what shared memory holds beside Q (at most 8); q8_0 gives the rest to the raw rows
    static constexpr bool copies = NT == 1 && BR <= 64 && D <= 128 && !Q8;  // of rows in each quarter (below)
    static constexpr int  sumb   = copies ? 2 * 4 * 8 * 16 * 4 : 0;
    static constexpr int room   = 232448 - 2400 - sumb - ring;
    // q8_0: K has a ring of two chunks, V one of one or two, the raw rows the rest
    static constexpr int NS     = !Q8 ? (room / chunk < 8 ? room / chunk : 8) : BR < 128 && !PREC ? 4 : 3;
    static constexpr int raw    = ring + NS * chunk;
    static constexpr int NG     = !Q8 ? 0 : (room - NS * chunk) / (4 * kRawB) < 3 ? (room - NS * chunk) / (4 * kRawB) : 3;
    static constexpr int NR     = 4 * NG;                      // raw slots: a ring of NG for each converter group
    static constexpr int red    = raw + NR * kRawB;            // f32 [2][2][128]
    static constexpr int sum    = red + 2 * 2 * kBM * 4;       // f32 [2][4][8][16]
    static constexpr int bar    = sum + sumb;
    static constexpr int nbar   = 2 * NS + 2 * NR + 2 + 2 + 2 + 1;
    static constexpr int misc   = bar + nbar * 8;
    static constexpr int total  = misc + 64;
    static constexpr int alloc  = total;  // dynamic shared memory starts on 1024 bytes (checked by the kernel)
    static constexpr int threads = (kSmWarps + 4 + (Q8 ? kConv : 0)) * 32;  // MMA and producers: the third warpgroup
    static_assert(alloc <= 232448, "shared memory");
    static_assert(Q8 || (NS >= 3 && NS >= CH), "the producers' waits; the wait for V rows that become zeros");
    static_assert(NS * chunk >= kMaxSeqs * 8, "the plan's sums fit the ring");
};

__device__ __forceinline__ void tma4(uint32_t dst, const CUtensorMap * m, int x, int y, int z, int w, uint64_t * bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];" ::"r"(dst),
        "l"(m), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
        : "memory");
}

// One lane of a converged warp. Tensor-core and TMA instructions take their operands from uniform registers: issued
// under elect in warp-uniform code they cost a few cycles each, under `lane == 0` the compiler has to loop over lanes
// that might differ (measured: 190 cycles per product).
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

// A from tensor memory (K-major f16 pairs, lane = row)
__device__ __forceinline__ void mma_f16_ta(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(id), "r"(accumulate), "r"(0u)
        : "memory");
}

__device__ __forceinline__ void ld32(uint32_t t, uint32_t * r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
        "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(t));
}
__device__ __forceinline__ void st32(uint32_t t, const uint32_t * r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(t),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// 32 bytes at a time: a row per lane makes every store of a warp 32 separate sectors, whole ones this way
__device__ __forceinline__ void st_row8(void * p, const uint32_t * r) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]),
                 "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// a wait that ran out marks the kernel's status; the thread then waits for nothing more (its results are void, its
// accesses stay in bounds) so that every role comes to its end
__device__ __forceinline__ void wait_bar(uint64_t * bar, uint32_t parity, int32_t * status, bool & bad) {
    if (bad) return;
    for (uint32_t i = 0; i < kProbes; i++) {
        if (mbar_try_wait(bar, parity)) return;
    }
    bad = true;
    atomicExch(status, kErrWaitFull);
}

// 64 q8_0 values (two blocks, 68 bytes from byte 68 QR of a row) to f16 = round(d * q): the 128-byte row of a swizzled
// plane, 16-byte chunk c at place c ^ (t & 7). The 80 bytes from 64 QR are read in 16-byte loads (rows of 272 bytes: no
// bank conflicts across tokens); the quarter starts QR words into them.
template <int QR> __device__ __forceinline__ void convert_q8(const uint8_t * row, uint8_t * dst_row, int t) {
    uint32_t      w[20];
    const uint4 * src = reinterpret_cast<const uint4 *>(row + 64 * QR);
#pragma unroll
    for (int c = 0; c < 5; c++) {
        const uint4 u = src[c];
        w[4 * c] = u.x; w[4 * c + 1] = u.y; w[4 * c + 2] = u.z; w[4 * c + 3] = u.w;
    }
    const __half2 bias = __halves2half2(__ushort_as_half(0x6480u), __ushort_as_half(0x6480u));  // 1024 + 128
#pragma unroll
    for (int bb = 0; bb < 2; bb++) {
        const int od = 4 * QR + 34 * bb;
        uint32_t  dw;  // d twice
        asm("prmt.b32 %0, %1, %1, %2;" : "=r"(dw) : "r"(w[od >> 2]), "r"((od & 3) ? 0x3232u : 0x1010u));
        const __half2 dd = *reinterpret_cast<const __half2 *>(&dw);
        uint32_t      f[16];
#pragma unroll
        for (int m = 0; m < 16; m++) {
            const int      o  = od + 2 + 2 * m;  // even: the pair sits in one word
            const uint32_t wx = w[o >> 2] ^ 0x80808080u;
            uint32_t       mg;
            asm("prmt.b32 %0, %1, %2, %3;" : "=r"(mg) : "r"(wx), "r"(0x64u), "r"(((o >> 1) & 1) ? 0x4342u : 0x4140u));
            __half2 h = __hsub2(*reinterpret_cast<const __half2 *>(&mg), bias);  // exact: |q| <= 128
            h         = __hmul2(h, dd);
            f[m]      = *reinterpret_cast<const uint32_t *>(&h);
        }
#pragma unroll
        for (int c = 0; c < 4; c++) {
            *reinterpret_cast<uint4 *>(dst_row + (((4 * bb + c) ^ (t & 7)) << 4)) =
                make_uint4(f[4 * c], f[4 * c + 1], f[4 * c + 2], f[4 * c + 3]);
        }
    }
}

template <int D, int NT, int BR, bool PREC, bool Q8>
__global__ void __launch_bounds__(Lay<D, NT, BR, PREC, Q8>::threads, 1)
    fa_paged_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                    const __grid_constant__ PArgs a) {
    using Ly           = Lay<D, NT, BR, PREC, Q8>;
    constexpr int BMN  = BR * NT;
    constexpr int CH   = Ly::CH;
    constexpr int BN   = Ly::BN;
    constexpr int NS   = Ly::NS;
    constexpr int MM   = BR <= 64 ? 64 : 128; // rows of a product
    constexpr int NC   = NT == 2 ? 128 : BN / 2;  // score columns per softmax thread
    constexpr int OC   = NT == 2 ? D : D / 2; // output columns per softmax thread
    // An item of at most 8 rows (decoding) would leave all its softmax to the two warps of tensor memory's first quarter:
    // 64 columns of a row in each thread take 1.3 us a tile, the loads of one of head_dim 64 take 0.7. So its rows stand in
    // each quarter's 16 rows once more, and every quarter takes 16 of a half's 64 columns (P is 0 in the others), 0.8 us:
    // four partial rows with maxima and sums of their own, added up at the item's end. 32 sequences decoding: head_dim 128
    // 118 us, without copies 127; 64 185 and 224; 256 117 and 114 (its tiles load for 2.9 us), so not there.
    constexpr bool COPIES = Ly::copies;
    extern __shared__ __align__(1024) uint8_t sm[];
    uint64_t * kvfull  = reinterpret_cast<uint64_t *>(sm + Ly::bar);
    uint64_t * kvempty = kvfull + NS;
    uint64_t * rfull   = kvempty + NS;
    uint64_t * rempty  = rfull + Ly::NR;
    uint64_t * s_full  = rempty + Ly::NR;  // [2]
    uint64_t * p_rdy   = s_full + 2;       // [2]
    uint64_t * pv_done = p_rdy + 2;        // [2] per row tile (NT = 2) or in turn
    uint64_t * q_full  = pv_done + 2;
    uint32_t * tptr    = reinterpret_cast<uint32_t *>(sm + Ly::misc);
    int *      first   = reinterpret_cast<int *>(sm + Ly::misc + 8);       // s, h, rt, off of the part's first unit
    int64_t *  range   = reinterpret_cast<int64_t *>(sm + Ly::misc + 24);  // part start, end, units in all, parts
    float *    red     = reinterpret_cast<float *>(sm + Ly::red);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    bool      bad = false;
    if (smem_u32(sm) & 1023u) {  // the swizzled operands need it; the linker places the only shared array so
        if (tid == 0) atomicExch(a.status, kErrWaitFull);
        pdl_wait();
        return;
    }

    if (tid == 0) {
        for (int i = 0; i < NS; i++) {
            mbar_init(&kvfull[i], Q8 ? kConv / 2 : 1);
            mbar_init(&kvempty[i], 1);
        }
        for (int i = 0; i < Ly::NR; i++) {
            mbar_init(&rfull[i], 1);
            mbar_init(&rempty[i], 4);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_rdy[i], NT == 2 ? 4 : 8);
            mbar_init(&pv_done[i], 1);
        }
        mbar_init(q_full, kSmWarps);
        fence_mbar_init();
        first[0] = -1;
    }
    if (warp == kSmWarps) tc::tmem_alloc(tptr, 512);
    if (warp == kSmWarps + 1 && lane == 0) {
        prefetch_tmap(&mk);
        prefetch_tmap(&mv);
    }
    pdl_launch_dependents();
    pdl_wait();

    // ---------------- plan: this CTA's part of the line of units ----------------
    // (q8_0: its sums end within the ring, and TMA writes behind it)
    plan_part<BMN, BN, !Q8>(a, reinterpret_cast<int *>(sm + Ly::ring), reinterpret_cast<int *>(sm + Ly::red), first, range);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tbase = *tptr;
    const uint32_t tO    = tbase;        // row tile q: columns q * D
    const uint32_t tS    = tbase + 256;  // buffer b: columns 256 + 128 b
    if (tid == 0) a.desc[2 * blockIdx.x] = make_int4(0, 0, 0, 0);

    Walk w;
    w.s         = first[0];
    bool active = w.s >= 0;
    if (active) {
        w.h   = first[1];
        w.rt  = first[2];
        w.off = first[3];
        w.rem = w.part = range[1] - range[0];
        walk_load<BMN>(a, w);
        walk_item<BMN, BN>(a, w);
    }

    // registers go to the softmax warps (a row of scores each): the launch's 168 (q8_0: 72) per thread, shared out anew
    if (warp < kSmWarps) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Q8 ? 128 : 200));
        // ---------------- softmax ----------------
        const int wg = warp >> 2, wq = warp & 3;
        // row of the tile: its tensor-memory lane, or with M = 64 16 rows in the lower lanes of each quarter
        const int row0 = MM == 64 ? 16 * wq + (lane & 15) : 32 * wq + lane, tl = 32 * wq + lane;
        const int q    = NT == 2 ? wg : 0;                              // row tile
        const int c0   = NT == 2 ? 0 : NC * wg;                         // first score column of this thread
        uint32_t  rc0 = 0, sc[2] = { 0, 0 }, pvc = 0, pvw = 0, turn = 0, items = 0;
        // Q rows of an item to shared memory: 16-byte chunks of 8 dims, 128-byte swizzle. q_issue starts the copies (f32 rows:
        // does nothing yet), q_finish ends with the rows there and the MMA warp told. For the next item q_issue runs as
        // soon as the last scores of the one before are there (its Q is read no more) and q_finish behind its last P: the
        // next scores are then on their way during the epilogue.
        auto q_rows = [&](const Walk & w, bool finish) {
            const int rb = w.rt * BMN + q * BR, rows = max(0, min(BR, w.n * a.G - rb));
            if (PREC == finish && rows > 0) {
                constexpr int per = D / 8, step = (NT == 2 ? 128 : 256) / per;  // rows apart of a thread's chunks
                const int     u0 = NT == 2 ? (tid & 127) : tid, c = u0 % per;
                uint8_t *     d0 = sm + Ly::q + q * Ly::qparts * Ly::qtile + (c >> 3) * (BR * 128);
                // rows behind the last one are zeros: what they give goes nowhere, but random rows heat the products (a
                // 1000 W card lowers its clock for it)
                const int cut = COPIES && rows <= 8 ? 15 : 255;  // row r of the tile holds row r & cut
                auto      source = [&](int r) {
                    const int rr = rb + min(r & cut, rows - 1), t = a.byG.div(rr), h = w.h * a.G + (rr - t * a.G);
                    return a.q + (int64_t) (w.r0 + t) * a.qnb1 + (int64_t) h * a.qnb2;
                };
                auto dest = [&](int r) { return d0 + r * 128 + (((c & 7) ^ (r & 7)) << 4); };
                if constexpr (!PREC) {
#pragma unroll
                    for (int k = 0; k < (BR + step - 1) / step; k++) {
                        const int r = u0 / per + k * step;
                        if (BR % step && r >= BR) break;
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dest(r))), "l"(source(r) + 16 * c), "r"((r & cut) < rows ? 16 : 0) : "memory");
                    }
                } else {
                    constexpr int NK = (BR + step - 1) / step, UN = NK < 4 ? NK : 4;  // rows of a thread, in flight
#pragma unroll 1
                    for (int k0 = 0; k0 < NK; k0 += UN) {
                        float4 x[UN][2];
#pragma unroll
                        for (int k = 0; k < UN; k++) {
                            const float4 * src = reinterpret_cast<const float4 *>(source(u0 / per + (k0 + k) * step)) + 2 * c;
                            x[k][0] = __ldg(src);
                            x[k][1] = __ldg(src + 1);
                        }
#pragma unroll
                        for (int k = 0; k < UN; k++) {
                            if (((u0 / per + (k0 + k) * step) & cut) >= rows) x[k][0] = x[k][1] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                            const float f[8] = { x[k][0].x, x[k][0].y, x[k][0].z, x[k][0].w,
                                                 x[k][1].x, x[k][1].y, x[k][1].z, x[k][1].w };
                            uint32_t    hw[4], lw[4];
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                const __half2 h2 = __floats2half2_rn(f[2 * e], f[2 * e + 1]);
                                const __half2 l2 = __floats2half2_rn(f[2 * e] - __low2float(h2), f[2 * e + 1] - __high2float(h2));
                                hw[e] = *reinterpret_cast<const uint32_t *>(&h2);
                                lw[e] = *reinterpret_cast<const uint32_t *>(&l2);
                            }
                            const int r = u0 / per + (k0 + k) * step;
                            if ((BR % (UN * step)) && r >= BR) break;
                            uint8_t * d = dest(r);
                            *reinterpret_cast<uint4 *>(d)             = make_uint4(hw[0], hw[1], hw[2], hw[3]);
                            *reinterpret_cast<uint4 *>(d + Ly::qtile) = make_uint4(lw[0], lw[1], lw[2], lw[3]);
                        }
                    }
                }
            }
            if (finish) {
                if constexpr (!PREC) asm volatile("cp.async.wait_all;" ::: "memory");
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(q_full);
            }
        };
        auto q_issue  = [&](const Walk & w) { q_rows(w, false); };
        auto q_finish = [&](const Walk & w) { q_rows(w, true); };
        for (bool boot = true; active; boot = false) {  // first a turn without an item, which brings the first one's rows
            const int     n = w.sp.nkv && !boot ? w.take : 0;
            const int     R    = w.n * a.G;
            const int     rb   = w.rt * BMN + q * BR;               // first row of this tile
            const int     rows = max(0, min(BR, R - rb));
            const bool    cop  = COPIES && rows <= 8;
            const int     row  = cop ? row0 & 15 : row0;
            const bool    mine = (MM == 128 || lane < 16) && row < rows;  // this thread's row exists
            const bool    some = cop || MM / 4 * wq < rows;               // the warp has a row
            // the next item, and its rows on their way to L2: from memory they take 2.4 us
            Walk       nw   = w;
            const bool more = boot || walk_next<BMN, BN>(a, nw);
            if (more && nw.sp.nkv && !boot) {
                constexpr int per = D * (PREC ? 4 : 2) / 128;  // lines of a row
                const int     nr  = min(BMN, nw.n * a.G - nw.rt * BMN);
                for (int u = tid; u < nr * per; u += kSmWarps * 32) {
                    const int rr = nw.rt * BMN + u / per, t = a.byG.div(rr), h = nw.h * a.G + (rr - t * a.G);
                    asm volatile("prefetch.global.L2 [%0];" ::"l"(a.q + (int64_t) (nw.r0 + t) * a.qnb1 + (int64_t) h * a.qnb2 + u % per * 128));
                }
            }
            // the row's visible tokens
            const int tok = mine ? a.byG.div(rb + row) : 0;  // of the sequence's new ones
            const int pos = w.kv - w.n + tok;
            const int vhi = mine ? min(pos + 1, w.sp.hi) : 0;
            const int vlo = a.window > 0 ? max(w.sp.lo, (int) max((int64_t) INT32_MIN, (int64_t) pos - a.window + 1)) : 0;
            // what every row of the warp sees
            const int wlo = __reduce_max_sync(0xffffffffu, mine ? vlo : 0), whi = __reduce_min_sync(0xffffffffu, mine ? vhi : INT32_MAX);
            // tokens that every row of the tile sees: no masking there
            const int pmin = w.kv - w.n + a.byG.div(rb), pmax = w.kv - w.n + a.byG.div(rb + max(rows, 1) - 1);
            const int ahi = min(pmin + 1, w.sp.hi);
            const int alo = a.window > 0 ? (int) max((int64_t) 0, (int64_t) pmax - a.window + 1) : 0;
            float     m = -INFINITY, l = 0.0f;
            const bool run = NT == 1 || q == 0 || rows > 0;  // this warp group has units
            // waits until this row tile's first `upto` products P V are done, phase by phase: a parity wait must neither
            // skip a phase nor come after the next one. NT = 1 asks late (two products may end before a slow warp
            // looks), so its products take two barriers in turn, each of which waits for this warp's next P
            auto pv_wait = [&](uint32_t upto) {
                for (; pvw < upto; pvw++) {
                    if constexpr (NT == 2) {
                        wait_bar(&pv_done[q], pvw & 1, a.status, bad);
                    } else {
                        wait_bar(&pv_done[pvw & 1], (pvw >> 1) & 1, a.status, bad);
                    }
                }
            };
            if (n > 0) {
                // a group without units must not arrive for a later item before the other has arrived for this one
                if (!run) wait_bar(q_full, items & 1, a.status, bad);
                items++;
            }
            const bool ahead = more && nw.sp.nkv;  // the next item has rows to bring
            if (ahead && (n == 0 || !run)) {
                q_issue(nw);
                q_finish(nw);
            }
            if (boot) continue;
            // one tile of scores, W columns of a row in each thread of this warp: maximum, exponentials, P
            auto tile = [&](auto width, int i, int t0, uint32_t tb) {
                constexpr int W  = decltype(width)::value;
                const int     cw = W < NC ? c0 + W * wq : c0;
                float         s[W];
                float         mt = -INFINITY;
                if (some) {
                    if constexpr (W >= 32) {
#pragma unroll
                        for (int c = 0; c < W; c += 32) ld32(tb + cw + c, reinterpret_cast<uint32_t *>(s) + c);
                    } else {
                        tc::ld_cols<W>(tb + cw, reinterpret_cast<uint32_t *>(s));
                    }
                    tc::wait_ld();
                    if (a.softcap_l2 != 0.0f) {
#pragma unroll
                        for (int c = 0; c < W; c++) s[c] = a.softcap_l2 * tanhf(s[c] * a.qscale);
                    }
                    constexpr int MW = W < 32 ? W : 32;
                    // per 32 columns: all rows of the warp see them, none does, or lane by lane
                    if (t0 < alo || t0 + BN > ahi) {
#pragma unroll
                        for (int c = 0; c < W; c += MW) {
                            const int u0 = t0 + cw + c;
                            if (u0 >= wlo && u0 + MW <= whi) continue;
                            const int l0 = vlo - u0, h0 = vhi - u0;
#pragma unroll
                            for (int e = 0; e < MW; e++) s[c + e] = e >= l0 && e < h0 ? s[c + e] : -INFINITY;
                        }
                    }
                    float mx[4] = { s[0], s[1], s[2], s[3] };
#pragma unroll
                    for (int c = 4; c < W; c += 2) mx[(c >> 1) & 3] = max3(mx[(c >> 1) & 3], s[c], s[c + 1]);
                    mt = max3(mx[0], mx[1], fmaxf(mx[2], mx[3]));
                }
                if constexpr (NT == 1) {  // the other half of the row; both halves have read S before either writes P
                    float * rd = red + (turn & 1) * 2 * kBM;
                    turn++;
                    rd[wg * kBM + tl] = mt;
                    named_bar_sync(1 + wq, 64);
                    mt = fmaxf(mt, rd[(wg ^ 1) * kBM + tl]);
                }
                if (some) {
                    const float qs = a.softcap_l2 != 0.0f ? 1.0f : a.qscale;
                    mt *= qs;  // log2 units (qs > 0)
                    const bool up = mt > m + kLazy;
                    if (__any_sync(0xffffffffu, up)) {
                        const float mn = up ? mt : m, f = up ? ex2(m - mn) : 1.0f;
                        if (i > 0) {
                            l *= f;
                            pv_wait(pvc);
                            tc::fence_after();
                            const uint32_t to = tc::taddr(tO + q * D, wq, NT == 2 ? 0 : OC * wg);
#pragma unroll 1
                            for (int c = 0; c < OC; c += 32) {
                                uint32_t o[32];
                                ld32(to + c, o);
                                tc::wait_ld();
#pragma unroll
                                for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                                st32(to + c, o);
                            }
                        }
                        m = mn;
                    }
                    const float off = !mine ? INFINITY : (m == -INFINITY ? 0.0f : m) - kShift;  // rows that are none: P = 0
                    const f2    q2 = f2_pack(qs, qs), o2 = f2_pack(-off, -off);
                    f2          l2[2] = { 0ull, 0ull };
                    constexpr int CW = W < 64 ? W : 64;  // columns of a store
#pragma unroll
                    for (int c = 0; c < W; c += CW) {
                        uint32_t hi[CW / 2];
                        [[maybe_unused]] uint32_t lo[CW / 2];
#pragma unroll
                        for (int e = 0; e < CW / 2; e++) {
                            float x0, x1;
                            f2_unpack(f2_fma(f2_pack(s[c + 2 * e], s[c + 2 * e + 1]), q2, o2), x0, x1);
                            x0 = ex2(x0);
                            x1 = ex2(x1);
                            l2[e & 1] = f2_add(l2[e & 1], f2_pack(x0, x1));
                            const __half2 h2 = __floats2half2_rn(x0, x1);
                            hi[e]            = *reinterpret_cast<const uint32_t *>(&h2);
                            if constexpr (PREC) {
                                const __half2 r2 = __floats2half2_rn(x0 - __low2float(h2), x1 - __high2float(h2));
                                lo[e]            = *reinterpret_cast<const uint32_t *>(&r2);
                            }
                        }
                        if constexpr (W < NC) {  // this quarter's columns, zeros in the others'
#pragma unroll
                            for (int k = 0; k < 4; k++) {
                                uint32_t x[W / 2];
#pragma unroll
                                for (int e = 0; e < W / 2; e++) x[e] = k == wq ? hi[e] : 0;
                                tc::st_cols<W / 2>(tb + (c0 + W * k) / 2, x);
                                if constexpr (PREC) {
#pragma unroll
                                    for (int e = 0; e < W / 2; e++) x[e] = k == wq ? lo[e] : 0;
                                    tc::st_cols<W / 2>(tb + BN / 2 + (c0 + W * k) / 2, x);
                                }
                            }
                        } else if constexpr (CW == 64) {
                            st32(tb + (c0 + c) / 2, hi);
                            if constexpr (PREC) st32(tb + BN / 2 + (c0 + c) / 2, lo);
                        } else {
                            tc::st16(tb + (c0 + c) / 2, hi);
                            if constexpr (PREC) tc::st16(tb + BN / 2 + (c0 + c) / 2, lo);
                        }
                    }
                    float y0, y1;
                    f2_unpack(f2_add(l2[0], l2[1]), y0, y1);
                    l += y0 + y1;
                    tc::wait_st();
                }
            };
            for (int i = 0; run && i < n; i++) {
                const int b = NT == 2 ? q : (i & 1), t0 = w.tile(i) * BN;
                wait_bar(&s_full[b], sc[b] & 1, a.status, bad);
                sc[b]++;
                // done: these products were issued before this tile's scores
                if constexpr (NT == 2) {
                    pv_wait(pvc);
                } else if (pvc > 0) {
                    pv_wait(pvc - 1);
                }
                tc::fence_after();
                if (ahead && i == n - 1) q_issue(nw);
                const uint32_t tb = tc::taddr(tS + 128 * b, wq, 0);
                if constexpr (COPIES) {
                    if (cop) {
                        tile(std::integral_constant<int, NC / 4>{}, i, t0, tb);
                    } else {
                        tile(std::integral_constant<int, NC>{}, i, t0, tb);
                    }
                } else {
                    tile(std::integral_constant<int, NC>{}, i, t0, tb);
                }
                pvc++;
                if constexpr (!Q8) {
                    // V rows that no row of the item sees hold anything; 0 * NaN is NaN, so they become zeros
                    if ((NT == 1 || q == 0) && (t0 < w.sp.lo || t0 + BN > w.sp.hi)) {
                        // A wait by parity for this use of a slot passes at once while the use before it is still on its
                        // way, so all chunks up to NS before V's have to be there first. This tile's scores mean that
                        // those up to K of tile i are, whose last one stands 3 CH chunks before V's last: enough for
                        // NS >= 3 CH. Otherwise the next scores mean that K of tile i + 1 is there, the last before V
                        // (and V of tile i - 1: its products were issued before them); in the last tile that V is the
                        // last, and its products' end says so. Neither waits for this tile's P.
                        if constexpr (NT == 1 && NS < 3 * CH) {
                            if (i + 1 < n) {
                                wait_bar(&s_full[b ^ 1], sc[b ^ 1] & 1, a.status, bad);
                            } else {
                                pv_wait(pvc - 1);
                            }
                        }
                        const int z0 = max(0, w.sp.lo - t0), z1 = min(BN, w.sp.hi - t0);  // kept rows
#pragma unroll
                        for (int ch = 0; ch < CH; ch++) {
                            const uint32_t c = rc0 + v_pos<NT>(i, n) * CH + ch, slot = c % NS;
                            wait_bar(&kvfull[slot], (c / NS) & 1, a.status, bad);
                            uint8_t * vb = sm + Ly::ring + slot * Ly::chunk;
                            for (int u = NT == 2 ? (tid & 127) : tid; u < Ly::chunk / 16; u += NT == 2 ? 128 : 256) {
                                const int r = ch * Ly::vtok + (u >> 3) % Ly::vtok;
                                if (r < z0 || r >= z1) *reinterpret_cast<uint4 *>(vb + u * 16) = make_uint4(0, 0, 0, 0);
                            }
                        }
                        fence_proxy_async_smem();
                    }
                }
                tc::fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_rdy[b]);
                if (ahead && i == n - 1) q_finish(nw);
            }
            // ---------------- the item's end ----------------
            if (run && n > 0) {
                pv_wait(pvc);
                tc::fence_after();
            }
            const bool whole = w.off == 0 && w.take == w.sp.units, wide = a.wide != 0;
            float share = 1.0f;  // of a copy's sums in the row's
            if constexpr (NT == 1) {
                float * rd = red + (turn & 1) * 2 * kBM;
                turn++;
                if (!cop || lane < 16) rd[wg * kBM + tl] = l;
                if (COPIES && cop) {
                    if (wg == 0 && lane < 16) rd[kBM + tl + 16] = m;  // lanes that hold no row
                    named_bar_sync(5, kSmWarps * 32);
                    float M = -INFINITY, L = 0.0f;
#pragma unroll
                    for (int k = 0; k < 4; k++) M = fmaxf(M, rd[kBM + 32 * k + 16 + (lane & 15)]);
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const float mk = rd[kBM + 32 * k + 16 + (lane & 15)];
                        L += (mk == -INFINITY && M > mk ? 0.0f : ex2(M == -INFINITY ? 0.0f : mk - M)) * (rd[32 * k + (lane & 15)] + rd[kBM + 32 * k + (lane & 15)]);
                    }
                    share = m == -INFINITY ? 0.0f : ex2(m - M);
                    m     = M;
                    l     = L;
                } else {
                    named_bar_sync(1 + wq, 64);
                    l += rd[(wg ^ 1) * kBM + tl];
                }
            }
            const int     o0 = NT == 2 ? 0 : OC * wg;
            const int     head = w.h * a.G + (rb + row - tok * a.G);
            const int     slot = 2 * blockIdx.x + (w.off == 0 ? 1 : 0);
            float         f    = 1.0f;
            if (whole) {
                float L = l;
                if (a.sinks && mine) {
                    const float sk = a.sinks[head] * kLog2e;
                    // relative to the larger of the two maxima
                    if (sk > m) {
                        const float d = m == -INFINITY ? 0.0f : ex2(m - sk);
                        L             = l * d + exp2f(kShift);
                        f             = d;
                    } else if (sk > -INFINITY) {
                        L += ex2(sk - m + kShift);
                    }
                }
                f = L == 0.0f ? 0.0f : f / L;  // a NaN stays one
            } else if (mine && (NT == 2 || wg == 0) && !(cop && wq > 0)) {
                a.part_ms[(int64_t) slot * a.prow + q * BR + row] = make_float2(m, l);
            }
            if (COPIES && cop) {
                // 16 columns at a time: the four copies' share of 8 rows, added up by 64 threads of this half
                float *   sm_sum = reinterpret_cast<float *>(sm + Ly::sum) + wg * (4 * 8 * 16);
                const int u = tid & 127, orow = u >> 3, ocol = (u & 7) * 2;  // of the sums
                const int otok = a.byG.div(rb + min(orow, rows - 1)), ohead = w.h * a.G + (rb + min(orow, rows - 1) - otok * a.G);
                const float of = whole ? __shfl_sync(0xffffffffu, f, orow & 7) : 1.0f;
                uint8_t *   od = a.dst + (int64_t) ohead * a.dnb1 + (int64_t) (w.r0 + otok) * a.dnb2;
                float *     oa = a.part_acc + ((int64_t) slot * a.prow + min(orow, rows - 1)) * D;
#pragma unroll 1
                for (int c = 0; c < OC; c += 16) {
                    uint32_t o[16];
                    if (n > 0) {
                        tc::ld16(tc::taddr(tO, wq, o0 + c), o);
                        tc::wait_ld();
                        if (lane < 8) {
                            float * to = sm_sum + (wq * 8 + lane) * 16;
#pragma unroll
                            for (int e = 0; e < 16; e += 4) {
                                *reinterpret_cast<float4 *>(to + e) =
                                    make_float4(__uint_as_float(o[e]) * share, __uint_as_float(o[e + 1]) * share,
                                                __uint_as_float(o[e + 2]) * share, __uint_as_float(o[e + 3]) * share);
                            }
                        }
                    }
                    named_bar_sync(6 + wg, 128);
                    if (orow < rows) {
                        float2 x = make_float2(0.0f, 0.0f);
                        if (n > 0) {
#pragma unroll
                            for (int k = 0; k < 4; k++) {
                                const float2 y = *reinterpret_cast<const float2 *>(sm_sum + (k * 8 + orow) * 16 + ocol);
                                x.x += y.x;
                                x.y += y.y;
                            }
                        }
                        if (!whole) {
                            *reinterpret_cast<float2 *>(oa + o0 + c + ocol) = x;
                        } else {
                            x.x = of != 0.0f ? x.x * of : 0.0f;
                            x.y = of != 0.0f ? x.y * of : 0.0f;
                            if constexpr (PREC) {
                                *reinterpret_cast<float2 *>(od + 4 * (o0 + c + ocol)) = x;
                            } else {
                                *reinterpret_cast<__half2 *>(od + 2 * (o0 + c + ocol)) = __floats2half2_rn(x.x, x.y);
                            }
                        }
                    }
                    named_bar_sync(6 + wg, 128);
                }
            } else if (some && run) {
                uint8_t * dst = a.dst;
                float *   acc = a.part_acc;
                if (mine) {
                    dst += (int64_t) head * a.dnb1 + (int64_t) (w.r0 + tok) * a.dnb2;
                    acc += ((int64_t) slot * a.prow + q * BR + row) * D;
                }
#pragma unroll 1
                for (int c = 0; c < OC; c += 32) {
                    uint32_t o[32];
                    if (n > 0) {
                        ld32(tc::taddr(tO + q * D, wq, o0 + c), o);
                        tc::wait_ld();
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; e++) o[e] = 0;
                    }
                    if (!mine) continue;
                    if (!whole) {
#pragma unroll
                        for (int e = 0; e < 32; e += 8) st_row8(acc + o0 + c + e, o + e);
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; e++) o[e] = __float_as_uint(f != 0.0f ? __uint_as_float(o[e]) * f : 0.0f);
                        if constexpr (PREC) {
#pragma unroll
                            for (int e = 0; e < 32; e += 4) {
                                if (wide) {
                                    if ((e & 7) == 0) st_row8(dst + 4 * (o0 + c + e), o + e);
                                } else {
                                    *reinterpret_cast<uint4 *>(dst + 4 * (o0 + c + e)) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                                }
                            }
                        } else {
                            uint32_t h[16];
#pragma unroll
                            for (int k = 0; k < 16; k++) {
                                const __half2 h2 = __floats2half2_rn(__uint_as_float(o[2 * k]), __uint_as_float(o[2 * k + 1]));
                                h[k]             = *reinterpret_cast<const uint32_t *>(&h2);
                            }
#pragma unroll
                            for (int k = 0; k < 16; k += 4) {
                                if (wide) {
                                    if ((k & 7) == 0) st_row8(dst + 2 * (o0 + c) + 4 * k, h + k);
                                } else {
                                    *reinterpret_cast<uint4 *>(dst + 2 * (o0 + c) + 4 * k) = make_uint4(h[k], h[k + 1], h[k + 2], h[k + 3]);
                                }
                            }
                        }
                    }
                }
            }
            tc::fence_before();  // O is read: the next item's products may write it
            if (tid == 0 && !whole && w.off == 0) {
                // this CTA opens an item that others go on with: parts of it, for the merge
                const int64_t end = range[0] + (range[1] - range[0] - w.rem) + w.sp.units;
                const int     e   = part_of_end(range[2], range[3], end, blockIdx.x);
                a.desc[2 * blockIdx.x + 1] = make_int4(w.rt * BMN, min(BMN, R - w.rt * BMN), 0, 0);
                a.desc[2 * blockIdx.x]     = make_int4(e - (int) blockIdx.x + 1, w.h, w.r0, 0);
            }
            rc0 += 2 * n * CH;
            w      = nw;
            active = more;
        }
    } else if (!Q8 || warp < kSmWarps + 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Q8 ? 56 : 104));
        if (warp > kSmWarps && (!Q8 || warp < kSmWarps + 3)) {
            // ---------------- producers ----------------
            // f16: the warps take the chunks in turn. What a warp does once per chunk (entries, waits) took some 1200 cycles
            // when all three shared every chunk's boxes, more than the chunk's loads themselves (32 sequences decoding 127 us,
            // in turn 118; 2048 rows over 32768 tokens 1.58 and 1.40 ms; seven sequences of 4000 135 and 139 us). A wait by
            // parity for the release of slot use c / NS - 1 is safe though a warp has not seen the uses between: its wait for
            // chunk c - 3 means that all chunks up to c - 3 - NS are read, so c - 2 NS is (NS >= 3).
            // q8_0: one warp brings K's raw rows, one V's
            const int pw = warp - kSmWarps - 1;
            uint32_t  rc = 0, issued = 0;     // chunks before the item (q8_0: raw slots so far); end of those brought by this warp
            const int box = a.box;            // q8_0: at most kRawTok
            const int nsub = BN / box;       // boxes per 128 tokens: 2, 4 or 8
            for (; active; active = walk_next<BMN, BN>(a, w)) {
                const int n = w.sp.nkv ? w.take : 0;
                const int32_t * row = reinterpret_cast<const int32_t *>(a.table + (int64_t) w.s * a.tstride);
                // lane j: page and place of the tile's j-th box, -1 when no row sees it
                auto entry = [&](int pos, int & in) -> int {
                    bool isk;
                    int  i;
                    if (Q8) {
                        i = pos;
                    } else {
                        at_pos<NT>(pos, n, isk, i);
                    }
                    const int tok = w.tile(i) * BN + lane * box;
                    if (lane >= nsub || tok >= w.sp.hi || tok + box <= w.sp.lo) return -1;
                    const int pi = a.byPage.div(tok);
                    in           = tok - pi * a.page;
                    const int pg = row[pi];
                    return pg < 0 || pg >= a.n_pages ? a.n_pages : pg;  // no page: outside the map, reads as zeros
                };
                if constexpr (Q8) {
                    int in_next = 0, e_next = n ? entry(0, in_next) : -1;
                    for (int pos = 0; pos < n; pos++) {
                        const int e = e_next, in = in_next;
                        if (pos + 1 < n) e_next = entry(pos + 1, in_next);  // in flight during this tile's waits
                        if (e == a.n_pages) atomicExch(a.status, kErrPage);
                        const CUtensorMap * m = pw == 0 ? &mk : &mv;
                        constexpr uint32_t NG   = Ly::NG;
                        constexpr int      NRAW = BN / kRawTok;
                        const int     per  = kRawTok / box;  // boxes per raw slot: 1 or 2
#pragma unroll 1
                        for (int r = 0; r < NRAW; r++, rc++) {
                            const uint32_t own  = rc >> 1;  // tokens 32 r .. are for group r % 2 of K's or V's two
                            const int      slot = (pw * 2 + (r & 1)) * NG + own % NG;
                            if (own >= NG) wait_bar(&rempty[slot], (own / NG - 1) & 1, a.status, bad);
                            if (bad) break;
                            const uint32_t seen = __ballot_sync(0xffffffffu, e >= 0) >> (r * per) & ((1u << per) - 1);
                            if (elect_one()) mbar_arrive_expect_tx(&rfull[slot], __popc(seen) * box * 272);
                            __syncwarp();
                            for (int j = 0; j < per; j++) {
                                const int ee = __shfl_sync(0xffffffffu, e, r * per + j);
                                const int ii = __shfl_sync(0xffffffffu, in, r * per + j);
                                if (ee >= 0 && elect_one()) {
                                    tma4(smem_u32(sm + Ly::raw + slot * kRawB) + j * box * 272, m, 0, ii, w.h, ee, &rfull[slot]);
                                }
                                __syncwarp();
                            }
                        }
                    }
                } else {
                    const uint32_t nc  = 2 * n * CH;  // chunks of the item
                    uint32_t       cl  = (kProd + pw - rc % kProd) % kProd;
                    int            in = 0, e = cl < nc ? entry(cl / CH, in) : -1;
                    for (; cl < nc; cl += kProd) {
                        const int      ch = cl % CH;
                        const uint32_t c = rc + cl, slot = c % NS;
                        if (e == a.n_pages) atomicExch(a.status, kErrPage);
                        bool isk;
                        int  i;
                        at_pos<NT>(cl / CH, n, isk, i);
                        if (c >= NS) wait_bar(&kvempty[slot], (c / NS - 1) & 1, a.status, bad);
                        if (bad) break;
                        issued = c + 1;
                        // boxes of the chunk: K all tokens and D / CH dims, V tokens 128 / CH and all dims
                        const int      planes = isk ? D / 64 / CH : D / 64;
                        const int      ns = isk ? nsub : nsub / CH;
                        const int      sub0 = isk ? 0 : ch * ns, p0 = isk ? ch * planes : 0, rows = isk ? BN : Ly::vtok;
                        const uint32_t seen = __ballot_sync(0xffffffffu, e >= 0) >> sub0 & ((1u << ns) - 1);
                        const uint32_t at   = smem_u32(sm + Ly::ring + slot * Ly::chunk);
                        const CUtensorMap * m = isk ? &mk : &mv;
                        if (elect_one()) mbar_arrive_expect_tx(&kvfull[slot], __popc(seen) * planes * box * 128);
                        __syncwarp();
#pragma unroll
                        for (int j = 0; j < 8; j++) {  // at most 8 boxes along the tokens
                            if (!(seen >> j & 1)) continue;
                            const int ee = __shfl_sync(0xffffffffu, e, sub0 + j), ii = __shfl_sync(0xffffffffu, in, sub0 + j);
                            if (elect_one()) {
#pragma unroll
                                for (int pl = 0; pl < D / 64; pl++) {
                                    if (pl < planes) tma4(at + (pl * rows + j * box) * 128, m, (p0 + pl) * 64, ii, w.h, ee, &kvfull[slot]);
                                }
                            }
                            __syncwarp();
                        }
                        if (cl + kProd < nc) e = entry((cl + kProd) / CH, in);  // its wait overlaps the next slot's
                    }
                    rc += nc;
                }
                if (bad) break;
            }
            if (bad) {  // the loads in flight land before this CTA's shared memory goes
                if constexpr (Q8) {
                    for (uint32_t c = rc > 2 * Ly::NG ? rc - 2 * Ly::NG : 0; c < rc; c++) {
                        const uint32_t own = c >> 1;
                        mbar_wait(&rfull[(pw * 2 + (c & 1)) * Ly::NG + own % Ly::NG], (own / Ly::NG) & 1);
                    }
                } else {
                    for (uint32_t c = issued > NS ? issued - NS : 0; c < issued; c++) {
                        if (c % kProd == (uint32_t) pw) mbar_wait(&kvfull[c % NS], (c / NS) & 1);
                    }
                }
            }
        } else if (warp == kSmWarps) {
            // ---------------- MMA ----------------
            // the warp walks together, one elected lane issues
            constexpr uint32_t idqk = tc::idesc(tc::kD_F32, tc::kAB_F16, tc::kAB_F16, tc::kKMajor, tc::kKMajor, Ly::ktok, MM);
            constexpr uint32_t idpv = tc::idesc(tc::kD_F32, tc::kAB_F16, tc::kAB_F16, tc::kKMajor, tc::kMNMajor, D, MM);
            constexpr uint64_t sw   = 2ull << 61;
            const uint64_t     qd0  = tc::sdesc(smem_u32(sm + Ly::q), 16, 1024) | sw;  // addresses step by bytes / 16
            const uint64_t     kd0  = tc::sdesc(smem_u32(sm + Ly::ring), 16, 1024) | sw;
            const uint64_t     vd0  = tc::sdesc(smem_u32(sm + Ly::ring), Ly::vtok * 128, 1024) | sw;
            uint32_t           rc0 = 0, items = 0, pc0 = 0, pc1 = 0, pvn = 0;
            // slot and use of a tile's chunk in the ring (rc0: chunks before the item; q8_0: tiles)
            auto chunk_at = [&](bool isk, int i, int n, int ch, uint32_t & use) -> uint32_t {
                uint32_t c;
                if constexpr (Q8) {
                    c = CH * (rc0 + i) + ch;
                    constexpr uint32_t nv = NS - 2;
                    use = isk ? c / 2 : c / nv;
                    return isk ? c % 2 : 2 + c % nv;
                } else {
                    c   = rc0 + (isk ? k_pos<NT>(i) : v_pos<NT>(i, n)) * CH + ch;
                    use = c / NS;
                    return c % NS;
                }
            };
            for (Walk nw; active; w = nw) {
                const int n  = __shfl_sync(0xffffffffu, w.sp.nkv ? w.take : 0, 0);
                const int nr = w.n * a.G - w.rt * BMN;
                nw           = w;  // looked up now: behind the last product it would wait among the epilogue's stores
                active       = walk_next<BMN, BN>(a, nw);
                if (n == 0) continue;
                const int nq = __shfl_sync(0xffffffffu, NT == 2 && nr > BR ? 2 : 1, 0);
                wait_bar(q_full, items & 1, a.status, bad);
                items++;
                tc::fence_after();
                // products of one chunk (the elected lane)
                auto qk_chunk = [&](uint32_t slot, int b, int q, int ch) {
                    const uint64_t kd = kd0 + slot * (Ly::chunk / 16), qd = qd0 + q * (Ly::qparts * Ly::qtile / 16);
                    const uint32_t d  = tS + 128 * b + (Q8 ? ch * Ly::ktok : 0);
#pragma unroll
                    for (int j = 0; j < Ly::kdim / 16; j++) {
                        const int      jj = Q8 ? j : ch * (Ly::kdim / 16) + j;  // k-step over all dims
                        const uint64_t bd = kd + ((j >> 2) * (Ly::ktok * 128) + (j & 3) * 32) / 16;
#pragma unroll
                        for (int part = 0; part < Ly::qparts; part++) {
                            tc::mma_f16(d, qd + (part * Ly::qtile + (jj >> 2) * (BR * 128) + (jj & 3) * 32) / 16, bd, idqk,
                                        (uint32_t) (jj > 0 || part > 0));
                        }
                    }
                };
                auto pv_chunk = [&](uint32_t slot, int b, int q, int ch, bool first) {
                    const uint64_t vd = vd0 + slot * (Ly::chunk / 16);
#pragma unroll
                    for (int j = 0; j < Ly::vtok / 16; j++) {
                        const int jj = ch * (Ly::vtok / 16) + j;
#pragma unroll
                        for (int part = 0; part < Ly::qparts; part++) {
                            mma_f16_ta(tO + q * D, tS + 128 * b + part * (BN / 2) + jj * 8, vd + j * 2048 / 16, idpv,
                                       (uint32_t) (!first || jj > 0 || part > 0));
                        }
                    }
                };
                uint32_t use;
                if constexpr (NT == 1) {
                    auto qk = [&](int i) {
#pragma unroll
                        for (int ch = 0; ch < CH; ch++) {
                            const uint32_t slot = chunk_at(true, i, n, ch, use);
                            wait_bar(&kvfull[slot], use & 1, a.status, bad);
                            tc::fence_after();
                            __syncwarp();
                            if (elect_one()) {
                                qk_chunk(slot, i & 1, 0, ch);
                                tc::commit(&kvempty[slot]);
                                if (ch == CH - 1) tc::commit(&s_full[i & 1]);
                            }
                            __syncwarp();
                        }
                    };
                    qk(0);
                    for (int i = 0; i < n; i++, pvn++) {
                        if (i + 1 < n) qk(i + 1);
                        // V first: it is there before P in most turns, and P's arrival is what the products wait for
                        // (a V ring of one chunk: its second half comes after the first half's products)
                        constexpr int FIRST = Q8 && NS == 3 && CH == 2 ? 1 : CH;
                        uint32_t      sl[CH];
#pragma unroll
                        for (int ch = 0; ch < CH; ch++) {
                            sl[ch] = chunk_at(false, i, n, ch, use);
                            if (ch < FIRST) wait_bar(&kvfull[sl[ch]], use & 1, a.status, bad);
                        }
                        uint32_t & pc = (i & 1) ? pc1 : pc0;
                        wait_bar(&p_rdy[i & 1], pc & 1, a.status, bad);
                        pc++;
#pragma unroll
                        for (int c0 = 0; c0 < CH; c0 += FIRST) {
                            if (c0 > 0) wait_bar(&kvfull[sl[c0]], use & 1, a.status, bad);
                            tc::fence_after();
                            __syncwarp();
                            if (elect_one()) {
#pragma unroll
                                for (int ch = c0; ch < c0 + FIRST; ch++) {
                                    pv_chunk(sl[ch], i & 1, 0, ch, i == 0);
                                    tc::commit(&kvempty[sl[ch]]);
                                }
                                if (c0 + FIRST == CH) tc::commit(&pv_done[pvn & 1]);
                            }
                            __syncwarp();
                        }
                    }
                } else {  // one chunk per tile; K and V are waited for once, before the first row tile's P
                    uint32_t ks = chunk_at(true, 0, n, 0, use), vs = 0;
                    wait_bar(&kvfull[ks], use & 1, a.status, bad);
                    tc::fence_after();
                    __syncwarp();
                    if (elect_one()) {
                        for (int q = 0; q < nq; q++) {
                            qk_chunk(ks, q, q, 0);
                            if (q == nq - 1) tc::commit(&kvempty[ks]);
                            tc::commit(&s_full[q]);
                        }
                    }
                    __syncwarp();
                    for (int i = 0; i < n; i++) {
                        vs = chunk_at(false, i, n, 0, use);
                        wait_bar(&kvfull[vs], use & 1, a.status, bad);
                        if (i + 1 < n) {
                            ks = chunk_at(true, i + 1, n, 0, use);
                            wait_bar(&kvfull[ks], use & 1, a.status, bad);
                        }
                        for (int q = 0; q < nq; q++) {
                            uint32_t & pc = q ? pc1 : pc0;
                            wait_bar(&p_rdy[q], pc & 1, a.status, bad);
                            pc++;
                            tc::fence_after();
                            __syncwarp();
                            if (elect_one()) {
                                pv_chunk(vs, q, q, 0, i == 0);
                                if (q == nq - 1) tc::commit(&kvempty[vs]);
                                tc::commit(&pv_done[q]);
                                if (i + 1 < n) {
                                    qk_chunk(ks, q, q, 0);
                                    if (q == nq - 1) tc::commit(&kvempty[ks]);
                                    tc::commit(&s_full[q]);
                                }
                            }
                            __syncwarp();
                        }
                    }
                }
                rc0 += Q8 ? n : 2 * n * CH;
            }
        }
    } else if constexpr (Q8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(48));
        // ---------------- converters (q8_0): raw rows -> f16 chunks ----------------
        // warp = (K or V; group: 32 of a chunk's 64 tokens; quarter of the row: dims 64 qr .. 64 qr + 63, one swizzled plane).
        // A job is 32 tokens: wait, load, unpack, store and fence take 0.7 us for 250 instructions, so 16 warps work at
        // once; K and V have chunks, raw rows and warps of their own, so that the next K does not queue behind a V that
        // waits for its place. A group takes every use of its raw slots, and of the chunks that it fills, in order: a wait
        // by parity must not skip one.
        const int  qr = warp & 3, grp = ((warp - kSmWarps - 4) >> 2) & 1;
        const bool isk = warp < kSmWarps + 4 + kConv / 2;
        uint32_t   own = 0;  // chunks so far
        for (; active; active = walk_next<BMN, BN>(a, w)) {
            const int n = w.sp.nkv ? w.take : 0;
            for (int i = 0; i < CH * n; i++, own++) {
                const uint32_t ring = isk ? 2 : NS - 2, at = (isk ? 0 : 2) + own % ring;
                const int      slot = ((isk ? 0 : 2) + grp) * Ly::NG + own % Ly::NG;
                if (own >= ring) wait_bar(&kvempty[at], (own / ring - 1) & 1, a.status, bad);
                wait_bar(&rfull[slot], (own / Ly::NG) & 1, a.status, bad);
                uint8_t *       dst = sm + Ly::ring + at * Ly::chunk + qr * (64 * 128) + (32 * grp + lane) * 128;
                const uint8_t * src = sm + Ly::raw + slot * kRawB + lane * 272;
                switch (qr) {
                    case 0: convert_q8<0>(src, dst, lane); break;
                    case 1: convert_q8<1>(src, dst, lane); break;
                    case 2: convert_q8<2>(src, dst, lane); break;
                    default: convert_q8<3>(src, dst, lane); break;
                }
                // V rows that no row of the item sees hold anything; 0 * NaN is NaN, so they become zeros
                const int tok = w.tile(i / CH) * BN + 64 * (i % CH) + 32 * grp + lane;
                if (!isk && (tok < w.sp.lo || tok >= w.sp.hi)) {
#pragma unroll
                    for (int c = 0; c < 8; c++) *reinterpret_cast<uint4 *>(dst + 16 * c) = make_uint4(0, 0, 0, 0);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&rempty[slot]);
                    mbar_arrive(&kvfull[at]);
                }
            }
        }
    }
    __syncwarp();
    tc::fence_before();
    __syncthreads();
    if (warp == kSmWarps) tc::tmem_free(tbase, 512);
}

// The records of an item cut between CTAs, joined in the order of the cuts. CTA c opens the item (record 2c + 1), CTAs
// c + 1 .. c + parts - 1 go on with it (records 2(c + 1), 2(c + 2), ...). Few parts (prompts: two or three, hundreds of
// rows): a warp per row. Many (long caches, few rows): the CTA's 8 warps share out a row's parts, every eighth each, and join
// in shared memory. The border by whole calls over 8000 tokens (a warp per row / shared out, us), where both meet at some 1.5
// rows per part: 6 rows in 37 parts 23.1 / 18.3, 54 in 37 25.4 / 23.8, 24 in 18 25.5 / 25.5, 54 in 18 27.7 / 28.7, 54 in 12
// 36.4 / 38.5 (24 / 4 heads of 256); 4 rows in 9 parts 22.6 / 22.0, 64 in 9 36.5 / 40.9 (32 / 8 heads of 128). Tiles of more
// rows have 16 CTAs per item: 126 rows in 148 parts 58 / 66. Four records of a lane in flight: 16 took so many registers that the cut items of 18 prompts of 64
// tokens were joined in 41 us instead of 17.
// A CTA looks after the items that `per` parts of the line open (8 where every warp has a part of its own: few of those open one).
// records of a row at a time: eight where an item has hundreds (one row over 30000 q4_0 tokens, 24 / 4 heads of 256: 30 us, four at a
// time 38; 32 / 8 heads of 128 the same, 16 sequences of 4000 tokens 41 and 38)
template <int D, int PER> constexpr int kMergeStep = PER > 1 && D == 256 ? 8 : 4;

// PER: parts that a CTA looks after
template <int D, bool F32, int PER>
__global__ void __launch_bounds__(256, kMergeStep<D, PER> == 4 ? 4 : 2) fa_paged_merge_kernel(const __grid_constant__ PArgs a) {
    constexpr int MO = kMergeStep<D, PER>;
    constexpr int V  = D / 32;  // values per lane, in pairs or fours side by side
    constexpr int VW = V >= 4 ? 4 : 2;
    __shared__ float part_s[8][D];
    __shared__ float l_s[8], m_s[8];
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t  open = 1;
    if constexpr (PER > 1) open = __ballot_sync(0xffffffffu, lane < PER && a.desc[2 * (blockIdx.x * PER + lane)].x != 0);
    for (; open; open = PER > 1 ? open & (open - 1) : 0) {
        const int  c  = blockIdx.x * PER + (PER > 1 ? __ffs(open) - 1 : 0);
        const int4 d0 = a.desc[2 * c], d1 = a.desc[2 * c + 1];
        const int  parts = d0.x;
        if (parts == 0) return;
        const bool many = 2 * d1.y <= 3 * parts && d1.y <= 64;
        for (int row = many ? blockIdx.y : blockIdx.y * 8 + warp; row < d1.y; row += many ? gridDim.y : gridDim.y * 8) {
            const int tok = a.byG.div(d1.x + row), h = d0.y * a.G + (d1.x + row - tok * a.G);
            auto      rec = [&](int p) { return (int64_t) (2 * (c + p) + (p == 0 ? 1 : 0)) * a.prow + row; };
            float     M = -INFINITY, L = 0.0f, acc[V];  // of this warp's parts
#pragma unroll
            for (int e = 0; e < V; e++) acc[e] = 0.0f;
            const int first = many ? warp : 0, step = many ? 8 : 1;
            for (int p0 = first; p0 < parts; p0 += MO * step) {
                float  x[MO][V];
                float2 ms[MO];
#pragma unroll
                for (int k = 0; k < MO; k++) {
                    const int p = p0 + k * step;
                    ms[k]       = make_float2(0.0f, 0.0f);
                    if (p < parts) {
                        ms[k]             = __ldcg(a.part_ms + rec(p));
                        const float * src = a.part_acc + rec(p) * D + lane * VW;
#pragma unroll
                        for (int e = 0; e < V; e += VW) {
                            if constexpr (VW == 4) {
                                const float4 f = __ldcg(reinterpret_cast<const float4 *>(src + 32 * e));
                                x[k][e] = f.x; x[k][e + 1] = f.y; x[k][e + 2] = f.z; x[k][e + 3] = f.w;
                            } else {
                                const float2 f = __ldcg(reinterpret_cast<const float2 *>(src + 32 * e));
                                x[k][e] = f.x; x[k][e + 1] = f.y;
                            }
                        }
                    }
                }
                float mn = M;
#pragma unroll
                for (int k = 0; k < MO; k++) mn = ms[k].y == 0.0f ? mn : fmaxf(mn, ms[k].x);
                if (mn > M) {
                    const float f = ex2(M - mn);  // 0 the first time
                    L *= f;
#pragma unroll
                    for (int e = 0; e < V; e++) acc[e] *= f;
                    M = mn;
                }
#pragma unroll
                for (int k = 0; k < MO; k++) {
                    if (!(ms[k].y == 0.0f)) {  // a record without weight may hold anything; a NaN stays one
                        const float w = ex2(ms[k].x - M);
                        L             = fmaf(w, ms[k].y, L);
#pragma unroll
                        for (int e = 0; e < V; e++) acc[e] = fmaf(w, x[k][e], acc[e]);
                    }
                }
            }
            const float sk = a.sinks ? a.sinks[h] * kLog2e : -INFINITY;
            // weights relative to the larger of the maximum and the sink: of the sums so far, of the sink
            auto with_sink = [&](float m, float & ws) {
                const float top = fmaxf(m, sk);
                ws              = sk > -INFINITY ? ex2(sk - top + kShift) : 0.0f;
                return m > -INFINITY ? ex2(m - top) : 0.0f;
            };
            uint8_t *   dst  = a.dst + (int64_t) h * a.dnb1 + (int64_t) (d0.z + tok) * a.dnb2;
            if (!many) {
                float       ws;
                const float wm = with_sink(M, ws);
                L              = L * wm + ws;
                const float f  = L == 0.0f ? 0.0f : wm / L;
#pragma unroll
                for (int e = 0; e < V; e += VW) {
#pragma unroll
                    for (int k = 0; k < VW; k += 2) {
                        const int at = 32 * e + lane * VW + k;
                        if constexpr (F32) {
                            *reinterpret_cast<float2 *>(dst + 4 * at) = make_float2(acc[e + k] * f, acc[e + k + 1] * f);
                        } else {
                            *reinterpret_cast<__half2 *>(dst + 2 * at) = __floats2half2_rn(acc[e + k] * f, acc[e + k + 1] * f);
                        }
                    }
                }
            } else {
#pragma unroll
                for (int e = 0; e < V; e += VW) {
#pragma unroll
                    for (int k = 0; k < VW; k++) part_s[warp][32 * e + lane * VW + k] = acc[e + k];
                }
                if (lane == 0) {
                    l_s[warp] = L;
                    m_s[warp] = M;
                }
                __syncthreads();
                float m = -INFINITY, wt[8], ws;
#pragma unroll
                for (int w = 0; w < 8; w++) m = fmaxf(m, m_s[w]);
                const float wm = with_sink(m, ws);
                L              = ws;
#pragma unroll
                for (int w = 0; w < 8; w++) {
                    wt[w] = m_s[w] > -INFINITY ? ex2(m_s[w] - m) * wm : 0.0f;
                    L     = fmaf(wt[w], l_s[w], L);
                }
                const float f = L == 0.0f ? 0.0f : 1.0f / L;
                for (int at = threadIdx.x; at < D; at += 256) {
                    float o = 0.0f;
#pragma unroll
                    for (int w = 0; w < 8; w++) o = fmaf(wt[w], part_s[w][at], o);
                    if constexpr (F32) {
                        reinterpret_cast<float *>(dst)[at] = o * f;
                    } else {
                        reinterpret_cast<__half *>(dst)[at] = __float2half_rn(o * f);
                    }
                }
                __syncthreads();
            }
        }
    }
}

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                 const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_fn() {
    static EncodeTiled fn = [] {
        void *                          p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess) {
            p = nullptr;
        }
        return reinterpret_cast<EncodeTiled>(p);
    }();
    return fn;
}

// Rows of a CTA's tile by the sequences' average (of the row buffer, padding included: the host knows no more): at most kFew
// (decoding, verifying): one tile of kFew rows, whose Q takes less than half the shared memory of 128 and leaves it to the
// K/V ring. The products have M = 64 there (decode 146 us with 128, 130 with 64): their last 8 rows read what lies behind Q
// and go nowhere. kFew: what lets a q8_0 cache's rings (4 chunks, 8 raw slots) stand beside Q; it holds 9 tokens of 6 heads.
// More: 128 rows, and with head_dim <= 128 two such tiles that share K/V. f32 rows over a q8_0 cache: always kFew (Q's two
// parts of 128 rows do not fit beside the rings). 24 sequences of 500 to 8192 tokens, kFew / full tiles, us by rows of a
// sequence and KV head:
//   32 / 8 heads of 128, f16 rows: 4: 91 / 144, 48: 114 / 160, 64: 205 / 169, 128: 303 / 164; f32: 56: 136 / 221, 64: 187 / 173
//   28 / 4 heads of 128: 28: 64 / 83, 63: 89 / 82, 140: 135 / 91
//   24 / 4 heads of 256, f16: 6: 87 / 84, 54: 83 / 79, 72: 135 / 88; f32: 6: 95 / 98, 54: 122 / 128, 72: 209 / 130
//   the same over q8_0, f16: 6: 149 / 142, 24: 113 / 115, 54: 130 / 140, 72: 217 / 134
// Mixtures, for which the average says little: 64 single tokens beside a prompt of 500 rows 343 / 494 (takes kFew), 8 beside it
// 92 / 105 (takes full tiles), 64 beside 2000 rows 479 / 508 (full). Padding: 32 single tokens in a buffer of 512 rows take
// full tiles, 184 us instead of 111.
struct Tile {
    int nt, br;
};
Tile tile_of(int T, int S, int G, int D, int kv_type, bool f32) {
    if (kv_type == SRHPM_TYPE_Q4_0) return { 1, q4_rows(T, S, G, f32) };
    if ((kv_type == SRHPM_TYPE_Q8_0 && f32) || (int64_t) T * G <= (int64_t) S * kFew) return { 1, kFew };
    return { D <= 128 ? 2 : 1, 128 };
}

template <int D, int NT, int BR, bool PREC, bool Q8>
int launch_paged(srhpm_ctx * ctx, const PArgs & a, const CUtensorMap & mk, const CUtensorMap & mv, cudaStream_t stream) {
    using Ly = Lay<D, NT, BR, PREC, Q8>;
    auto                         kern = fa_paged_kernel<D, NT, BR, PREC, Q8>;
    static std::atomic<unsigned> done{ 0 };
    const unsigned               bit = 1u << (ctx->device & 31);
    if (!(done.load() & bit)) {
        const int st = cuda_status(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Ly::alloc));
        if (st != SRHPM_OK) return st;
        done.fetch_or(bit);
    }
    int st = cuda_status(launch_k_pdl(kern, dim3(ctx->num_sms), dim3(Ly::threads), Ly::alloc, stream, mk, mv, a));
    ctx->launches.fetch_add(1);
    if (st != SRHPM_OK) return st;
    return merge_launch(ctx, a, D, PREC, BR == kFew ? std::min(32, a.prow) : 16, stream);
}

template <int D, bool PREC, bool Q8>
int launch_tile(srhpm_ctx * ctx, Tile t, const PArgs & a, const CUtensorMap & mk, const CUtensorMap & mv, cudaStream_t stream) {
    if (t.br == kFew) return launch_paged<D, 1, kFew, PREC, Q8>(ctx, a, mk, mv, stream);
    if constexpr (PREC && Q8) return SRHPM_ERR_INVALID;  // tile_of gives it kFew rows
    else return launch_paged<D, D <= 128 ? 2 : 1, 128, PREC, Q8>(ctx, a, mk, mv, stream);
}

// Bytes of K's (and of V's) pages as f16 where a q4_0 cache is unpacked once (unpack_q4.cu) and the f16 form attends: f16 rows, more
// than 1.5 head_dim of them per sequence and KV head. Against tiles unpacked as they come, over 30000 tokens: head_dim 256, 384 rows
// 134 us (tiles 125), 600 rows 160 (183); 128, 128 rows 106 (95), 256 rows 117 (127); 64, 64 rows 106 (74), 100 rows 111 (135). Not
// f32 rows, whose sums the f16 form keeps in the tensor cores (off by 2e-5 to 5e-5 over 20000 tokens; fa_paged_q4.cu 6e-6), nor pools
// beyond kMostUnpacked, which were made q4_0 so that they fit.
constexpr size_t kMostUnpacked = (size_t) 512 << 20;
size_t unpacked_bytes(int T, int S, int G, const PagedCache & c, bool f32) {
    if (c.type != SRHPM_TYPE_Q4_0 || f32 || (int64_t) T * G * 2 <= (int64_t) S * c.D * 3) return 0;
    const size_t n = (size_t) c.n_pages * c.page * c.Hkv * c.D * 2;
    return n <= kMostUnpacked ? n : 0;
}

// parts that the line of units is cut into on each SM
int parts_of(int kv_type, Tile t, int D) { return kv_type == SRHPM_TYPE_Q4_0 ? q4_parts(t.br, D) : 1; }

int record_rows(int T, int G, Tile t) { return (int) std::min<int64_t>((int64_t) t.br * t.nt, (int64_t) T * G); }

}  // namespace

bool fap::encode_rows(void * map, const void * p, uint64_t width, int tokens, int64_t pages, int64_t nb1, int64_t nb3, int box, int tokens_box) {
    EncodeTiled enc = encode_fn();
    if (!enc) return false;
    const cuuint64_t dims[3] = { width, (cuuint64_t) tokens, (cuuint64_t) pages }, st[2] = { (cuuint64_t) nb1, (cuuint64_t) nb3 };
    const cuuint32_t bx[3] = { (cuuint32_t) box, (cuuint32_t) tokens_box, 1 }, es[3] = { 1, 1, 1 };
    return enc(static_cast<CUtensorMap *>(map), CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void *>(p), dims, st, bx, es,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int fap::merge_launch(srhpm_ctx * ctx, const PArgs & a, int D, bool f32, int rows_y, cudaStream_t stream, int parts) {
    auto one  = D == 64    ? (f32 ? fa_paged_merge_kernel<64, true, 1> : fa_paged_merge_kernel<64, false, 1>)
                : D == 128 ? (f32 ? fa_paged_merge_kernel<128, true, 1> : fa_paged_merge_kernel<128, false, 1>)
                           : (f32 ? fa_paged_merge_kernel<256, true, 1> : fa_paged_merge_kernel<256, false, 1>);
    auto eight = D == 64    ? (f32 ? fa_paged_merge_kernel<64, true, 8> : fa_paged_merge_kernel<64, false, 8>)
                 : D == 128 ? (f32 ? fa_paged_merge_kernel<128, true, 8> : fa_paged_merge_kernel<128, false, 8>)
                            : (f32 ? fa_paged_merge_kernel<256, true, 8> : fa_paged_merge_kernel<256, false, 8>);
    const int per = parts > 1 ? 8 : 1;
    const int st  = cuda_status(launch_k_pdl(per > 1 ? eight : one, dim3(ctx->num_sms * parts / per, rows_y), dim3(256), 0, stream, a));
    ctx->launches.fetch_add(1);
    return st;
}

size_t fa_paged_work_size(const srhpm_ctx * ctx, int T, int H, int S, const PagedCache & c, bool f32) {
    const int D = c.D, G = H / c.Hkv;
    if (size_t n = unpacked_bytes(T, S, G, c, f32)) {
        PagedCache f = c;
        f.type       = SRHPM_TYPE_F16;
        return 2 * n + 128 + fa_paged_work_size(ctx, T, H, S, f, f32);
    }
    const Tile   t     = tile_of(T, S, G, D, c.type, f32);
    const size_t parts = (size_t) ctx->num_sms * parts_of(c.type, t, D);
    const size_t recs  = 2 * parts * record_rows(T, G, t);
    return recs * D * sizeof(float) + align16(recs * sizeof(float2)) + 2 * parts * sizeof(int4) + 32;
}

int fa_paged_run(srhpm_ctx * ctx, const FaPagedView & v, void * wdata, size_t wsize, cudaStream_t stream) {
    const int D = v.c.D, G = v.H / v.c.Hkv;
    if (v.S > kMaxSeqs || (int64_t) v.T * G + 2 * kBM > INT32_MAX) return SRHPM_UNSUPPORTED;
    // a sequence's units per KV head are counted in 32 bits: tiles of 56 rows or more times tiles of 64 tokens or more
    const int64_t seen = std::min<int64_t>((int64_t) v.cols * v.c.page, INT32_MAX);
    if (v.c.type != SRHPM_TYPE_Q4_0 && ((int64_t) v.T * G / kFew + 1) * (seen / 64 + 1) > INT32_MAX) return SRHPM_UNSUPPORTED;
    if (v.c.type == SRHPM_TYPE_Q4_0 && ((int64_t) v.T * G / 8 + 1) * (seen / 16 + 1) > INT32_MAX) return SRHPM_UNSUPPORTED;
    if (wdata == nullptr || wsize < fa_paged_work_size(ctx, v.T, v.H, v.S, v.c, v.f32)) return SRHPM_ERR_WORKSPACE;
    if (const size_t n = unpacked_bytes(v.T, v.S, G, v.c, v.f32)) {
        uint8_t *   base = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(wdata) + 127) & ~(uintptr_t) 127);
        FaPagedView f    = v;
        const int   st   = unpack_q4_run(ctx, v, base, base + n, stream);
        if (st != SRHPM_OK) return st;
        f.c.type = SRHPM_TYPE_F16;
        f.c.k    = base;
        f.c.v    = base + n;
        f.c.knb2 = f.c.vnb2 = (int64_t) D * 2;
        f.c.knb1 = f.c.vnb1 = f.c.knb2 * v.c.Hkv;
        f.c.knb3 = f.c.vnb3 = f.c.knb1 * v.c.page;
        return fa_paged_run(ctx, f, base + 2 * n, wsize - (size_t) (base + 2 * n - static_cast<uint8_t *>(wdata)), stream);
    }
    const Tile tl = tile_of(v.T, v.S, G, D, v.c.type, v.f32);
    PArgs      a;
    a.q       = v.q;
    a.qnb1    = v.qnb1;
    a.qnb2    = v.qnb2;
    a.dst     = v.dst;
    a.dnb1    = v.dnb1;
    a.dnb2    = v.dnb2;
    a.wide    = ((reinterpret_cast<uintptr_t>(v.dst) | v.dnb1 | v.dnb2) & 31) == 0;
    a.table   = v.table;
    a.tstride = v.tstride;
    a.cols    = v.cols;
    a.page    = v.c.page;
    a.n_pages = (int) v.c.n_pages;
    a.q_start = v.q_start;
    a.kv_len  = v.kv_len;
    a.S       = v.S;
    a.T       = v.T;
    a.H       = v.H;
    a.Hkv     = v.c.Hkv;
    a.G       = G;
    a.window  = v.window;
    a.byG     = FastDiv::of((uint32_t) G);
    a.byPage  = FastDiv::of((uint32_t) v.c.page);
    a.qscale     = v.softcap != 0.0f ? v.scale / v.softcap : v.scale * kLog2e;
    a.softcap_l2 = v.softcap * kLog2e;
    a.sinks      = v.sinks;
    a.prow       = record_rows(v.T, G, tl);
    const size_t recs = (size_t) 2 * ctx->num_sms * parts_of(v.c.type, tl, D) * a.prow;
    uint8_t *    wb   = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(wdata) + 31) & ~(uintptr_t) 31);
    a.part_acc = reinterpret_cast<float *>(wb);
    a.part_ms  = reinterpret_cast<float2 *>(wb + recs * D * sizeof(float));
    a.desc     = reinterpret_cast<int4 *>(wb + recs * D * sizeof(float) + align16(recs * sizeof(float2)));
    a.status   = ctx->d_status;

    if (v.c.type == SRHPM_TYPE_Q4_0) return q4_run(ctx, a, v.c, tl.br, v.f32, stream);
    const bool q8 = v.c.type == SRHPM_TYPE_Q8_0;
    a.box = q8 ? kRawTok : 64;
    while (a.page % a.box) a.box >>= 1;  // the page is a multiple of 16

    EncodeTiled enc = encode_fn();
    if (!enc) return SRHPM_ERR_CUDA;
    CUtensorMap mk, mv;
    for (int i = 0; i < 2; i++) {
        const cuuint64_t row = q8 ? 272 : (cuuint64_t) D * 2;
        // a dimension of one element never steps: any valid stride
        auto str = [&](int64_t nb, int64_t ne) { return ne > 1 ? (cuuint64_t) nb : row; };
        const cuuint64_t dims[4] = { q8 ? 68 : (cuuint64_t) D, (cuuint64_t) v.c.page, (cuuint64_t) v.c.Hkv, (cuuint64_t) v.c.n_pages };
        const cuuint64_t st[3]   = { str(i ? v.c.vnb1 : v.c.knb1, v.c.page), str(i ? v.c.vnb2 : v.c.knb2, v.c.Hkv),
                                     str(i ? v.c.vnb3 : v.c.knb3, v.c.n_pages) };
        const cuuint32_t box[4]  = { q8 ? 68u : 64u, (cuuint32_t) a.box, 1, 1 }, es[4] = { 1, 1, 1, 1 };
        const CUresult   r = enc(i ? &mv : &mk, q8 ? CU_TENSOR_MAP_DATA_TYPE_UINT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 4,
                                 const_cast<uint8_t *>(i ? v.c.v : v.c.k), dims, st, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                 q8 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B,
                                 CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (r != CUDA_SUCCESS) return SRHPM_ERR_INVALID;
    }
    if (q8) return v.f32 ? launch_tile<256, true, true>(ctx, tl, a, mk, mv, stream) : launch_tile<256, false, true>(ctx, tl, a, mk, mv, stream);
    if (D == 64) return v.f32 ? launch_tile<64, true, false>(ctx, tl, a, mk, mv, stream) : launch_tile<64, false, false>(ctx, tl, a, mk, mv, stream);
    if (D == 128) return v.f32 ? launch_tile<128, true, false>(ctx, tl, a, mk, mv, stream) : launch_tile<128, false, false>(ctx, tl, a, mk, mv, stream);
    return v.f32 ? launch_tile<256, true, false>(ctx, tl, a, mk, mv, stream) : launch_tile<256, false, false>(ctx, tl, a, mk, mv, stream);
}

}  // namespace srhpm
