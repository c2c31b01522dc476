// Pages given back and moved together (srhpm_page_free, srhpm_page_compact) by host threads at once on one context, each over a pool,
// books and stream of its own. The pools differ in size by a factor of 800, and with them what a launch asks of its kernel: each
// call has to succeed however the others' fall between its steps, and to leave what a lone call leaves.
#include <cuda_runtime.h>

#include <cstdint>
#include <cstdio>
#include <cstring>
#include <string>
#include <thread>
#include <vector>

#include "srhpm_b200.h"

namespace {

constexpr int kHeld = 20, kCalls = 20000;  // the one sequence holds the pool's last pages

struct Book {
    int          pages;
    int32_t *    dev;  // table [kHeld], refs, free list, head, freed, rows / begin / end, held, src, dst, moves, used
    cudaStream_t stream;
    int          bad = 0;
    int32_t *    table() const { return dev; }
    int32_t *    refs() const { return dev + kHeld; }
    int32_t *    list() const { return refs() + pages; }
    int32_t *    src() const { return list() + pages; }
    int32_t *    dst() const { return src() + pages / 2; }
    int32_t *    word(int i) const { return dst() + pages / 2 + i; }
};

bool ok(cudaError_t e, const char * what) {
    if (e != cudaSuccess) std::printf("%s: %s\n", what, cudaGetErrorString(e));
    return e == cudaSuccess;
}

void run(srhpm_ctx * ctx, Book * b, bool compact) {
    srhpm_tensor t;
    std::memset(&t, 0, sizeof t);
    t.type  = SRHPM_TYPE_I32;
    t.ne[0] = kHeld;
    t.ne[1] = t.ne[2] = t.ne[3] = 1;
    t.nb[0] = 4;
    t.nb[1] = t.nb[2] = t.nb[3] = 4 * kHeld;
    t.data = b->table();
    for (int i = 0; i < kCalls; i++) {
        const int st = compact ? srhpm_page_compact(ctx, &t, b->word(2), b->refs(), b->pages, b->list(), b->src(), b->dst(), b->word(3),
                                                    b->word(4), b->stream)
                               // an empty range: what counts is the launch
                               : srhpm_page_free(ctx, b->word(5), nullptr, b->word(5), 1, &t, b->refs(), b->pages, b->list(), b->pages,
                                                 b->word(0), b->word(1), b->stream);
        b->bad += st != SRHPM_OK;
        if (i % 256 == 255) cudaStreamSynchronize(b->stream);
    }
    cudaStreamSynchronize(b->stream);
}

}  // namespace

int main() {
    srhpm_ctx * ctx = nullptr;
    if (srhpm_ctx_create(0, &ctx) != SRHPM_OK) {
        std::printf("no context\n");
        return 1;
    }
    int wrong = 0;
    for (bool compact : { false, true }) {
        std::vector<Book> books;
        for (int pages : { 5000, 1 << 22, 100000, 9000 }) {
            Book                 b{ pages, nullptr, nullptr };
            std::vector<int32_t> h((size_t) kHeld + 3 * (size_t) pages + 8, 0);
            for (int i = 0; i < kHeld; i++) h[i] = pages - kHeld + i;
            for (int i = 0; i < pages; i++) h[kHeld + pages + i] = i;
            int32_t * w = &h[kHeld + 3 * (size_t) pages];
            w[0] = w[2] = kHeld;
            if (!ok(cudaMalloc(&b.dev, 4 * h.size()), "malloc") || !ok(cudaMemcpy(b.dev, h.data(), 4 * h.size(), cudaMemcpyHostToDevice), "copy") ||
                !ok(cudaStreamCreate(&b.stream), "stream")) {
                return 1;
            }
            books.push_back(b);
        }
        std::vector<std::thread> threads;
        for (Book & b : books) threads.emplace_back(run, ctx, &b, compact);
        for (std::thread & t : threads) t.join();
        if (!ok(cudaDeviceSynchronize(), "synchronize")) return 1;
        for (Book & b : books) {
            std::vector<int32_t> h((size_t) kHeld + 3 * (size_t) b.pages + 8);
            if (!ok(cudaMemcpy(h.data(), b.dev, 4 * h.size(), cudaMemcpyDeviceToHost), "copy")) return 1;
            const int32_t *list = &h[kHeld + b.pages], *src = list + b.pages, *dst = src + b.pages / 2;
            int           differ = 0;
            for (int i = 0; i < kHeld; i++) {
                differ += h[i] != (compact ? i : b.pages - kHeld + i);
                if (compact) differ += src[i] != b.pages - kHeld + i || dst[i] != i;
            }
            for (int i = compact ? kHeld : 0; i < b.pages; i++) differ += list[i] != i;
            if (b.bad || differ) std::printf("%s, %d pages: %d of %d calls refused, %d numbers differ\n", compact ? "compact" : "free", b.pages, b.bad, kCalls, differ);
            wrong += b.bad + differ;
            cudaFree(b.dev);
            cudaStreamDestroy(b.stream);
        }
    }
    int32_t code = 0;
    if (srhpm_ctx_check(ctx, &code) != SRHPM_OK) {
        std::printf("device status %d\n", code);
        wrong++;
    }
    srhpm_ctx_destroy(ctx);
    std::printf(wrong ? "FAILED\n" : "ok\n");
    return wrong != 0;
}
