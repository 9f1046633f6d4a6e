// The paged KV cache: where a sequence's rows lie in a pool of pages.
//
// A pool holds n_pages pages of page_size = 2^shift positions, every row in the
// contiguous caches' layout: fp16 [n_pages page_size][n_kv][256], or the int8
// format of capacity n_pages page_size (all values, then all scales). Position
// p of sequence b is row table[b stride + (p >> shift)] << shift | p % page_size.
// An entry outside [0, n_pages), and a position past the table's max_pages
// columns, is an absent page: the kernels never form an address from it. Its
// rows are not written, read back as zeros and are not attended to.
#pragma once

#include "fl_common.hpp"

#include <limits.h>

namespace fl {

constexpr int PAGE_MIN = 16;        // positions a page, at least (half an attention tile)
constexpr int PAGED_HD = 256;

struct Pages {
    const int* table;
    long long stride;
    int max_pages, n_pages, shift;
};

// The page id of a sequence's page column `col`, -1 where it is absent.
__device__ __forceinline__ int page_id(const Pages& p, long long seq, int col) {
    if ((unsigned)col >= (unsigned)p.max_pages) return -1;
    const int id = p.table[seq * p.stride + col];
    return (unsigned)id < (unsigned)p.n_pages ? id : -1;
}

// The pool row of a position, -1 where its page is absent or pos < 0.
__device__ __forceinline__ long long page_row(const Pages& p, long long seq, int pos) {
    if (pos < 0) return -1;
    const int id = page_id(p, seq, pos >> p.shift);
    return id < 0 ? -1 : ((long long)id << p.shift) + (pos & ((1 << p.shift) - 1));
}

// The sequence of packed token i: how many of starts[1 .. B] are <= i (B: a token
// behind the last sequence). Whole waves; one round of loads for B <= 64.
__device__ __forceinline__ int seq_of(const int* starts, int B, int i) {
    const int lane = threadIdx.x & 63;
    int n = 0;
    for (int b0 = 0; b0 < B; b0 += 64) {
        const int b = b0 + lane;
        n += __popcll(__ballot(b < B && starts[b < B ? b + 1 : B] <= i));
    }
    return n;
}

// The host's checks of a pool and its table, and the kernels' view of them.
inline int make_pages(const void* kpool, const void* vpool, int q8, int n_pages, int page_size,
                      const int* pages, int max_pages, long long pages_stride, int B,
                      int n_kv_heads, int head_dim, Pages& out) {
    FL_REQUIRE(kpool && vpool && pages, "null pointer");
    FL_REQUIRE(q8 == 0 || q8 == 1, "q8 must be 0 or 1");
    FL_REQUIRE(head_dim == PAGED_HD, "head_dim must be 256");
    FL_REQUIRE(n_kv_heads >= 1 && n_kv_heads <= 1024, "1 <= n_kv_heads <= 1024");
    FL_REQUIRE(page_size >= PAGE_MIN && (page_size & (page_size - 1)) == 0 && page_size <= (1 << 24),
               "page_size must be a power of two, 16 or more");
    FL_REQUIRE(n_pages >= 1 && max_pages >= 1, "n_pages, max_pages >= 1");
    FL_REQUIRE((long long)n_pages * page_size <= INT_MAX && (long long)max_pages * page_size <= INT_MAX - 1024,
               "n_pages * page_size, max_pages * page_size < 2^31");
    FL_REQUIRE(pages_stride >= max_pages || B <= 1, "pages_stride >= max_pages");
    FL_REQUIRE(B >= 1 && B <= FL_PAGED_MAX_SEQS, "1 <= B <= FL_PAGED_MAX_SEQS");
    FL_REQUIRE(((uintptr_t)kpool & 15) == 0 && ((uintptr_t)vpool & 15) == 0, "16-byte aligned pools");
    out = {pages, pages_stride, max_pages, n_pages, __builtin_ctz((unsigned)page_size)};
    return FL_OK;
}

}  // namespace fl
