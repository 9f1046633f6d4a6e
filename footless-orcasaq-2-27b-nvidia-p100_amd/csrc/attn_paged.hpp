// Attention over the paged KV cache (kv_pages.hpp): what the decode and the prefill
// kernels share.
//
// The query of a token at position p sees the rows r <= p with r > p - window or
// r < sinks (window 0: all r <= p) whose page is present:
//   z = f16_sat(sum_r e^(scale q.k_r - m) v_r / sum_r e^(scale q.k_r - m) * sigmoid(gate)),
// the gate factor only where a gate is given, rounded once; a query that sees no row
// gives 0. Scores, maxima, sums and O are fp32.
#pragma once

#include "kv_pages.hpp"

#include <atomic>

#include <math.h>

namespace {

using fl::Pages;
using fl::PAGED_HD;

struct Sight {
    int window, sinks;
};

// Softmax weights are held as 2^(s - m), s in log2 units, and go into the product with v in
// fp16. A column's reference m is put P_BELOW under its running maximum and moves only when a
// tile's maximum passes m + P_TOP, so O and l are rescaled on few tiles: weights are at most
// 2^15 (finite in fp16), and the step of fp16's subnormals, 2^-24, is at most 2^-31 of the
// largest weight. With m at the maximum it is 2^-24 of it, and many rows that together weigh
// something beside a heavy first token round to nothing, or to twice their weight: 700 rows of
// 2^-22.7 each were off by 19 %. O, l and the partials' (m, l) carry the same factor.
constexpr float P_BELOW = 7.f, P_TOP = 15.f;
typedef float f32x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }
// the low n bits (none for n <= 0, all from 32 up)
__device__ __forceinline__ uint32_t low_bits(int n) {
    return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u;
}

// The masks of a 32-row tile at row r0 whose 16-row halves lie on pages id0 and id1, a
// bit a row.
struct TileMask {
    int r0, sinks;
    uint32_t here;   // rows on present pages
    __device__ __forceinline__ TileMask(int r0, int id0, int id1, int sinks) : r0(r0), sinks(sinks) {
        here = (id0 < 0 ? 0u : 0xFFFFu) | (id1 < 0 ? 0u : 0xFFFF0000u);
    }
    // of [lo, hi) and [0, min(sinks, hi))
    __device__ __forceinline__ uint32_t rows(int lo, int hi) const {
        return here & low_bits(hi - r0) & (~low_bits(lo - r0) | low_bits(sinks - r0));
    }
    // are they all in it
    __device__ __forceinline__ bool all(int lo, int hi) const {
        return here == ~0u && r0 + 32 <= hi && (r0 >= lo || r0 + 32 <= sinks);
    }
};

// The pages of a sequence's tiles first, first + 2^lg, ... <= last, asked for in that
// order: lane l of a wave holds the table's entry for half l & 1 of the (l / 2)-th of 32
// tiles, and the next 32 tiles' are loaded while those are used (a table entry a tile
// would put its latency in front of every tile's loads). The entries are checked when
// they are taken, on the scalar unit, so that nothing waits for the loads before.
template <class Row0>
struct PageIdsOf {
    const int* row;
    const Pages& pg;
    Row0 row0;
    int last, lg, base, now, next;
    __device__ __forceinline__ int load(int j) const {
        const int lane = threadIdx.x & 63;
        const int r = row0(min(j + ((lane >> 1) << lg), last)) + 16 * (lane & 1);
        return row[min(r >> pg.shift, pg.max_pages - 1)];   // (rows past the table are masked)
    }
    __device__ __forceinline__ PageIdsOf(const Pages& pg, int seq, int first, int last, int lg, Row0 row0)
        : row(pg.table + seq * pg.stride), pg(pg), row0(row0), last(last), lg(lg), base(first) {
        now = load(first);
        next = load(first + (32 << lg));
    }
    // the pages of tile j's halves, -1 where absent
    __device__ __forceinline__ void at(int j, int& id0, int& id1) {
        if (j - base >= 32 << lg) {
            base += 32 << lg;
            now = next;
            next = load(base + (32 << lg));
        }
        const int l = 2 * ((j - base) >> lg);
        id0 = __builtin_amdgcn_readlane(now, l);
        id1 = __builtin_amdgcn_readlane(now, l + 1);
        id0 = (unsigned)id0 < (unsigned)pg.n_pages ? id0 : -1;
        id1 = (unsigned)id1 < (unsigned)pg.n_pages ? id1 : -1;
    }
};
template <class Row0>
__device__ __forceinline__ PageIdsOf<Row0> page_ids(const Pages& pg, int seq, int first, int last, int lg,
                                                    Row0 row0) {
    return PageIdsOf<Row0>(pg, seq, first, last, lg, row0);
}

// A wave-uniform address in global memory (scalar base, 32-bit lane offsets; a
// generic pointer would make flat loads, whose wait the LDS barrier includes).
typedef const __attribute__((address_space(1))) char* gptr;
__device__ __forceinline__ gptr uni_global(const char* p) { return (gptr)uniform_ptr(p); }
template <class V>
__device__ __forceinline__ V load_g(gptr base, uint32_t off) {
    return *(const __attribute__((address_space(1))) V*)(base + off);
}
template <class V>
__device__ __forceinline__ V stream_g(gptr base, uint32_t off) {   // read once: non-temporal
    return __builtin_nontemporal_load((const __attribute__((address_space(1))) V*)(base + off));
}

// four values with f16_sat's range and NaNs, converted in pairs
__device__ __forceinline__ f16x4 f16_sat4(f32x4 v) {
    return __builtin_elementwise_maximum(
        __builtin_elementwise_minimum(__builtin_convertvector(v, f16x4), (f16x4)(f16)65504.f),
        (f16x4)(f16)-65504.f);
}
// sigmoid on the transcendental unit (about 2 ulp; 1 / (1 + e^-x), a NaN stays one)
__device__ __forceinline__ float fast_sigmoid(float x) {
    return __builtin_amdgcn_rcpf(1.f + fast_exp2(x * -FL_LOG2E));
}

// The current device's CU count, looked up once per device.
int cu_count() {
    static std::atomic<int> cached[64];
    int dev = 0, n = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
    if ((n = cached[dev].load()) > 0) return n;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0)
        n = 256;
    cached[dev].store(n);
    return n;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }
size_t up16(size_t n) { return (n + 15) & ~(size_t)15; }

int check_heads(const void* q, int q_pitch, const void* z, int z_pitch, int gated, int n_q_heads,
                int n_kv_heads, float scale, int window, int sinks) {
    FL_REQUIRE(q && z, "null pointer");
    FL_REQUIRE(scale > 0.f && scale < INFINITY, "scale > 0");
    FL_REQUIRE(n_q_heads >= 1 && n_q_heads <= 4096 && n_q_heads % n_kv_heads == 0,
               "n_q_heads % n_kv_heads");
    FL_REQUIRE(q_pitch >= (gated ? 2 : 1) * PAGED_HD && q_pitch % 8 == 0,
               "q_pitch >= head_dim (2 head_dim with the gate), % 8");
    FL_REQUIRE(z_pitch >= PAGED_HD && z_pitch % 4 == 0, "z_pitch >= head_dim, % 4");
    FL_REQUIRE(aligned16(q) && ((uintptr_t)z & 7) == 0, "q 16-byte, z 8-byte aligned");
    FL_REQUIRE(window >= 0 && sinks >= 0, "window, sinks >= 0");
    return FL_OK;
}

}  // namespace
