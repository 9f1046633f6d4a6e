// The paged KV cache's store and its reading back: packed rows of several
// sequences to and from their pages, fp16 or in the int8 format (kv_pages.hpp).
//
// Store: row(pos0[b] + i) <- k[starts[b] + i], int8: per 32 dims the scale
// s = f16(absmax / 127) and rint(x / s) -- kv_store / kv_store_q8's values.
// Load: k[starts[b] + i] <- row(pos0[b] + i), int8: f16(byte s), the value that
// the attention kernels form; rows of an absent page read as zeros.
//
// One wavefront a token, four a workgroup: a token's page is one table entry, and all its
// kv heads are one run of memory on both sides. A lane moves 8 dims (16 bytes of fp16) a
// step, so a 32-dim block is a quad of lanes and its absmax two DPP exchanges. Bound by the
// memory: five contexts of 231k rows in all read back in 178 us (946 MB, 5.3 TB/s; a 2 GiB
// copy reaches 4.9), 13606 int8 rows stored in 20 us and read back in 14.5 (4.3 and 5.9
// TB/s); with the correctly rounded divisions of the contiguous store it took 25. A few
// rows are the lookup's chain of loads (starts, position, table entry) and the launch:
// 3 us for 48, the rows' own loads running meanwhile.
#include "kv_pages.hpp"

#include <math.h>

using fl::Pages;
using fl::PAGED_HD;

namespace {

constexpr int PG_WAVES = 4;            // tokens a workgroup
constexpr int CHUNKS = PAGED_HD / 8;   // 8-dim chunks a head row
constexpr int STEP = 2;                // chunks of K and of V that a lane has in flight

// x / d for d > 0 with r about 1 / d: the product and one correction of it. An exact
// quotient comes out exact, any other within 2 ulp.
__device__ __forceinline__ float div_near(float x, float d, float r) {
    const float q = x * r;
    return fmaf(fmaf(-q, d, x), r, q);
}

// 8 halves of a 32-dim block (4 lanes) in the int8 format, q8_store_row's values. The
// correctly rounded divisions there are most of a store's instructions and are not needed:
// x and the scale s are fp16, so x / s is a half integer exactly or far more than div_near's
// error (2^-15 at most) away from one, and rint takes the same side. With s normal x / s is at
// most 127.1, and |2x - (2n + 1) s| a multiple of the smaller of their units, and x >= s / 4
// there: at least 2^-13 away. With s subnormal (absmax / 127 rounded to a step of 2^-24) x / s
// is at most 190.5, clamped to 127 on both ways, and x and s are multiples of 2^-24 with s <
// 2^-14: at least 2^-11 away. So is absmax / 127, rounded to fp16: 127 t is no multiple of any
// unit near it unless exact.
__device__ __forceinline__ void q8_put(f16x8 x, signed char* vals, f16* scale, bool first) {
    f16x8 m = __builtin_elementwise_abs(x);
    f16x4 m4 = __builtin_elementwise_max((f16x4){m[0], m[1], m[2], m[3]}, (f16x4){m[4], m[5], m[6], m[7]});
    float a = fmaxf(fmaxf((float)m4[0], (float)m4[1]), fmaxf((float)m4[2], (float)m4[3]));
    a = fmaxf(a, dpp_xor1(a));
    a = fmaxf(a, dpp_xor2(a));
    const f16 sh = (f16)(a < INFINITY ? div_near(a, 127.f, 1.f / 127.f) : a);
    const bool on = sh > (f16)0.f;
    const float r = on ? __builtin_amdgcn_rcpf((float)sh) : 0.f;
    const float s = (float)sh < INFINITY ? (float)sh : 0.f;   // (an infinite scale: x / inf = 0)
    u32x2 packed = {0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float v = (float)x[e];
        const int n = (int)__builtin_amdgcn_fmed3f(rintf(div_near(v, s, r)), -127.f, 127.f);
        packed[e >> 2] |= (uint32_t)(n & 0xff) << (8 * (e & 3));
    }
    *(u32x2*)vals = on ? packed : (u32x2){0, 0};
    if (first) *scale = sh;
}

__device__ __forceinline__ f16x8 q8_get(const signed char* vals, f16 s) {
    const u32x2 b = *(const u32x2*)vals;
    const f16x4 lo = q8_deq4(b.x, (f16x2){s, s}), hi = q8_deq4(b.y, (f16x2){s, s});
    return (f16x8){lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}

// chunk c (of n_kv 32) of pool row `row`; the scales follow the pool's values
template <bool Q8>
__device__ __forceinline__ void put_chunk(void* pool, const Pages& pg, int n_kv, long long row,
                                          int c, f16x8 x) {
    const size_t at = (size_t)row * n_kv * CHUNKS + c;
    if constexpr (Q8) {
        f16* scales = (f16*)((char*)pool + (((size_t)pg.n_pages << pg.shift) * n_kv) * PAGED_HD);
        q8_put(x, (signed char*)pool + 8 * at, scales + (at >> 2), (c & 3) == 0);
    } else {
        ((f16x8*)pool)[at] = x;
    }
}
template <bool Q8>
__device__ __forceinline__ f16x8 get_chunk(const void* pool, const Pages& pg, int n_kv, long long row,
                                           int c) {
    const size_t at = (size_t)row * n_kv * CHUNKS + c;
    if constexpr (Q8) {
        const f16* scales =
            (const f16*)((const char*)pool + (((size_t)pg.n_pages << pg.shift) * n_kv) * PAGED_HD);
        return q8_get((const signed char*)pool + 8 * at, scales[at >> 2]);
    } else {
        return ((const f16x8*)pool)[at];
    }
}

template <bool Q8>
__global__ void __launch_bounds__(64 * PG_WAVES)
paged_store_kernel(const f16* __restrict__ k, const f16* __restrict__ v, long long k_stride,
                   long long v_stride, void* __restrict__ kpool, void* __restrict__ vpool,
                   const Pages pg, const int* __restrict__ starts, const int* __restrict__ pos0,
                   int B, int N, int n_kv) {
    const int i = blockIdx.x * PG_WAVES + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (i >= N) return;                                   // wave-uniform
    // the first STEP chunks' loads run while the page is looked up
    const int chunks = n_kv * CHUNKS;
    const f16 *ki = k + i * k_stride, *vi = v + i * v_stride;
    f16x8 kx[STEP], vx[STEP];
    auto load = [&](int c0) {
#pragma unroll
        for (int u = 0; u < STEP; ++u) {
            const int c = c0 + 64 * u;
            if (c < chunks) kx[u] = *(const f16x8*)(ki + 8 * c), vx[u] = *(const f16x8*)(vi + 8 * c);
        }
    };
    load(lane);
    const int seq = fl::seq_of(starts, B, i);
    if (seq >= B || i < starts[seq]) return;              // outside every sequence
    const long long pos = (long long)pos0[seq] + (i - starts[seq]);
    const long long row = pos < 0 || pos > INT_MAX ? -1 : fl::page_row(pg, seq, (int)pos);
    if (row < 0) return;
    for (int c0 = lane; c0 < chunks; c0 += 64 * STEP) {
        if (c0 != lane) load(c0);
#pragma unroll
        for (int u = 0; u < STEP; ++u) {
            const int c = c0 + 64 * u;
            if (c < chunks) {
                put_chunk<Q8>(kpool, pg, n_kv, row, c, kx[u]);
                put_chunk<Q8>(vpool, pg, n_kv, row, c, vx[u]);
            }
        }
    }
}

template <bool Q8>
__global__ void __launch_bounds__(64 * PG_WAVES)
paged_load_kernel(const void* __restrict__ kpool, const void* __restrict__ vpool, const Pages pg,
                  const int* __restrict__ starts, const int* __restrict__ pos0, f16* __restrict__ k,
                  f16* __restrict__ v, long long k_stride, long long v_stride, int zero_rest, int B,
                  int N, int n_kv) {
    const int i = blockIdx.x * PG_WAVES + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (i >= N) return;                                   // wave-uniform
    const int seq = fl::seq_of(starts, B, i);
    long long row = -1;
    bool inside = false;
    if (seq < B && i >= starts[seq]) {
        const long long pos = (long long)pos0[seq] + (i - starts[seq]);
        inside = pos >= 0;
        row = pos < 0 || pos > INT_MAX ? -1 : fl::page_row(pg, seq, (int)pos);
    }
    if (!inside && !zero_rest) return;                    // outside every sequence
    for (int c = lane; c < n_kv * CHUNKS; c += 64) {
        f16x8 kx = (f16x8)(0), vx = (f16x8)(0);
        if (row >= 0) {
            kx = get_chunk<Q8>(kpool, pg, n_kv, row, c);
            vx = get_chunk<Q8>(vpool, pg, n_kv, row, c);
        }
        *(f16x8*)(k + i * k_stride + 8 * c) = kx;
        *(f16x8*)(v + i * v_stride + 8 * c) = vx;
    }
}

int check_rows(const void* k, const void* v, long long k_stride, long long v_stride, const int* starts,
               const int* pos0, int N, int n_kv, int head_dim) {
    FL_REQUIRE(k && v && starts && pos0, "null pointer");
    FL_REQUIRE(N >= 0, "N >= 0");
    FL_REQUIRE(k_stride >= (long long)n_kv * head_dim && v_stride >= (long long)n_kv * head_dim,
               "token strides >= n_kv_heads * head_dim");
    FL_REQUIRE(k_stride % 8 == 0 && v_stride % 8 == 0 && ((uintptr_t)k & 15) == 0 &&
                   ((uintptr_t)v & 15) == 0, "k, v 16-byte aligned, strides % 8");
    return FL_OK;
}

}  // namespace

extern "C" {

int fl_paged_kv_store(const void* k, const void* v, long long k_stride, long long v_stride,
                      void* kpool, void* vpool, int q8, int n_pages, int page_size,
                      const int* pages, int max_pages, long long pages_stride, const int* starts,
                      const int* pos0, int B, int N, int n_kv_heads, int head_dim,
                      fl_stream_t stream) {
    Pages pg;
    int rc = fl::make_pages(kpool, vpool, q8, n_pages, page_size, pages, max_pages, pages_stride, B,
                            n_kv_heads, head_dim, pg);
    if (rc) return rc;
    rc = check_rows(k, v, k_stride, v_stride, starts, pos0, N, n_kv_heads, head_dim);
    if (rc) return rc;
    if (N == 0) return FL_OK;
    auto kernel = q8 ? paged_store_kernel<true> : paged_store_kernel<false>;
    hipLaunchKernelGGL(kernel, dim3((N + PG_WAVES - 1) / PG_WAVES), dim3(64 * PG_WAVES), 0,
                       (hipStream_t)stream, (const f16*)k, (const f16*)v, k_stride, v_stride, kpool,
                       vpool, pg, starts, pos0, B, N, n_kv_heads);
    return fl::check_launch("paged_kv_store");
}

int fl_paged_kv_load(const void* kpool, const void* vpool, int q8, int n_pages, int page_size,
                     const int* pages, int max_pages, long long pages_stride, const int* starts,
                     const int* pos0, void* k, void* v, long long k_stride, long long v_stride,
                     int zero_rest, int B, int N, int n_kv_heads, int head_dim, fl_stream_t stream) {
    Pages pg;
    int rc = fl::make_pages(kpool, vpool, q8, n_pages, page_size, pages, max_pages, pages_stride, B,
                            n_kv_heads, head_dim, pg);
    if (rc) return rc;
    rc = check_rows(k, v, k_stride, v_stride, starts, pos0, N, n_kv_heads, head_dim);
    if (rc) return rc;
    if (N == 0) return FL_OK;
    auto kernel = q8 ? paged_load_kernel<true> : paged_load_kernel<false>;
    hipLaunchKernelGGL(kernel, dim3((N + PG_WAVES - 1) / PG_WAVES), dim3(64 * PG_WAVES), 0,
                       (hipStream_t)stream, kpool, vpool, pg, starts, pos0, (f16*)k, (f16*)v,
                       k_stride, v_stride, zero_rest, B, N, n_kv_heads);
    return fl::check_launch("paged_kv_load");
}

}  // extern "C"
