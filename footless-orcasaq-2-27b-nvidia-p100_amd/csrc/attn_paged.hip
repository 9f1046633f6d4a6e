// Attention over the paged KV cache (kv_pages.hpp): chunks of new tokens of
// several sequences, and one to a few tokens a sequence.
//
// The query of a token at position p sees the rows r <= p with r > p - window or
// r < sinks (window 0: all r <= p) whose page is present:
//   z = f16_sat(sum_r e^(scale q.k_r - m) v_r / sum_r e^(scale q.k_r - m)),
// then z = f16_sat(z sigmoid(gate)) where a gate is given; a query that sees no
// row gives 0. Sums, maxima and products are fp32; int8 rows enter as
// f16(byte scale), like everywhere in this library.
//
// One wavefront a (token, q head): a lane holds 4 dims, the dot product is a
// wave sum, the softmax runs along with one maximum and sum.
#include "kv_pages.hpp"

using fl::Pages;
using fl::PAGED_HD;

namespace {

constexpr int MAX_SEQS = FL_PAGED_MAX_SEQS_PREFILL;

// Packed chunks: sequence b's tokens are start[b] .. start[b + 1] - 1, the first
// at position pos0[b].
struct Chunks {
    int n;
    int start[MAX_SEQS + 1];
    int pos0[MAX_SEQS];
};

struct Sight {
    int window, sinks;
};

__device__ __forceinline__ float wave_sum(float v) {
    v += dpp_xor1(v);
    v += dpp_xor2(v);
    v += lane_xor(v, 4);
    v += lane_xor(v, 8);
    v += lane_xor(v, 16);
    return pair32_sum(v);
}

template <bool Q8>
__device__ __forceinline__ f16x4 row4(const void* pool, const Pages& pg, int n_kv, long long row, int h,
                                      int lane) {
    const size_t hr = (size_t)row * n_kv + h;
    if constexpr (Q8) {
        const f16* scales =
            (const f16*)((const char*)pool + (((size_t)pg.n_pages << pg.shift) * n_kv) * PAGED_HD);
        const f16 s = scales[hr * 8 + (lane >> 3)];
        return q8_deq4(*(const uint32_t*)((const char*)pool + hr * PAGED_HD + 4 * lane), (f16x2){s, s});
    } else {
        return *(const f16x4*)((const f16*)pool + hr * PAGED_HD + 4 * lane);
    }
}

// seq's query at position p, head `head` of q row `qrow`, to zrow
template <bool Q8>
__device__ void attend_row(const f16* qrow, const f16* gate, f16* zrow, const void* kpool,
                           const void* vpool, const Pages& pg, long long seq, int p, int h, int n_kv,
                           float sl2, Sight sight) {
    const int lane = threadIdx.x & 63;
    const f16x4 q = *(const f16x4*)(qrow + 4 * lane);
    float m = -INFINITY, l = 0.f;
    f32x4 o = (f32x4)(0.f);
    auto walk = [&](int lo, int hi) {
        for (int r = lo; r < hi; ++r) {
            const long long row = fl::page_row(pg, seq, r);
            if (row < 0) continue;
            const f16x4 k = row4<Q8>(kpool, pg, n_kv, row, h, lane);
            const f16x4 v = row4<Q8>(vpool, pg, n_kv, row, h, lane);
            float s = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) s = fmaf((float)q[e], (float)k[e], s);
            s = wave_sum(s) * sl2;
            const float mn = fmaxf(m, s), c = fast_exp2(m - mn), e2 = fast_exp2(s - mn);
            m = mn;
            l = l * c + e2;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = fmaf(e2, (float)v[e], o[e] * c);
        }
    };
    const int lo = sight.window > 0 ? max(0, p - sight.window + 1) : 0;
    if (lo > 0) walk(0, min(sight.sinks, lo));
    walk(lo, p + 1);
    f16x4 out;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        out[e] = f16_sat(l == 0.f ? 0.f : o[e] / l);
        if (gate != nullptr) out[e] = f16_sat((float)out[e] * sigmoid_f((float)gate[4 * lane + e]));
    }
    *(f16x4*)(zrow + 4 * lane) = out;
}

template <bool Q8>
__global__ void __launch_bounds__(64)
prefill_rows_kernel(const f16* __restrict__ q, int q_pitch, const void* kpool, const void* vpool,
                    const Pages pg, const Chunks ch, f16* __restrict__ z, int z_pitch, int gated,
                    int n_q, int n_kv, float sl2, Sight sight) {
    const int i = blockIdx.x, head = blockIdx.y;
    int seq = 0;
    while (i >= ch.start[seq + 1]) ++seq;
    const size_t rh = (size_t)i * n_q + head;
    const f16* qrow = q + rh * q_pitch;
    attend_row<Q8>(qrow, gated ? qrow + PAGED_HD : nullptr, z + rh * z_pitch, kpool, vpool, pg, seq,
                   ch.pos0[seq] + i - ch.start[seq], head / (n_q / n_kv), n_kv, sl2, sight);
}

template <bool Q8>
__global__ void __launch_bounds__(64)
decode_rows_kernel(const f16* __restrict__ q, int q_pitch, const void* kpool, const void* vpool,
                   const Pages pg, const int* __restrict__ pos0, f16* __restrict__ z, int z_pitch,
                   const f16* __restrict__ gate, int T, int n_q, int n_kv, float sl2, Sight sight) {
    const int i = blockIdx.x, head = blockIdx.y, b = i / T;
    const size_t rh = (size_t)i * n_q + head;
    const long long end = (long long)pg.max_pages << pg.shift;
    const long long p = min((long long)pos0[b] + (i - b * T), end - 1);
    attend_row<Q8>(q + rh * q_pitch, gate ? gate + rh * q_pitch : nullptr, z + rh * z_pitch, kpool,
                   vpool, pg, b, (int)p, head / (n_q / n_kv), n_kv, sl2, sight);
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

int check_heads(const void* q, int q_pitch, const void* z, int z_pitch, int gated, int n_q_heads,
                int n_kv_heads, int window, int sinks) {
    FL_REQUIRE(q && z, "null pointer");
    FL_REQUIRE(n_q_heads >= 1 && n_q_heads <= 4096 && n_q_heads % n_kv_heads == 0,
               "n_q_heads % n_kv_heads");
    FL_REQUIRE(q_pitch >= (gated ? 2 : 1) * PAGED_HD && q_pitch % 8 == 0,
               "q_pitch >= head_dim (2 head_dim with the gate), % 8");
    FL_REQUIRE(z_pitch >= PAGED_HD && z_pitch % 4 == 0, "z_pitch >= head_dim, % 4");
    FL_REQUIRE(aligned16(q) && ((uintptr_t)z & 7) == 0, "q 16-byte, z 8-byte aligned");
    FL_REQUIRE(window >= 0 && sinks >= 0, "window, sinks >= 0");
    return FL_OK;
}

// the chunks of a call; total tokens in ch.start[B]
int make_chunks(const int* Ts, const int* pos0s, int B, int max_pages, int page_size, Chunks& ch) {
    FL_REQUIRE(Ts && pos0s, "null pointer");
    FL_REQUIRE(B >= 1 && B <= MAX_SEQS, "1 <= B <= FL_PAGED_MAX_SEQS_PREFILL");
    ch.n = B;
    long long at = 0;
    for (int b = 0; b < B; ++b) {
        FL_REQUIRE(Ts[b] >= 0 && pos0s[b] >= 0, "T, pos0 >= 0");
        FL_REQUIRE((long long)pos0s[b] + Ts[b] <= (long long)max_pages * page_size,
                   "pos0 + T <= max_pages * page_size");
        ch.start[b] = (int)at;
        ch.pos0[b] = pos0s[b];
        at += Ts[b];
        FL_REQUIRE(at <= (1 << 24), "at most 2^24 tokens a call");
    }
    ch.start[B] = (int)at;
    return FL_OK;
}

}  // namespace

extern "C" {

size_t fl_attention_prefill_paged_work_bytes(const int* Ts, const int* pos0s, int B, int n_q_heads,
                                             int n_kv_heads, int head_dim, int window, int sinks,
                                             int q8) {
    return 0;
}

int fl_attention_prefill_paged(const void* q, int q_pitch, const void* kpool, const void* vpool,
                               int q8, int n_pages, int page_size, const int* pages, int max_pages,
                               long long pages_stride, const int* Ts, const int* pos0s, int B,
                               int n_q_heads, int n_kv_heads, int head_dim, float scale, int window,
                               int sinks, int gated, void* z, int z_pitch, void* work,
                               size_t work_bytes, fl_stream_t stream) {
    Pages pg;
    int rc = fl::make_pages(kpool, vpool, q8, n_pages, page_size, pages, max_pages, pages_stride, B,
                            n_kv_heads, head_dim, pg);
    if (rc) return rc;
    rc = check_heads(q, q_pitch, z, z_pitch, gated, n_q_heads, n_kv_heads, window, sinks);
    if (rc) return rc;
    Chunks ch;
    rc = make_chunks(Ts, pos0s, B, max_pages, page_size, ch);
    if (rc) return rc;
    if (ch.start[B] == 0) return FL_OK;
    auto kernel = q8 ? prefill_rows_kernel<true> : prefill_rows_kernel<false>;
    hipLaunchKernelGGL(kernel, dim3(ch.start[B], n_q_heads), dim3(64), 0, (hipStream_t)stream,
                       (const f16*)q, q_pitch, kpool, vpool, pg, ch, (f16*)z, z_pitch, gated,
                       n_q_heads, n_kv_heads, scale * FL_LOG2E, Sight{window, sinks});
    return fl::check_launch("attention_prefill_paged");
}

size_t fl_attn_decode_paged_work_bytes(int B, int T, int n_q_heads, int n_kv_heads, int head_dim) {
    return 0;
}

int fl_attn_decode_paged(const void* qg, int q_pitch, const void* kpool, const void* vpool, int q8,
                         int n_pages, int page_size, const int* pages, int max_pages,
                         long long pages_stride, const int* pos0, int B, int T, int n_q_heads,
                         int n_kv_heads, int head_dim, float scale, int window, int sinks, int gated,
                         void* z, int z_pitch, void* work, size_t work_bytes, fl_stream_t stream) {
    Pages pg;
    int rc = fl::make_pages(kpool, vpool, q8, n_pages, page_size, pages, max_pages, pages_stride, B,
                            n_kv_heads, head_dim, pg);
    if (rc) return rc;
    rc = check_heads(qg, q_pitch, z, z_pitch, gated, n_q_heads, n_kv_heads, window, sinks);
    if (rc) return rc;
    FL_REQUIRE(pos0, "null pointer");
    FL_REQUIRE(T >= 1 && (long long)T * (n_q_heads / n_kv_heads) <= 32,
               "T * n_q_heads / n_kv_heads <= 32");
    auto kernel = q8 ? decode_rows_kernel<true> : decode_rows_kernel<false>;
    hipLaunchKernelGGL(kernel, dim3(B * T, n_q_heads), dim3(64), 0, (hipStream_t)stream,
                       (const f16*)qg, q_pitch, kpool, vpool, pg, pos0, (f16*)z, z_pitch,
                       gated ? (const f16*)qg + PAGED_HD : nullptr, T, n_q_heads, n_kv_heads,
                       scale * FL_LOG2E, Sight{window, sinks});
    return fl::check_launch("attn_decode_paged");
}

}  // extern "C"
