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

#include <algorithm>
#include <atomic>
#include <type_traits>

#include <math.h>

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
        const float v = l == 0.f ? 0.f : o[e] / l;
        out[e] = f16_sat(gate != nullptr ? v * sigmoid_f((float)gate[4 * lane + e]) : v);
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

// ---------------------------------------------------------------------------
// Decode / verify: T rows a sequence, T G <= 32 query rows a kv head.
//
// The sequences' visible rows as 32-row tiles, a sequence behind the other, make
// one stream a kv head; the stream is cut into equal runs, one a workgroup,
// wherever the cuts fall, so that a batch of unlike contexts fills the chip. Every
// wave finds its run from pos0 itself (a wave scan over the sequences' tiles: no
// host work, so a captured call follows the positions), walks its pieces (a
// sequence's part of the run) and leaves each piece's partial in slot b + run:
// from one piece to the next the sequence or the run steps on, so slots are
// distinct. The merge weighs a sequence's partials and applies the gate.
//
// A tile: wave w takes kv rows 16 (w & 1) .. + 15 and dims 128 (w >> 1) .. + 127,
// so that its 16 rows lie in one page and each row is read in whole lines. The
// query rows are the N columns (32) of S^T = K Q^T on 16x16x32 MFMAs; the two
// waves' partial scores are added through LDS; a lane pair then holds a column, the
// softmax is in-lane and one exchange, and P is the B operand of O^T = V^T P^T
// (V^T transposed through LDS into the slice of the wave that owns its 64 dims).
// ---------------------------------------------------------------------------
constexpr int DT = 32;              // rows a tile
constexpr int D_THREADS = 256;
constexpr int VTP = 36;             // halves a d row of the V^T slices (32 + pad)
constexpr float RESCALE_LOG2 = 8.f;
constexpr int SEQ_COST = 2;         // a further piece's fixed cost in tiles (its q, its partial)
constexpr int RUN_MIN = 2;          // tiles a run, at least

struct DecPart {
    int2* meta;      // [B]: a sequence's first run and its number of partials
    float* pm;       // [slot][n_kv][R], log2 units
    float* pd;
    float* pacc;     // [slot][n_kv][R][256], unnormalised
};

// A sequence's rows in sight of its T tokens: [lo, hi) and [0, min(sinks, hi)),
// as tiles: the first `s` ones, then those from `a` on, n in all.
struct DecSeq {
    int lo0, hi0, lo1, hi1;   // of its first and of its last token
    int s, a, n;
    __device__ __forceinline__ int row0(int j) const { return DT * (j < s ? j : a + j - s); }
};
__device__ __forceinline__ void token_range(long long p, int window, int cap, int& lo, int& hi) {
    hi = (int)max(0ll, min(p + 1, (long long)cap));
    lo = window > 0 ? (int)max(0ll, min(p - window + 1, (long long)INT_MAX)) : 0;
}
__device__ __forceinline__ DecSeq dec_seq(int pos0, int T, const Sight& sight, int cap) {
    DecSeq d;
    token_range(pos0, sight.window, cap, d.lo0, d.hi0);
    token_range((long long)pos0 + T - 1, sight.window, cap, d.lo1, d.hi1);
    d.a = d.lo0 / DT;
    const int e = (d.hi1 + DT - 1) / DT;
    const int sk = min(sight.sinks, d.hi1);
    d.s = sight.window > 0 ? min((sk + DT - 1) / DT, d.a) : 0;
    d.n = d.s + max(0, e - d.a);
    return d;
}

// inclusive sum over the lanes 0 .. l
__device__ __forceinline__ long long wave_scan(int v) {
    const int lane = threadIdx.x & 63;
    long long x = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const long long y = __shfl_up(x, d, 64);
        if (lane >= d) x += y;
    }
    return x;
}
__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ long long uni64(long long x) {
    return ((long long)uni((int)(x >> 32)) << 32) | (uint32_t)uni((int)x);
}

// One tile in flight: K[row 16 (w & 1) + (l & 15)][128 (w >> 1) + 32 (l / 16) + 8 ks
// + 0..7] and V[row 16 (w & 1) + 4 (l & 3) + i][128 (w >> 1) + 8 (l / 4) + 0..7].
struct TileF16 {
    f16x8 k[4], v[4];
};
struct TileQ8 {
    u32x4 k[2];
    u32x2 v[4];
    uint32_t sc;   // lanes < 32 K scales, above V scales: row (l & 15), blocks 4 (w >> 1)
                   // + 2 ((l >> 4) & 1) + 0, 1
};

// `at`: the pool row of the wave's first row (its 16 rows are consecutive)
__device__ __forceinline__ void load_tile(TileF16& t, const char* kp, const char* vp, const Pages&,
                                          long long at, int n_kv, int h, int lane, int w) {
    const uint32_t rs = (uint32_t)n_kv * (2 * PAGED_HD);
    const long long base = at * rs + (2 * PAGED_HD) * h + 256 * (w >> 1);
    const f16x8* ks = (const f16x8*)(kp + base + ((lane & 15) * rs + 64 * (lane >> 4)));
#pragma unroll
    for (int i = 0; i < 4; ++i) t.k[i] = ks[i];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        t.v[i] = __builtin_nontemporal_load(
            (const f16x8*)(vp + base + ((4 * (lane & 3) + i) * rs + 16 * (lane >> 2))));
}
__device__ __forceinline__ void load_tile(TileQ8& t, const char* kp, const char* vp, const Pages& pg,
                                          long long at, int n_kv, int h, int lane, int w) {
    const uint32_t rs = (uint32_t)n_kv * PAGED_HD;
    const long long base = at * rs + PAGED_HD * h + 128 * (w >> 1);
    const u32x4* ks = (const u32x4*)(kp + base + ((lane & 15) * rs + 32 * (lane >> 4)));
    t.k[0] = ks[0];
    t.k[1] = ks[1];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        t.v[i] = __builtin_nontemporal_load(
            (const u32x2*)(vp + base + ((4 * (lane & 3) + i) * rs + 8 * (lane >> 2))));
    const long long sc0 = (((long long)pg.n_pages << pg.shift) * n_kv) * PAGED_HD;
    const char* sp = (lane < 32 ? kp : vp) + sc0 + (at * n_kv + h) * 16 + 8 * (w >> 1);
    t.sc = *(const uint32_t*)(sp + ((lane & 15) * (16 * n_kv) + 4 * ((lane >> 4) & 1)));
}

__device__ __forceinline__ TileF16 expand(const TileF16& t, int) { return t; }
__device__ __forceinline__ TileF16 expand(const TileQ8& q, int lane) {
    TileF16 r;
    // lane (l & 15) + 16 (l / 32)'s dword, half (l / 16) & 1; V 32 lanes above
    auto of = [&](int from) {
        const uint32_t p = (uint32_t)__builtin_amdgcn_ds_bpermute(from << 2, (int)q.sc);
        const f16 s = __builtin_bit_cast(f16x2, p)[(lane >> 4) & 1];
        return (f16x2){s, s};
    };
    const int bl = 16 * (lane >> 5);
    const f16x2 ks2 = of((lane & 15) + bl);
    auto eight = [](uint32_t a, uint32_t b, f16x2 s) {
        const f16x4 lo = q8_deq4(a, s), hi = q8_deq4(b, s);
        return (f16x8){lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    };
    r.k[0] = eight(q.k[0].x, q.k[0].y, ks2);
    r.k[1] = eight(q.k[0].z, q.k[0].w, ks2);
    r.k[2] = eight(q.k[1].x, q.k[1].y, ks2);
    r.k[3] = eight(q.k[1].z, q.k[1].w, ks2);
#pragma unroll
    for (int i = 0; i < 4; ++i) r.v[i] = eight(q.v[i].x, q.v[i].y, of(32 + bl + 4 * (lane & 3) + i));
    return r;
}

template <bool Q8>
__global__ void __launch_bounds__(D_THREADS, Q8 ? 2 : 1)
paged_decode_kernel(const f16* __restrict__ qg, int q_pitch, const char* __restrict__ kp,
                    const char* __restrict__ vp, const Pages pg, const int* __restrict__ pos0, int B,
                    int T, int n_q, int n_kv, int runs, float sl2, const Sight sight,
                    const DecPart out) {
    __shared__ __attribute__((aligned(16))) f32x4 s_part[2][2][4][64];
    __shared__ __attribute__((aligned(16))) f16 s_vt[2][4][64][VTP];
    const int h = blockIdx.x % n_kv, run = blockIdx.x / n_kv;
    const int tid = threadIdx.x, lane = tid & 63;
    const int w = uni(tid >> 6);
    const int hh = lane >> 5, ql = lane & 31;
    const int G = n_q / n_kv, R = T * G;
    const int cap = pg.max_pages << pg.shift;
    const int seq_cost = B > 1 ? SEQ_COST : 1;   // (not 0: a sequence without rows has its place too)

    // the whole stream, and this run's [u, u_end) of it
    auto units = [&](int b) { return dec_seq(pos0[b], T, sight, cap).n + seq_cost; };
    long long total = 0;
    for (int b0 = 0; b0 < B; b0 += 64) {
        const int b = b0 + lane;
        total += uni64(__shfl(wave_scan(b < B ? units(b) : 0), 63, 64));
    }
    // (a little over total / runs: no run is left over)
    const long long per =
        max((long long)((float)total * (1.0001f / (float)runs)) + 1, (long long)RUN_MIN);
    long long u = run * per;
    const long long u_end = min(u + per, total);
    if (u >= u_end) return;   // (the whole workgroup)
    // the sequence that u lies in, and where it starts
    int b = 0;
    long long su = 0;
    for (int b0 = 0; b0 < B; b0 += 64) {
        const int bb = b0 + lane;
        const int un = bb < B ? units(bb) : 0;
        const long long incl = wave_scan(un) + su;
        const int before = __popcll(__ballot(bb < B && incl <= u));
        b = b0 + before;
        if (before < 64) {
            su = uni64(__shfl(incl - un, before, 64));
            break;
        }
        su = uni64(__shfl(incl, 63, 64));
    }
    b = uni(b);

    int tick = 0;   // tiles done: the LDS buffers' turn
    for (;;) {
        const DecSeq d = dec_seq(uni(pos0[b]), T, sight, cap);
        const long long eu = su + d.n + seq_cost;
        const long long pe = min(u_end, eu);
        if (u == su && h == 0 && tid == 0) {
            const long long first = d.n > 0 ? (su + seq_cost) / per : 0;
            out.meta[b] = make_int2((int)first, d.n > 0 ? (int)((eu - 1) / per - first) + 1 : 0);
        }
        const int j0 = (int)max(0ll, u - su - seq_cost), j1 = (int)max(0ll, pe - su - seq_cost);
        if (j1 > j0) {
            // this lane's query column: token tq, q head h G + gq
            const bool qvalid = ql < R;
            const int tq = qvalid ? ql / G : 0, gq = qvalid ? ql - tq * G : 0;
            int qlo, qhi;
            token_range((long long)pos0[b] + tq, sight.window, cap, qlo, qhi);
            // Q[column 16 nb + (l & 15)][128 (w >> 1) + 32 (l / 16) + 8 ks + 0..7]
            f16x8 qreg[8];
#pragma unroll
            for (int nb = 0; nb < 2; ++nb) {
                const int c = 16 * nb + (lane & 15);
                const bool ok = c < R;
                const int t = ok ? c / G : 0, g = ok ? c - t * G : 0;
                const f16* qrow = qg + (((size_t)b * T + t) * n_q + h * G + g) * q_pitch +
                                  128 * (w >> 1) + 32 * (lane >> 4);
#pragma unroll
                for (int ks = 0; ks < 4; ++ks)
                    qreg[4 * nb + ks] = ok ? *(const f16x8*)(qrow + 8 * ks) : (f16x8)(0);
            }
            // page ids of 64 half tiles, a lane each: list tile jb + l / 2, half l & 1
            auto load_ids = [&](int jb) {
                const int j = jb + (lane >> 1);
                return j < j1 ? fl::page_id(pg, b, (d.row0(j) + 16 * (lane & 1)) >> pg.shift) : -1;
            };
            int jb = j0, ids = load_ids(jb), ids_next = load_ids(jb + 32);

            f32x16 o0 = (f32x16)(0.f), o1 = (f32x16)(0.f);
            float m_run = -1e30f, l_run = 0.f;

            typedef typename std::conditional<Q8, TileQ8, TileF16>::type Raw;
            struct Slot {
                Raw raw;
                int id0, id1;
            };
            auto load = [&](Slot& t, int j) {
                if (j - jb >= 32) {
                    jb += 32;
                    ids = ids_next;
                    ids_next = load_ids(jb + 32);
                }
                const int l = 2 * (j - jb);
                t.id0 = __builtin_amdgcn_readlane(ids, l);
                t.id1 = __builtin_amdgcn_readlane(ids, l + 1);
                // the wave's half; an absent page reads page 0 (masked, and v taken as 0)
                const int id = (w & 1) ? t.id1 : t.id0;
                const int in_page = (d.row0(j) + 16 * (w & 1)) & ((1 << pg.shift) - 1);
                load_tile(t.raw, kp, vp, pg, ((long long)max(id, 0) << pg.shift) + in_page, n_kv, h,
                          lane, w);
            };
            auto body = [&](const Slot& t, int j) {
                const int buf = tick & 1;
                TileF16 r = expand(t.raw, lane);
                const int r0 = d.row0(j);
                // every token sees every row of the tile (uniform)
                const bool whole = (t.id0 | t.id1) >= 0 && r0 + DT <= d.hi0 &&
                                   (r0 >= d.lo1 || r0 + DT <= sight.sinks);
                if (!whole) {
                    // rows that no token sees may hold anything: their v must not
                    // meet the product, where 0 x NaN is a NaN
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int row = r0 + 16 * (w & 1) + 4 * (lane & 3) + i;
                        const bool any = ((w & 1) ? t.id1 : t.id0) >= 0 && row < d.hi1 &&
                                         (row >= d.lo0 || row < sight.sinks);
                        r.v[i] = any ? r.v[i] : (f16x8)(0);
                    }
                }
                f32x4 c0 = (f32x4)(0.f), c1 = (f32x4)(0.f);
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) {
                    c0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(r.k[ks], qreg[ks], c0, 0, 0, 0);
                    c1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(r.k[ks], qreg[4 + ks], c1, 0, 0, 0);
                }
                // 16x16x32: lane 16 g + i holds rows 4 g .. + 3 of column i; stored
                // where the 32x32 layout reads rows 8 r4 + 4 hh .. + 3 of column ql
                const int g = lane >> 4, lp = (lane & 15) + 32 * (g & 1);
                s_part[buf][w >> 1][2 * (w & 1) + (g >> 1)][lp] = c0;
                s_part[buf][w >> 1][2 * (w & 1) + (g >> 1)][lp + 16] = c1;
                // V, transposed to [d][kv], for the wave that owns dims 64 w' ..
                const int owner = 2 * (w >> 1) + (lane >> 5), d0 = 8 * ((lane >> 2) & 7);
                const int kv0 = 16 * (w & 1) + 4 * (lane & 3);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    *(f16x4*)&s_vt[buf][owner][d0 + e][kv0] =
                        (f16x4){r.v[0][e], r.v[1][e], r.v[2][e], r.v[3][e]};
                // LDS written (the next tile's loads stay in flight across the barrier)
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
                float sc[16];
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4) {
                    const f32x4 t4 = s_part[buf][0][r4][lane] + s_part[buf][1][r4][lane];
#pragma unroll
                    for (int e = 0; e < 4; ++e) sc[4 * r4 + e] = t4[e];
                }
                if (!whole) {
#pragma unroll
                    for (int rr = 0; rr < 16; ++rr) {
                        const int row = r0 + 8 * (rr >> 2) + 4 * hh + (rr & 3);
                        const bool see = (rr < 8 ? t.id0 : t.id1) >= 0 && row < qhi &&
                                         (row >= qlo || row < sight.sinks);
                        sc[rr] = see ? sc[rr] : -INFINITY;
                    }
                }
                float mt = sc[0];
#pragma unroll
                for (int rr = 1; rr < 16; ++rr) mt = __builtin_elementwise_maximum(mt, sc[rr]);
                mt = pair32_max(mt) * sl2;
                // the running maximum only moves when the tile's is more than
                // RESCALE_LOG2 above it: p <= 256 is exact enough in fp16, and O and l
                // are rescaled on few tiles
                const bool grow = mt > m_run + RESCALE_LOG2;
                if (__any(grow)) {
                    const float m_new = grow ? mt : m_run, corr = fast_exp2(m_run - m_new);
                    m_run = m_new;
                    l_run *= corr;
                    o0 *= corr;
                    o1 *= corr;
                }
                float psum = 0.f;
                f16x8 pk[2];
#pragma unroll
                for (int rr = 0; rr < 16; ++rr) {
                    const float p = fast_exp2(fmaf(sc[rr], sl2, -m_run));
                    psum += p;
                    pk[rr >> 3][rr & 7] = (f16)p;
                }
                l_run += pair32_sum(psum);
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) {
                    auto frag = [&](int dd) {
                        const f16x4 lo4 = *(const f16x4*)&s_vt[buf][w][dd][16 * ks + 4 * hh];
                        const f16x4 hi4 = *(const f16x4*)&s_vt[buf][w][dd][16 * ks + 8 + 4 * hh];
                        return (f16x8){lo4[0], lo4[1], lo4[2], lo4[3], hi4[0], hi4[1], hi4[2], hi4[3]};
                    };
                    o0 = __builtin_amdgcn_mfma_f32_32x32x16_f16(frag(ql), pk[ks], o0, 0, 0, 0);
                    o1 = __builtin_amdgcn_mfma_f32_32x32x16_f16(frag(32 + ql), pk[ks], o1, 0, 0, 0);
                }
                ++tick;
            };
            // two tiles in registers: the next one's loads are issued ahead of this one's math
            Slot t[2];
            load(t[0], j0);
            for (int j = j0; j < j1; j += 2) {
                if (j + 1 < j1) load(t[1], j + 1);
                body(t[0], j);
                if (j + 1 >= j1) break;
                if (j + 2 < j1) load(t[0], j + 2);
                body(t[1], j + 1);
            }
            if (qvalid) {
                const size_t part = ((size_t)(b + run) * n_kv + h) * R + ql;
                float* dst = out.pacc + part * PAGED_HD + 64 * w + 4 * hh;
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4) {
                    *(f32x4*)(dst + 8 * r4) =
                        (f32x4){o0[4 * r4], o0[4 * r4 + 1], o0[4 * r4 + 2], o0[4 * r4 + 3]};
                    *(f32x4*)(dst + 32 + 8 * r4) =
                        (f32x4){o1[4 * r4], o1[4 * r4 + 1], o1[4 * r4 + 2], o1[4 * r4 + 3]};
                }
                if (w == 0 && hh == 0) {
                    out.pm[part] = m_run;
                    out.pd[part] = l_run;
                }
            }
        }
        u = pe;
        if (u >= u_end) return;
        su = eu;
        ++b;
    }
}

// z of every (token, q head) from its sequence's partials: z = f16_sat(sum_s e_s
// acc_s / sum_s e_s d_s sigmoid(gate)), e_s = 2^(m_s - M), rounded once. J waves a
// pair (4: few sequences, many partials each; 1: many sequences), lane l holding
// dims 4 l .. + 3, each wave's partials s = j, j + J, ... in batches whose loads are
// all issued before any is used, the J sums added in order through LDS.
constexpr int MG_BATCH = 8;
template <int J>
__global__ void __launch_bounds__(256)
paged_merge_kernel(const DecPart in, f16* __restrict__ z, int z_pitch, const f16* __restrict__ gate,
                   int g_pitch, int T, int n_q, int n_kv, int n_pairs) {
    __shared__ f32x4 s_num[4][64];
    __shared__ float s_den[4], s_mx[4];
    const int lane = threadIdx.x & 63, w = uni(threadIdx.x >> 6), j = w % J;
    const int rh = blockIdx.x * (4 / J) + w / J;
    if (rh >= n_pairs) return;   // (J waves alike; J 4: the whole workgroup)
    const int i = rh / n_q, head = rh - i * n_q, b = i / T;
    const int G = n_q / n_kv, h = head / G, R = T * G;
    const int2 m2 = in.meta[b];
    const int ns = m2.y;
    f16x4 gv = (f16x4)(0);
    if (gate != nullptr) gv = *(const f16x4*)(gate + (size_t)rh * g_pitch + 4 * lane);
    const size_t step = (size_t)n_kv * R;
    const size_t p0 = ((size_t)(b + m2.x) * n_kv + h) * R + (i - b * T) * G + head - h * G;
    f32x4 num = (f32x4)(0.f);
    float den = 0.f, M = -1e30f;
    for (int s = j; s < ns; s += MG_BATCH * J) {
        float mv[MG_BATCH], dv[MG_BATCH];
        f32x4 av[MG_BATCH];
#pragma unroll
        for (int k = 0; k < MG_BATCH; ++k) {
            const size_t at = p0 + (size_t)min(s + k * J, ns - 1) * step;
            mv[k] = in.pm[at];
            dv[k] = in.pd[at];
            av[k] = *(const f32x4*)(in.pacc + at * PAGED_HD + 4 * lane);
        }
        float bm = M;
#pragma unroll
        for (int k = 0; k < MG_BATCH; ++k) {
            const bool ok = s + k * J < ns;
            mv[k] = ok ? mv[k] : -1e30f;
            dv[k] = ok ? dv[k] : 0.f;
            av[k] = ok ? av[k] : (f32x4)(0.f);
            bm = fmaxf(bm, mv[k]);
        }
        const float corr = fast_exp2(M - bm);
        M = bm;
        num *= corr;
        den *= corr;
#pragma unroll
        for (int k = 0; k < MG_BATCH; ++k) {
            const float e = fast_exp2(mv[k] - M);
#pragma unroll
            for (int c = 0; c < 4; ++c) num[c] = fmaf(e, av[k][c], num[c]);
            den = fmaf(e, dv[k], den);
        }
    }
    if constexpr (J > 1) {
        s_num[w][lane] = num;
        if (lane == 0) s_den[w] = den, s_mx[w] = M;
        __syncthreads();
        if (w != 0) return;
        float Mg = s_mx[0];
        for (int k = 1; k < J; ++k) Mg = fmaxf(Mg, s_mx[k]);
        num = (f32x4)(0.f);
        den = 0.f;
        for (int k = 0; k < J; ++k) {
            const float e = fast_exp2(s_mx[k] - Mg);
            const f32x4 o = s_num[k][lane];
#pragma unroll
            for (int c = 0; c < 4; ++c) num[c] = fmaf(e, o[c], num[c]);
            den = fmaf(e, s_den[k], den);
        }
    }
    const float inv = den == 0.f ? 0.f : 1.f / den;   // (no row seen: 0)
    f16x4 out;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const float v = num[c] * inv;
        out[c] = f16_sat(gate != nullptr ? v * sigmoid_f((float)gv[c]) : v);
    }
    *(f16x4*)(z + (size_t)rh * z_pitch + 4 * lane) = out;
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

// runs a kv head: one workgroup a CU over fp16 pools, two over int8 ones
int dec_runs(int n_kv, bool q8) { return std::max(1, cu_count() * (q8 ? 2 : 1) / n_kv); }

size_t up16(size_t n) { return (n + 15) & ~(size_t)15; }
size_t dec_part(int B, int T, int n_q, int n_kv, int runs, char* work, DecPart& p) {
    const size_t rows = (size_t)(B + runs) * T * n_q;
    const size_t m = up16((size_t)B * sizeof(int2)), f = up16(rows * 4);
    p = {(int2*)work, (float*)(work + m), (float*)(work + m + f), (float*)(work + m + 2 * f)};
    return m + 2 * f + rows * PAGED_HD * 4;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

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
    rc = check_heads(q, q_pitch, z, z_pitch, gated, n_q_heads, n_kv_heads, scale, window, sinks);
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
    if (B < 1 || B > FL_PAGED_MAX_SEQS || n_kv_heads < 1 || n_q_heads < 1 || T < 1 ||
        n_q_heads % n_kv_heads || (long long)T * (n_q_heads / n_kv_heads) > 32 || head_dim != PAGED_HD)
        return 0;
    DecPart p;
    return dec_part(B, T, n_q_heads, n_kv_heads, dec_runs(n_kv_heads, true), nullptr, p);
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
    rc = check_heads(qg, q_pitch, z, z_pitch, gated, n_q_heads, n_kv_heads, scale, window, sinks);
    if (rc) return rc;
    FL_REQUIRE(pos0, "null pointer");
    FL_REQUIRE(T >= 1 && (long long)T * (n_q_heads / n_kv_heads) <= 32,
               "T * n_q_heads / n_kv_heads <= 32");
    DecPart part;
    const int runs = dec_runs(n_kv_heads, q8);
    if (dec_part(B, T, n_q_heads, n_kv_heads, runs, (char*)work, part) > work_bytes || !work) {
        fl::set_error("work: smaller than fl_attn_decode_paged_work_bytes");
        return FL_ESCRATCH;
    }
    FL_REQUIRE(aligned16(work), "16-byte aligned work");
    auto split = q8 ? paged_decode_kernel<true> : paged_decode_kernel<false>;
    hipLaunchKernelGGL(split, dim3(runs * n_kv_heads), dim3(D_THREADS), 0, (hipStream_t)stream,
                       (const f16*)qg, q_pitch, (const char*)kpool, (const char*)vpool, pg, pos0, B, T,
                       n_q_heads, n_kv_heads, runs, scale * FL_LOG2E, Sight{window, sinks}, part);
    rc = fl::check_launch("attn_decode_paged");
    if (rc) return rc;
    const int pairs = B * T * n_q_heads;
    const f16* gate = gated ? (const f16*)qg + PAGED_HD : nullptr;
    const bool wide = runs >= 2 * B;
    auto merge = wide ? paged_merge_kernel<4> : paged_merge_kernel<1>;
    hipLaunchKernelGGL(merge, dim3(wide ? pairs : (pairs + 3) / 4), dim3(256), 0, (hipStream_t)stream,
                       part, (f16*)z, z_pitch, gate, q_pitch, T, n_q_heads, n_kv_heads, pairs);
    return fl::check_launch("attn_decode_paged merge");
}

}  // extern "C"
