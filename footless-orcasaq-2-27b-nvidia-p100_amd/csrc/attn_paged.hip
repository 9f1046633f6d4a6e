// Decode / verify attention over the paged KV cache: one to a few tokens a sequence
// (attn_paged.hpp says what is computed).
#include "attn_paged.hpp"

#include <algorithm>

using fl::Pages;
using fl::PAGED_HD;

namespace {

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
// ---------------------------------------------------------------------------
constexpr int DT = 32;              // rows a tile
constexpr int D_WAVES = 4;

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
// (p saturates at 2^31 - 1, past any row)
__device__ __forceinline__ void token_range(int p0, int t, int window, int cap, int& lo, int& hi) {
    const int p = __builtin_elementwise_add_sat(p0, t);
    hi = max(0, min(p, cap - 1) + 1);
    lo = window > 0 ? max(0, __builtin_elementwise_sub_sat(p, window - 1)) : 0;
}
__device__ __forceinline__ DecSeq dec_seq(int pos0, int T, const Sight& sight, int cap) {
    DecSeq d;
    token_range(pos0, 0, sight.window, cap, d.lo0, d.hi0);
    token_range(pos0, T - 1, sight.window, cap, d.lo1, d.hi1);
    d.a = d.lo0 / DT;
    const int e = (d.hi1 + DT - 1) / DT;
    const int sk = min(sight.sinks, d.hi1);
    d.s = sight.window > 0 ? min((sk + DT - 1) / DT, d.a) : 0;
    d.n = d.s + max(0, e - d.a);
    return d;
}

// Query heads a kv head, and the token of a query row (rows under 32): r / G by a product.
struct QHeads {
    int G, inv;
    __device__ __forceinline__ int token(int r) const { return r * inv >> 16; }
};

// inclusive sum over the lanes 0 .. l (DPP row shifts, then the rows' totals)
__device__ __forceinline__ int wave_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, true);   // row_shr 1
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, true);   // row_bcast 15
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, true);   // row_bcast 31
    return x;
}
// How a stream is cut: runs a kv head, tiles a run at least, and what a sequence costs
// ahead of its tiles, in tiles. A workgroup may take 2, .. 2^heads_lg kv heads, and runs are
// that much shorter then (Run).
struct Cut {
    int runs, run_min, seq_cost, heads_lg;
};
constexpr int LONG_RUN = 64;    // tiles a run of one head
constexpr int SHORT_SEQ = 16;   // tiles a sequence, with its cost
// A workgroup's run of the stream: its kv heads, and the pieces one after the other.
struct Run {
    int h, heads_lg;          // kv heads h << heads_lg .. + 2^heads_lg - 1
    int run, per;             // runs are `per` units long
    int u, u_end;             // what is left of this one
    int b, su, cost;          // the sequence that u lies in, where it starts, units ahead of its tiles
    bool any;

    // Workgroups go to the 8 XCDs round-robin: the kv heads of a run go to one of them
    // (their rows share lines of scales), the runs to all.
    __device__ __forceinline__ Run(const int* pos0, int B, int T, int n_kv, const Cut& cut,
                                   const Sight& sight, int cap) {
        const int id = blockIdx.x, lane = threadIdx.x & 63;
        cost = B > 1 ? cut.seq_cost : 1;   // (not 0: a sequence without rows has its place too)
        auto units = [&](int s) { return dec_seq(pos0[s], T, sight, cap).n + cost; };
        int total = 0, scan = 0, un = 0;   // (of the last 64 sequences: the first ones if B <= 64)
        for (int b0 = 0; b0 < B; b0 += 64) {   // (the host has checked: under 2^31 tiles)
            un = b0 + lane < B ? units(b0 + lane) : 0;
            scan = wave_scan(un);
            total += __builtin_amdgcn_readlane(scan, 63);
        }
        // Waves of a workgroup that take all kv heads of a row read it whole: 64 contexts of
        // 30 - 50k 869 us against 937 with a head a workgroup, 64 of 100 - 32k 145 against 159,
        // 16 of 8k 58.4 against 60.2. With shorter runs the waves of a head rather go
        // through its tiles together (fewer partials): one context of 32k 27.9 against 42.0, 4
        // of 8k 24.7 against 29.7. Sequences shorter than their waves: 96 of 50 17.2 with two
        // heads, 19.2 with one, 22.1 with four.
        const int lg = total / LONG_RUN >= cut.runs ? 2 : total < SHORT_SEQ * B ? 1 : 0;
        heads_lg = min(lg, cut.heads_lg);
        const int runs = cut.runs << heads_lg, groups = n_kv >> heads_lg;
        const bool even = runs % 8 == 0;
        const int slot = even ? id >> 3 : id;
        h = slot % groups;
        run = even ? slot / groups * 8 + (id & 7) : slot / groups;
        // (a little over total / runs: no run is left over)
        per = max((int)((float)total * (1.0001f / (float)runs)) + 1, cut.run_min >> heads_lg);
        any = (long long)run * per < total;
        if (!any) return;
        u = run * per;
        u_end = (int)min((long long)u + per, (long long)total);
        b = su = 0;
        for (int b0 = 0; b0 < B; b0 += 64) {
            if (B > 64) {
                un = b0 + lane < B ? units(b0 + lane) : 0;
                scan = wave_scan(un);
            }
            const int before = __popcll(__ballot(b0 + lane < B && scan <= u - su));
            b = b0 + before;
            if (before < 64) {
                su += __builtin_amdgcn_readlane(scan - un, before);
                break;
            }
            su += __builtin_amdgcn_readlane(scan, 63);
        }
    }
    // The tiles [j0, j1) of sequence b that this run has, and the sequence's note for
    // the merge from the run that it starts in.
    __device__ __forceinline__ void piece(const DecSeq& d, const DecPart& out, int& j0, int& j1) const {
        const int eu = su + d.n + cost;
        if (u == su && h == 0 && threadIdx.x == 0) {
            const int first = d.n > 0 ? (su + cost) / per : 0;
            out.meta[b] = make_int2(first, d.n > 0 ? (eu - 1) / per - first + 1 : 0);
        }
        j0 = max(0, u - su - cost);
        j1 = max(0, min(u_end, eu) - su - cost);
    }
    // on to the next sequence; false at the run's end
    __device__ __forceinline__ bool next(const DecSeq& d) {
        u = su = su + d.n + cost;
        ++b;
        return u < u_end;
    }
};

// ---------------------------------------------------------------------------
// fp16 pools. The four waves share a tile: wave w takes kv rows 16 (w & 1) .. + 15 and
// dims 128 (w >> 1) .. + 127, so that its 16 rows lie in one page and each row is read
// in whole lines. The query rows are the N columns (32) of S^T = K Q^T on 16x16x32
// MFMAs; the two waves' partial scores are added through LDS; a lane pair then holds a
// column, the softmax is in-lane and one exchange, and P, rounded to fp16, is the B
// operand of O^T = V^T P^T (V^T transposed through LDS into the slice of the wave that
// owns its 64 dims).
//
// Bound by the memory: 6 contexts of 60 - 100k with 18 rows 345 us (2.33 GB, 6.7 TB/s), 64
// of 100 - 32k with 6 rows 230 (6.6). A wave a tile alone, as over int8 pools, takes 364 and
// 257: its 16 KiB of K and 16 of V a tile leave registers for one wave a SIMD. Two
// workgroups a CU: 358, and 4 contexts of 8k 33.7 against 29.5. V is read once by one
// workgroup, non-temporal; K as well, but its lines by four instructions each.
// A small call is two launches and their chains of loads (positions, table, rows;
// partials): one context of 500 9.7 us in a graph, where two empty ones take 3.1.
// ---------------------------------------------------------------------------
constexpr int VTP = 36;             // halves a d row of the V^T slices (32 + pad)
constexpr int RUN_MIN_F16 = 2;      // tiles a run, at least
constexpr int SEQ_COST_F16 = 2;     // a further piece's fixed cost in tiles (its q, its partial)

// A tile in flight: K[row 16 (w & 1) + (l & 15)][128 (w >> 1) + 32 (l / 16) + 8 s + 0..7]
// and V[row 16 (w & 1) + 4 (l & 3) + e][128 (w >> 1) + 8 (l / 4) + 0..7].
struct TileF16 {
    f16x8 k[4], v[4];
    int id0, id1;   // the pages of its halves
};

__global__ void __launch_bounds__(64 * D_WAVES)
paged_decode_f16_kernel(const f16* __restrict__ qg, int q_pitch, const char* __restrict__ kp,
                        const char* __restrict__ vp, const Pages pg, const int* __restrict__ pos0,
                        int B, int T, int n_q, int n_kv, const QHeads heads, const Cut cut, float sl2, const Sight sight,
                        const DecPart out) {
    __shared__ __attribute__((aligned(16))) f32x4 s_part[2][2][4][64];
    __shared__ __attribute__((aligned(16))) f16 s_vt[2][4][64][VTP];
    const int tid = threadIdx.x, lane = tid & 63;
    const int w = uni(tid >> 6);
    const int hh = lane >> 5, ql = lane & 31;
    const int G = heads.G, R = T * G;
    const int cap = pg.max_pages << pg.shift;
    Run run(pos0, B, T, n_kv, cut, sight, cap);
    if (!run.any) return;   // (the whole workgroup)
    const int h = run.h;
    // a lane's offsets from its wave's first row
    const uint32_t rs = 2 * PAGED_HD * n_kv, col = 2 * PAGED_HD * h + 256 * (w >> 1);
    const uint32_t ko = col + (lane & 15) * rs + 64 * (lane >> 4);
    uint32_t vo[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) vo[e] = col + (4 * (lane & 3) + e) * rs + 16 * (lane >> 2);

    int tick = 0;   // tiles done: the LDS buffers' turn
    for (;;) {
        const int b = uni(run.b);
        const DecSeq d = dec_seq(uni(pos0[b]), T, sight, cap);
        int j0, j1;
        run.piece(d, out, j0, j1);
        if (j1 > j0) {
            // this lane's query column: token tq, q head h G + gq
            const bool qvalid = ql < R;
            const int tq = qvalid ? heads.token(ql) : 0, gq = qvalid ? ql - tq * G : 0;
            int qlo, qhi;
            token_range(pos0[b], tq, sight.window, cap, qlo, qhi);
            // Q[column 16 nb + (l & 15)][128 (w >> 1) + 32 (l / 16) + 8 ks + 0..7]
            f16x8 qreg[8];
#pragma unroll
            for (int nb = 0; nb < 2; ++nb) {
                const int c = 16 * nb + (lane & 15);
                const bool ok = c < R;
                const int t = ok ? heads.token(c) : 0, g = ok ? c - t * G : 0;
                const f16* qrow = qg + (((size_t)b * T + t) * n_q + h * G + g) * q_pitch +
                                  128 * (w >> 1) + 32 * (lane >> 4);
#pragma unroll
                for (int ks = 0; ks < 4; ++ks)
                    qreg[4 * nb + ks] = ok ? *(const f16x8*)(qrow + 8 * ks) : (f16x8)(0);
            }
            auto ids = page_ids(pg, b, j0, j1 - 1, 0, [&](int j) { return d.row0(j); });

            f32x16 o0 = (f32x16)(0.f), o1 = (f32x16)(0.f);
            float m_run = -1e30f, l_run = 0.f;

            auto load = [&](TileF16& t, int j) {
                ids.at(j, t.id0, t.id1);
                // the wave's half; an absent page reads page 0 (masked, and v taken as 0)
                const int id = (w & 1) ? t.id1 : t.id0;
                const int in_page = (d.row0(j) + 16 * (w & 1)) & ((1 << pg.shift) - 1);
                const long long at = (((long long)max(id, 0) << pg.shift) + in_page) * rs;
                const gptr kb = uni_global(kp + at), vb = uni_global(vp + at);
#pragma unroll
                for (int s = 0; s < 4; ++s) t.k[s] = load_g<f16x8>(kb, ko + 16 * s);
#pragma unroll
                for (int e = 0; e < 4; ++e) t.v[e] = stream_g<f16x8>(vb, vo[e]);
            };
            auto body = [&](TileF16& t, int j) {
                const int buf = tick & 1;
                const int r0 = d.row0(j);
                const TileMask mask(r0, t.id0, t.id1, sight.sinks);
                const bool whole = mask.all(d.lo1, d.hi0);   // for every token (uniform)
                if (!whole) {
                    // rows that no token sees may hold anything: their v must not
                    // meet the product, where 0 x NaN is a NaN
                    const uint32_t any = mask.rows(d.lo0, d.hi1) >> (16 * (w & 1) + 4 * (lane & 3));
#pragma unroll
                    for (int i = 0; i < 4; ++i) t.v[i] = (any >> i) & 1 ? t.v[i] : (f16x8)(0);
                }
                f32x4 c0 = (f32x4)(0.f), c1 = (f32x4)(0.f);
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) {
                    c0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(t.k[ks], qreg[ks], c0, 0, 0, 0);
                    c1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(t.k[ks], qreg[4 + ks], c1, 0, 0, 0);
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
                        (f16x4){t.v[0][e], t.v[1][e], t.v[2][e], t.v[3][e]};
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
                    const uint32_t see = mask.rows(qlo, qhi) >> (4 * hh);
#pragma unroll
                    for (int rr = 0; rr < 16; ++rr)
                        sc[rr] = see & (1u << (8 * (rr >> 2) + (rr & 3))) ? sc[rr] : -INFINITY;
                }
                float mt = sc[0];
#pragma unroll
                for (int rr = 1; rr < 16; ++rr) mt = __builtin_elementwise_maximum(mt, sc[rr]);
                mt = pair32_max(mt) * sl2;
                const bool grow = mt > m_run + P_TOP;
                if (__any(grow)) {
                    const float m_new = grow ? mt - P_BELOW : m_run, corr = fast_exp2(m_run - m_new);
                    m_run = m_new;
                    l_run *= corr;
                    o0 *= corr;
                    o1 *= corr;
                }
                float psum = 0.f;
#pragma unroll
                for (int rr = 0; rr < 16; ++rr) {
                    sc[rr] = fast_exp2(fmaf(sc[rr], sl2, -m_run));
                    psum += sc[rr];
                }
                f16x8 pk[2];
#pragma unroll
                for (int ks = 0; ks < 2; ++ks)
                    pk[ks] = __builtin_convertvector(
                        (f32x8){sc[8 * ks], sc[8 * ks + 1], sc[8 * ks + 2], sc[8 * ks + 3],
                                sc[8 * ks + 4], sc[8 * ks + 5], sc[8 * ks + 6], sc[8 * ks + 7]}, f16x8);
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
            // Two tiles in registers: the next one's loads are issued ahead of this
            // one's math, and always (past the end the last tile's again): after a
            // conditional load the compiler's wait for this tile would drain them all.
            TileF16 t[2];
            load(t[0], j0);
            for (int j = j0; j < j1; j += 2) {
                load(t[1], min(j + 1, j1 - 1));
                body(t[0], j);
                load(t[0], min(j + 2, j1 - 1));
                if (j + 1 < j1) body(t[1], j + 1);
            }
            if (qvalid) {
                const size_t part = ((size_t)(b + run.run) * n_kv + h) * R + ql;
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
        if (!run.next(d)) return;
    }
}

// ---------------------------------------------------------------------------
// int8 pools. A wave takes tiles alone, over all 256 dims: no barrier and no exchange until
// the piece ends, where the O, maxima and sums of a head's waves are combined through LDS.
//   S^T (32 kv x 16 columns) = K Q^T      A operand: lane (i, g) row 16 rb + i, dims 32 ks
//                                         + 8 g .. + 7
//   softmax                               a lane holds column i's rows 4 g + e of both
//                                         halves; the maximum is exchanged only when
//                                         the reference moves (P_TOP)
//   O^T (256 dims) += V^T P^T             P as it lies: k slot (g, e) is row 4 g + e of
//                                         half e / 4; V^T by transposed LDS reads
// K and V come as whole rows, 16 bytes a lane, non-temporal, and are turned into operands
// through LDS: K as bytes, V as fp16. K of the next tile is requested once this one's is in
// LDS, V likewise, so one of them is always in flight.
//
// Bytes are exact in fp16. A 32-dim block is one k step, so its scale is applied to its fp32
// partial score and K is not rounded at all; V is f16(byte scale), and P goes in as two fp16
// terms: V's rounding is the only one of the products, and the error is that of fp16 pools,
// whose only one is P's. (With f16(byte scale) for K and V and P in one term it is 1.5 times
// as large.)
//
// What it reaches: 64 contexts of 100 - 32k 144 us (812 MB, 5.7 TB/s), 64 of 30 - 50k 865
// (6.3), 4 of 100k with 18 rows 169 (4.9). With 16 rows it is bound by the memory: without its
// products it takes as long, and what a workgroup's waves read at a time counts. K in operand
// order from memory (8 bytes a lane, 32 of a row an instruction), a head a workgroup and two
// workgroups of 4 waves a CU: 165; 8 waves with K through LDS 159; four heads a workgroup 145.
// With 17 - 32 rows O and Q leave a wave alone registers for one a SIMD, whose chain of
// products and conversions shows (4 of 100k 184 us, 151 without them; 4 of 8k 31), so a pair
// of waves shares a tile there: 169, 28.7. The columns shared out to two waves instead, each
// converting all of K and V: 229.
// ---------------------------------------------------------------------------
constexpr int K_PITCH = PAGED_HD + 16;       // bytes a K row in LDS (a b64 of 16 rows meets all banks)
constexpr int V_PITCH = 2 * PAGED_HD + 32;   // bytes a V row in LDS (the 32 spread rows over banks)
constexpr int O_PITCH = PAGED_HD + 4;        // floats a column of O in LDS
constexpr int PV_AHEAD = 2;                  // V^T fragments read ahead of their product
constexpr int SEQ_COST_Q8 = 6;               // a further piece's fixed cost in tiles (its first loads)

// A tile of K or V in flight: bytes [row 4 n + g][16 i .. + 15] and the scales of row l % 32,
// blocks 4 (l / 32) .. + 3.
struct Tile8 {
    u32x4 x[8];
    f16x4 sc;
};

// Where a call's pools and a lane's part of a row lie.
struct TileAt {
    const char *kp, *vp, *ks, *vs;   // values and scales
    uint32_t rs, vo, so;             // bytes a row; a lane's offsets
    bool upper;                      // its scales' half of the tile
    __device__ __forceinline__ TileAt(const char* kp_, const char* vp_, const Pages& pg, int n_kv, int h,
                                      int lane) {
        const int i = lane & 15, g = lane >> 4;
        kp = kp_, vp = vp_;
        rs = PAGED_HD * n_kv;
        const long long values = ((long long)pg.n_pages << pg.shift) * rs;
        ks = kp + values, vs = vp + values;
        vo = PAGED_HD * h + 16 * i + g * rs;
        so = 16 * h + 8 * (lane >> 5) + i * (rs / 16);
        upper = g & 1;
    }
    __device__ __forceinline__ f16x4 scales(const char* of, const long long (&at)[2]) const {
        const long long lo = at[0] * (rs / 16), hi = at[1] * (rs / 16);
        return *(const __attribute__((address_space(1))) f16x4*)((gptr)of + ((upper ? hi : lo) + so));
    }
    // at[half]: the pool row of the tile's 16-row halves
    __device__ __forceinline__ void load(Tile8& t, const char* rows, const char* sc,
                                         const long long (&at)[2]) const {
        t.sc = scales(sc, at);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const gptr b = uni_global(rows + at[half] * rs);
#pragma unroll
            for (int n = 0; n < 4; ++n) t.x[4 * half + n] = stream_g<u32x4>(b + 4 * n * rs, vo);
        }
        issued();
    }
    __device__ __forceinline__ void load_k(Tile8& t, const long long (&at)[2]) const { load(t, kp, ks, at); }
    __device__ __forceinline__ void load_v(Tile8& t, const long long (&at)[2]) const { load(t, vp, vs, at); }
    // the compiler would sink the loads to where they are used
    static __device__ __forceinline__ void issued() {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    }
};

// 8 bytes as the integers they are, exact in fp16 (q8_deq4 without the scale)
__device__ __forceinline__ f16x8 q8_ints(u32x2 b) {
    u32x4 r;
#pragma unroll
    for (int d = 0; d < 2; ++d) {
        const uint32_t u = b[d] ^ 0x80808080u;   // 1024 + (byte + 128), less 1152
        r[2 * d] = __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u);
        r[2 * d + 1] = __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u);
    }
    return __builtin_bit_cast(f16x8, r) - (f16x8)((f16)1152.f);
}
__device__ __forceinline__ f16x8 q8_values(uint32_t a, uint32_t b, f16 s) {
    const f16x4 lo = q8_deq4(a, (f16x2){s, s}), hi = q8_deq4(b, (f16x2){s, s});
    return (f16x8){lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}

// A V^T operand of 16 dims: lane (i, g) takes rows 4 g .. + 3 (and + 16) of dim i; it points
// at row 4 g + i / 4, dims 4 (i % 4) ..
__device__ __forceinline__ f16x8 v_frag(const char* at) {
    const f16x4 va =
        __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at));
    const f16x4 vb = __builtin_bit_cast(
        f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + 16 * V_PITCH)));
    return (f16x8){va[0], va[1], va[2], va[3], vb[0], vb[1], vb[2], vb[3]};
}

// Column c of the O's that the holders w0 .. w0 + step - 1 (of W) left in LDS, O_PITCH floats
// a column and `bytes` a holder, weighed against their common maximum, to partial `part`.
template <int W>
__device__ __forceinline__ void store_partial(const DecPart& out, size_t part, const float (*s_m)[16],
                                              const float (*s_l)[16], const char* s_o, int bytes, int w0,
                                              int step, int c, int lane) {
    float m = -1e30f, l = 0.f;
    f32x4 a = (f32x4)(0.f);
#pragma unroll
    for (int k = 0; k < W; ++k) m = fmaxf(m, s_m[w0 + min(k, step - 1)][c]);
#pragma unroll
    for (int k = 0; k < W; ++k) {   // (past the last holder: it once more, weighed 0)
        const int wk = w0 + min(k, step - 1);
        const float e = k < step ? fast_exp2(s_m[wk][c] - m) : 0.f;
        l = fmaf(e, s_l[wk][c], l);
        a += e * *(const f32x4*)(s_o + wk * bytes + (c * O_PITCH + 4 * lane) * 4);
    }
    *(f32x4*)(out.pacc + part * PAGED_HD + 4 * lane) = a;
    if (lane == 0) out.pm[part] = m, out.pd[part] = l;
}

// Up to 16 query rows.
constexpr int Q8_WAVES = 8;
__global__ void __launch_bounds__(64 * Q8_WAVES)
paged_decode_q8_kernel(const f16* __restrict__ qg, int q_pitch, const char* __restrict__ kp,
                       const char* __restrict__ vp, const Pages pg, const int* __restrict__ pos0, int B,
                       int T, int n_q, int n_kv, const QHeads heads, const Cut cut, float sl2, const Sight sight,
                       const DecPart out) {
    constexpr int W = Q8_WAVES;
    // K and V of a wave's tile while it walks, O of the waves when a piece ends
    constexpr int WAVE_B = std::max(DT * V_PITCH, 16 * O_PITCH * 4);
    __shared__ __attribute__((aligned(16))) char s_mem[W * WAVE_B];
    __shared__ float s_m[W][16], s_l[W][16];
    // the scales of a wave's tile, [K, V][block][row], V's rows in the order 8 (r % 4) + r / 4
    __shared__ __attribute__((aligned(16))) f16 s_sc[W][2][8][DT + 8];
    const int tid = threadIdx.x, lane = tid & 63;
    const int w = uni(tid >> 6);
    const int i = lane & 15, g = lane >> 4;
    const int G = heads.G, R = T * G;
    const int cap = pg.max_pages << pg.shift;
    char* const mine = s_mem + w * WAVE_B;
    Run run(pos0, B, T, n_kv, cut, sight, cap);
    if (!run.any) return;   // (the whole workgroup)
    // this wave's kv head; its tiles: the turn-th, and every step-th after it; w0 .. + step - 1
    // are the head's waves
    const int step_lg = 3 - run.heads_lg, step = 1 << step_lg;
    const int h = (run.h << run.heads_lg) + (w >> step_lg), turn = w & (step - 1), w0 = w - turn;
    const TileAt tiles(kp, vp, pg, n_kv, h, lane);

    for (;;) {
        const int b = uni(run.b);
        const DecSeq d = dec_seq(uni(pos0[b]), T, sight, cap);
        int j0, j1;
        run.piece(d, out, j0, j1);
        if (j1 > j0) {
            f32x4 o[16];
            float m_run = -1e30f, l_run = 0.f;   // l: of this lane's rows, summed when the piece ends
#pragma unroll
            for (int n = 0; n < 16; ++n) o[n] = (f32x4)(0.f);
            const int jw = j0 + turn;
            if (jw < j1) {
                auto ids = page_ids(pg, b, jw, j1 - 1, step_lg, [&](int j) { return d.row0(j); });
                // B operand: Q[column i][32 ks + 8 g + 0..7]; the column's rows in sight
                const bool ok = i < R;
                const int t = ok ? heads.token(i) : 0, gq = ok ? i - t * G : 0;
                const f16* qrow = qg + (((size_t)b * T + t) * n_q + h * G + gq) * q_pitch + 8 * g;
                f16x8 q[8];
#pragma unroll
                for (int s = 0; s < 8; ++s) q[s] = ok ? *(const f16x8*)(qrow + 32 * s) : (f16x8)(0);
                int lo, hi;
                token_range(pos0[b], t, sight.window, cap, lo, hi);
                struct Where {
                    int id0, id1, r0;
                    long long at[2];
                };
                auto where = [&](int j) {
                    Where x;
                    ids.at(j, x.id0, x.id1);
                    x.r0 = d.row0(j);
                    const int in_page = (1 << pg.shift) - 1;
                    // (an absent page: page 0 is read, its scores masked and its v taken as 0)
                    x.at[0] = ((long long)max(x.id0, 0) << pg.shift) + (x.r0 & in_page);
                    x.at[1] = ((long long)max(x.id1, 0) << pg.shift) + ((x.r0 + 16) & in_page);
                    return x;
                };
                Where x = where(jw);
                Tile8 kt, vt;
                tiles.load_k(kt, x.at);
                tiles.load_v(vt, x.at);
                const int j_last = jw + ((j1 - 1 - jw) & -step);
                for (int j = jw; j < j1; j += step) {
                    const Where xn = where(min(j + step, j_last));
                    const TileMask mask(x.r0, x.id0, x.id1, sight.sinks);
                    const bool whole = mask.all(d.lo1, d.hi0);   // for every token (uniform)
                    const int sc_row = lane & 31, sc_blk = 4 * (lane >> 5);
#pragma unroll
                    for (int e = 0; e < 4; ++e) s_sc[w][0][sc_blk + e][sc_row] = kt.sc[e];
#pragma unroll
                    for (int n = 0; n < 8; ++n) *(u32x4*)(mine + (4 * n + g) * K_PITCH + 16 * i) = kt.x[n];
                    tiles.load_k(kt, xn.at);
                    // scores: s[4 rb + e] of column i, row 16 rb + 4 g + e
                    float s[8];
                    const char* krow = mine + i * K_PITCH + 8 * g;
#pragma unroll
                    for (int rb = 0; rb < 2; ++rb) {
                        auto product = [&](int ks) {
                            return __builtin_amdgcn_mfma_f32_16x16x32_f16(
                                q8_ints(*(const u32x2*)(krow + 16 * rb * K_PITCH + 32 * ks)), q[ks],
                                (f32x4)(0.f), 0, 0, 0);
                        };
                        f32x4 c = (f32x4)(0.f), p = product(0);
#pragma unroll
                        for (int ks = 0; ks < 8; ++ks) {
                            // (the next block's product runs while this one's scale is applied)
                            const f32x4 pn = ks < 7 ? product(ks + 1) : p;
                            const f16x4 sc = *(const f16x4*)&s_sc[w][0][ks][16 * rb + 4 * g];
#pragma unroll
                            for (int e = 0; e < 4; ++e) c[e] = fmaf((float)sc[e], p[e], c[e]);
                            p = pn;
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[4 * rb + e] = c[e];
                    }
                    if (!whole) {
                        const uint32_t see = mask.rows(lo, hi) >> (4 * g);
#pragma unroll
                        for (int r = 0; r < 8; ++r)
                            s[r] = see & (1u << (16 * (r >> 2) + (r & 3))) ? s[r] : -INFINITY;
                    }
                    float mt = s[0];
#pragma unroll
                    for (int r = 1; r < 8; ++r) mt = __builtin_elementwise_maximum(mt, s[r]);
                    mt *= sl2;
                    if (__any(mt > m_run + P_TOP)) {
                        mt = fmaxf(mt, lane_xor(mt, 16));
                        mt = pair32_max(mt);
                        const float m_new = mt > m_run + P_TOP ? mt - P_BELOW : m_run;
                        const float corr = fast_exp2(m_run - m_new);
                        m_run = m_new;
                        l_run *= corr;
#pragma unroll
                        for (int n = 0; n < 16; ++n) o[n] *= corr;
                    }
                    f32x8 p;
#pragma unroll
                    for (int r = 0; r < 8; ++r) {
                        p[r] = fast_exp2(fmaf(s[r], sl2, -m_run));
                        l_run += p[r];
                    }
                    const f16x8 p_hi = __builtin_convertvector(p, f16x8);
                    const f16x8 p_lo =
                        __builtin_convertvector(p - __builtin_convertvector(p_hi, f32x8), f16x8);
                    // V to LDS as rows. Rows that no token sees may hold any scale: theirs is
                    // 0, since their v meets the product, where 0 x NaN is a NaN.
                    const bool on = whole || (mask.rows(d.lo0, d.hi1) >> sc_row & 1);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        s_sc[w][1][sc_blk + e][8 * (sc_row & 3) + (sc_row >> 2)] = on ? vt.sc[e] : (f16)0;
                    const f16x8 sc = *(const f16x8*)&s_sc[w][1][i >> 1][8 * g];
#pragma unroll
                    for (int n = 0; n < 8; ++n) {
                        char* row = mine + (4 * n + g) * V_PITCH + 32 * i;
                        *(f16x8*)row = q8_values(vt.x[n].x, vt.x[n].y, sc[n]);
                        *(f16x8*)(row + 16) = q8_values(vt.x[n].z, vt.x[n].w, sc[n]);
                    }
                    tiles.load_v(vt, xn.at);
                    // PV_AHEAD blocks of V^T are read ahead of their products
                    const char* vt0 = mine + (4 * g + (i >> 2)) * V_PITCH + 8 * (i & 3);
                    f16x8 fr[PV_AHEAD];
#pragma unroll
                    for (int n = 0; n < PV_AHEAD; ++n) fr[n] = v_frag(vt0 + 32 * n);
#pragma unroll
                    for (int n = 0; n < 16; ++n) {
                        const f16x8 a = fr[n % PV_AHEAD];
                        o[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, p_hi, o[n], 0, 0, 0);
                        o[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, p_lo, o[n], 0, 0, 0);
                        if (n + PV_AHEAD < 16) fr[n % PV_AHEAD] = v_frag(vt0 + 32 * (n + PV_AHEAD));
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    x = xn;
                }
            }
            // the piece's partial: the O of a head's waves weighed against their common maximum
            l_run += lane_xor(l_run, 16);
            l_run = pair32_sum(l_run);
            if (g == 0) s_m[w][i] = m_run, s_l[w][i] = l_run;
#pragma unroll
            for (int n = 0; n < 16; ++n) *(f32x4*)(mine + (i * O_PITCH + 16 * n + 4 * g) * 4) = o[n];
            __syncthreads();
            for (int c = turn; c < R; c += step)
                store_partial<W>(out, ((size_t)(b + run.run) * n_kv + h) * R + c, s_m, s_l, s_mem, WAVE_B, w0,
                                 step, c, lane);
            __syncthreads();
        }
        if (!run.next(d)) return;
    }
}

// 17 - 32 query rows: a pair of waves shares a tile, each converting 16 of its rows and
// holding 128 dims of O for all columns. Scores go through LDS, so both know every
// maximum; two barriers a round, in which each pair takes a tile. (Half of the pairs half a
// round later: 172; two workgroups of two pairs a CU 173, and 4 of 8k 31.7; the kv heads of
// a row in one workgroup, as below 17 rows: 175.)
constexpr int PAIRS = 4;
constexpr int S_PITCH = DT + 4;              // floats a column of scores in LDS

// half a tile of K or V in flight: bytes [row 4 n + g][16 i .. + 15] and the scales of row
// l % 16, blocks 4 (l / 16 % 2) .. + 3
struct HalfTile8 {
    u32x4 x[4];
    f16x4 sc;
};

__global__ void __launch_bounds__(128 * PAIRS)
paged_decode_q8_pairs_kernel(const f16* __restrict__ qg, int q_pitch, const char* __restrict__ kp,
                             const char* __restrict__ vp, const Pages pg, const int* __restrict__ pos0,
                             int B, int T, int n_q, int n_kv, const QHeads heads, const Cut cut, float sl2, const Sight sight,
                             const DecPart out) {
    // a pair's V while it walks, its O when a piece ends
    constexpr int PAIR_B = std::max(DT * V_PITCH, 16 * O_PITCH * 4);
    __shared__ __attribute__((aligned(16))) char s_v[PAIRS][PAIR_B];
    __shared__ __attribute__((aligned(16))) char s_k[2 * PAIRS][DT / 2 * K_PITCH];
    __shared__ __attribute__((aligned(16))) float s_s[PAIRS][32 * S_PITCH];
    __shared__ float s_m[PAIRS][16], s_l[PAIRS][16];
    // the scales of a wave's half, [K, V][block][row], V's rows in the order 4 (r % 4) + r / 4
    __shared__ __attribute__((aligned(16))) f16 s_sc[2 * PAIRS][2][8][DT / 2 + 8];
    const int tid = threadIdx.x, lane = tid & 63;
    const int w = uni(tid >> 6), pair = w >> 1, sub = w & 1;
    const int i = lane & 15, g = lane >> 4;
    const int G = heads.G, R = T * G;
    const int cap = pg.max_pages << pg.shift;
    Run run(pos0, B, T, n_kv, cut, sight, cap);
    if (!run.any) return;   // (the whole workgroup)
    const int h = run.h;
    const uint32_t rs = PAGED_HD * n_kv;   // bytes a row
    const long long values = ((long long)pg.n_pages << pg.shift) * rs;
    const uint32_t xo = PAGED_HD * h + 16 * i + g * rs;
    const uint32_t so = 16 * h + 8 * (g & 1) + i * (rs / 16);
    const int sc_row = i, sc_blk = 4 * (g & 1);
    auto load = [&](HalfTile8& t, const char* pool, long long at) {
        t.sc = load_g<f16x4>(uni_global(pool + values + at * (rs / 16)), so);
        const gptr b = uni_global(pool + at * rs);
#pragma unroll
        for (int n = 0; n < 4; ++n) t.x[n] = stream_g<u32x4>(b + 4 * n * rs, xo);
        asm volatile("" ::: "memory");   // (the compiler would sink the loads to where they are used)
        __builtin_amdgcn_sched_barrier(0);
    };
    // LDS written; the next tile's loads stay in flight across the barrier
    auto barrier = [] { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };

    for (;;) {
        const int b = uni(run.b);
        const DecSeq d = dec_seq(uni(pos0[b]), T, sight, cap);
        int j0, j1;
        run.piece(d, out, j0, j1);
        if (j1 > j0) {
            f32x4 o[2][8];   // O^T of dims 128 sub + 16 n + 4 g .. + 3, columns 16 nb + i
            float m_run[2], l_run[2];   // l: of this lane's rows, summed when the piece ends
            // B operand: Q[column 16 nb + i][32 ks + 8 g + 0..7]; the column's rows in sight
            f16x8 q[2][8];
            int lo[2], hi[2];
#pragma unroll
            for (int nb = 0; nb < 2; ++nb) {
                m_run[nb] = -1e30f, l_run[nb] = 0.f;
#pragma unroll
                for (int n = 0; n < 8; ++n) o[nb][n] = (f32x4)(0.f);
                const int c = 16 * nb + i;
                const bool ok = c < R;
                const int t = ok ? heads.token(c) : 0, gq = ok ? c - t * G : 0;
                const f16* row = qg + (((size_t)b * T + t) * n_q + h * G + gq) * q_pitch + 8 * g;
#pragma unroll
                for (int s = 0; s < 8; ++s) q[nb][s] = ok ? *(const f16x8*)(row + 32 * s) : (f16x8)(0);
                token_range(pos0[b], t, sight.window, cap, lo[nb], hi[nb]);
            }
            auto ids = page_ids(pg, b, min(j0 + pair, j1 - 1), j1 - 1, 2,
                                [&](int j) { return d.row0(j); });
            struct Where {
                int id0, id1, r0;
                long long at;   // the pool row of this wave's half
            };
            auto where = [&](int j) {
                Where x;
                ids.at(j, x.id0, x.id1);
                x.r0 = d.row0(j);
                // (an absent page: page 0 is read, its scores masked and its v taken as 0)
                x.at = ((long long)max(sub ? x.id1 : x.id0, 0) << pg.shift) +
                       ((x.r0 + 16 * sub) & ((1 << pg.shift) - 1));
                return x;
            };
            // a pair without a tile in the last round (or in any) has its last tile's loads again
            const int jw = min(j0 + pair, j1 - 1), j_last = jw + ((j1 - 1 - jw) & -PAIRS);
            Where x = where(jw);
            HalfTile8 kt, vt;
            load(kt, kp, x.at);
            load(vt, vp, x.at);
            for (int j = j0; j < j1; j += PAIRS) {   // (the workgroup's rounds: uniform)
                const bool mine = j + pair < j1;
                const Where xn = where(min(j + pair + PAIRS, j_last));
                const TileMask mask(x.r0, x.id0, x.id1, sight.sinks);
                const bool whole = mask.all(d.lo1, d.hi0);   // for every token (uniform)
                if (mine) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) s_sc[w][0][sc_blk + e][sc_row] = kt.sc[e];
#pragma unroll
                    for (int n = 0; n < 4; ++n) *(u32x4*)(s_k[w] + (4 * n + g) * K_PITCH + 16 * i) = kt.x[n];
                }
                load(kt, kp, xn.at);
                if (mine) {
                    // scores of column 16 nb + i, rows 16 sub + 4 g .. + 3
                    const char* krow = s_k[w] + i * K_PITCH + 8 * g;
                    f32x4 c[2], p[2], pn[2];
                    auto product = [&](int ks, f32x4 (&r)[2]) {
                        const f16x8 a = q8_ints(*(const u32x2*)(krow + 32 * ks));
#pragma unroll
                        for (int nb = 0; nb < 2; ++nb)
                            r[nb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, q[nb][ks], (f32x4)(0.f), 0, 0, 0);
                    };
                    product(0, p);
                    c[0] = c[1] = (f32x4)(0.f);
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks) {
                        // (the next block's product runs while this one's scale is applied)
                        if (ks < 7) product(ks + 1, pn);
                        const f16x4 sc = *(const f16x4*)&s_sc[w][0][ks][4 * g];
#pragma unroll
                        for (int nb = 0; nb < 2; ++nb) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) c[nb][e] = fmaf((float)sc[e], p[nb][e], c[nb][e]);
                            p[nb] = pn[nb];
                        }
                    }
#pragma unroll
                    for (int nb = 0; nb < 2; ++nb)
                        *(f32x4*)&s_s[pair][(16 * nb + i) * S_PITCH + 16 * sub + 4 * g] = c[nb];
                    // V to LDS as rows. Rows that no token sees may hold any scale: theirs is
                    // 0, since their v meets the product, where 0 x NaN is a NaN.
                    const bool on = whole || (mask.rows(d.lo0, d.hi1) >> (16 * sub + sc_row) & 1);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        s_sc[w][1][sc_blk + e][4 * (sc_row & 3) + (sc_row >> 2)] = on ? vt.sc[e] : (f16)0;
                    const f16x4 sc = *(const f16x4*)&s_sc[w][1][i >> 1][4 * g];
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        char* row = s_v[pair] + (16 * sub + 4 * n + g) * V_PITCH + 32 * i;
                        *(f16x8*)row = q8_values(vt.x[n].x, vt.x[n].y, sc[n]);
                        *(f16x8*)(row + 16) = q8_values(vt.x[n].z, vt.x[n].w, sc[n]);
                    }
                }
                load(vt, vp, xn.at);
                barrier();
                if (mine) {
                    f16x8 p_hi[2], p_lo[2];
#pragma unroll
                    for (int nb = 0; nb < 2; ++nb) {
                        const float* sr = &s_s[pair][(16 * nb + i) * S_PITCH + 4 * g];
                        const f32x4 s0 = *(const f32x4*)sr, s1 = *(const f32x4*)(sr + 16);
                        f32x8 s = {s0[0], s0[1], s0[2], s0[3], s1[0], s1[1], s1[2], s1[3]};
                        if (!whole) {
                            const uint32_t see = mask.rows(lo[nb], hi[nb]) >> (4 * g);
#pragma unroll
                            for (int r = 0; r < 8; ++r)
                                s[r] = see & (1u << (16 * (r >> 2) + (r & 3))) ? s[r] : -INFINITY;
                        }
                        float mt = s[0];
#pragma unroll
                        for (int r = 1; r < 8; ++r) mt = __builtin_elementwise_maximum(mt, s[r]);
                        mt *= sl2;
                        if (__any(mt > m_run[nb] + P_TOP)) {   // (as above; both waves alike)
                            mt = fmaxf(mt, lane_xor(mt, 16));
                            mt = pair32_max(mt);
                            const float m_new = mt > m_run[nb] + P_TOP ? mt - P_BELOW : m_run[nb];
                            const float corr = fast_exp2(m_run[nb] - m_new);
                            m_run[nb] = m_new;
                            l_run[nb] *= corr;
#pragma unroll
                            for (int n = 0; n < 8; ++n) o[nb][n] *= corr;
                        }
                        f32x8 p;
#pragma unroll
                        for (int r = 0; r < 8; ++r) {
                            p[r] = fast_exp2(fmaf(s[r], sl2, -m_run[nb]));
                            l_run[nb] += p[r];
                        }
                        p_hi[nb] = __builtin_convertvector(p, f16x8);
                        p_lo[nb] =
                            __builtin_convertvector(p - __builtin_convertvector(p_hi[nb], f32x8), f16x8);
                    }
                    const char* vt0 = s_v[pair] + (4 * g + (i >> 2)) * V_PITCH + 256 * sub + 8 * (i & 3);
                    f16x8 fr[PV_AHEAD];
#pragma unroll
                    for (int n = 0; n < PV_AHEAD; ++n) fr[n] = v_frag(vt0 + 32 * n);
#pragma unroll
                    for (int n = 0; n < 8; ++n) {
                        const f16x8 a = fr[n % PV_AHEAD];
#pragma unroll
                        for (int nb = 0; nb < 2; ++nb) {
                            o[nb][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, p_hi[nb], o[nb][n], 0, 0, 0);
                            o[nb][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, p_lo[nb], o[nb][n], 0, 0, 0);
                        }
                        if (n + PV_AHEAD < 8) fr[n % PV_AHEAD] = v_frag(vt0 + 32 * (n + PV_AHEAD));
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
                barrier();   // scores and V may be overwritten
                x = xn;
            }
            // the piece's partial: the O of the pairs weighed against their common
            // maximum, 16 columns at a time
#pragma unroll
            for (int nb = 0; nb < 2; ++nb) {
                float l = l_run[nb];
                l += lane_xor(l, 16);
                l = pair32_sum(l);
                if (g == 0 && sub == 0) s_m[pair][i] = m_run[nb], s_l[pair][i] = l;
#pragma unroll
                for (int n = 0; n < 8; ++n)
                    *(f32x4*)(s_v[pair] + (i * O_PITCH + 128 * sub + 16 * n + 4 * g) * 4) = o[nb][n];
                __syncthreads();
                for (int c = 2 * pair + sub; c < min(R - 16 * nb, 16); c += 2 * PAIRS)
                    store_partial<PAIRS>(out, ((size_t)(b + run.run) * n_kv + h) * R + 16 * nb + c, s_m, s_l,
                                         s_v[0], PAIR_B, 0, PAIRS, c, lane);
                __syncthreads();
            }
        }
        if (!run.next(d)) return;
    }
}

// z of every (token, q head) from its sequence's partials: z = f16_sat(sum_s e_s
// acc_s / sum_s e_s d_s sigmoid(gate)), e_s = 2^(m_s - M), rounded once. J waves a
// pair (4: few sequences, many partials each; 1: many sequences), lane l holding
// dims 4 l .. + 3, each wave's partials s = j, j + J, ... in batches whose loads are
// all issued before any is used, the J sums added in order through LDS.
// (a small call runs its code once, and fetching it shows: with batches of 2, 4, 8, 16 one
// context of 500 10.0, 10.0, 10.65, 11.1 us, one of 4k 14.0, 13.9, 15.2, 15.1)
constexpr int MG_BATCH = 4;
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
    const float inv = 1.f / den;
    f16x4 out;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const float v = num[c] * inv;
        // (no row seen: 0, whatever the gate and the rows that other tokens see hold)
        out[c] = den == 0.f ? (f16)0.f : f16_sat(gate != nullptr ? v * fast_sigmoid((float)gv[c]) : v);
    }
    *(f16x4*)(z + (size_t)rh * z_pitch + 4 * lane) = out;
}

// A workgroup a CU.
Cut dec_cut(int n_kv, bool q8, int rows) {
    Cut c = {std::max(1, cu_count() / n_kv), RUN_MIN_F16, SEQ_COST_F16, 0};
    if (q8) {
        c.run_min = rows > 16 ? PAIRS : Q8_WAVES, c.seq_cost = SEQ_COST_Q8;
        if (rows <= 16) c.heads_lg = std::min(2, __builtin_ctz((unsigned)n_kv));
    }
    return c;
}
int most_runs(const Cut& c) { return c.runs << c.heads_lg; }

size_t dec_part(int B, int T, int n_q, int n_kv, int runs, char* work, DecPart& p) {
    const size_t rows = (size_t)(B + runs) * T * n_q;
    const size_t m = up16((size_t)B * sizeof(int2)), f = up16(rows * 4);
    p = {(int2*)work, (float*)(work + m), (float*)(work + m + f), (float*)(work + m + 2 * f)};
    return m + 2 * f + rows * PAGED_HD * 4;
}

}  // namespace

extern "C" {

size_t fl_attn_decode_paged_work_bytes(int B, int T, int n_q_heads, int n_kv_heads, int head_dim) {
    if (B < 1 || B > FL_PAGED_MAX_SEQS || n_kv_heads < 1 || n_q_heads < 1 || T < 1 ||
        n_q_heads % n_kv_heads || (long long)T * (n_q_heads / n_kv_heads) > 32 || head_dim != PAGED_HD)
        return 0;
    DecPart p;
    const Cut cut = dec_cut(n_kv_heads, true, T * (n_q_heads / n_kv_heads));   // (fp16: as many or fewer)
    return dec_part(B, T, n_q_heads, n_kv_heads, most_runs(cut), nullptr, p);
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
    FL_REQUIRE((((long long)max_pages << pg.shift) / DT + 8) * B < INT_MAX,
               "B * max_pages * page_size < 2^36");
    DecPart part;
    const int rows = T * (n_q_heads / n_kv_heads);
    const Cut cut = dec_cut(n_kv_heads, q8, rows);
    const int runs = most_runs(cut);
    if (dec_part(B, T, n_q_heads, n_kv_heads, runs, (char*)work, part) > work_bytes || !work) {
        fl::set_error("work: smaller than fl_attn_decode_paged_work_bytes");
        return FL_ESCRATCH;
    }
    FL_REQUIRE(aligned16(work), "16-byte aligned work");
    const dim3 grid(cut.runs * n_kv_heads);
    const int G = n_q_heads / n_kv_heads;
    const QHeads heads = {G, 65536 / G + 1};   // exact for rows up to 32
    const float sl2 = scale * FL_LOG2E;
    const Sight sight = {window, sinks};
    if (!q8)
        hipLaunchKernelGGL(paged_decode_f16_kernel, grid, dim3(64 * D_WAVES), 0, (hipStream_t)stream,
                           (const f16*)qg, q_pitch, (const char*)kpool, (const char*)vpool, pg, pos0, B, T,
                           n_q_heads, n_kv_heads, heads, cut, sl2, sight, part);
    else
        hipLaunchKernelGGL(rows > 16 ? paged_decode_q8_pairs_kernel : paged_decode_q8_kernel, grid,
                           dim3(64 * Q8_WAVES), 0, (hipStream_t)stream,
                           (const f16*)qg, q_pitch, (const char*)kpool, (const char*)vpool, pg, pos0, B, T,
                           n_q_heads, n_kv_heads, heads, cut, sl2, sight, part);
    rc = fl::check_launch("attn_decode_paged");
    if (rc) return rc;
    const int pairs = B * T * n_q_heads;
    const f16* gate = gated ? (const f16*)qg + PAGED_HD : nullptr;
    // Four waves a pair where a sequence has 4 partials or more, were its stream as long as it
    // may be (over int8 a long one has 2^heads_lg times a short one's runs, and the lengths are
    // on the device), one where it has fewer. One wave / four, us: fp16 one context of 500 11.3 /
    // 9.6, 4 of 8k 31.5 / 28.5, 16 of 2k 28.3 / 27.9, 20 of 60 9.6 / 10.1, 96 of 60 18.1 / 19.6;
    // int8 4 of 8k 27.0 / 23.9, 24 of 8k 83.7 / 82.5, 40 of 100 - 32k 105.0 / 100.5 (the longest
    // has dozens), 64 of them 147.0 / 145.3; the price, short int8 streams that count as long:
    // 40 of 2k 46.1 / 47.1, 64 of 2k 64.3 / 65.1, 64 of 60 14.4 / 15.5.
    const bool wide = runs >= 4 * B;
    auto merge = wide ? paged_merge_kernel<4> : paged_merge_kernel<1>;
    hipLaunchKernelGGL(merge, dim3(wide ? pairs : (pairs + 3) / 4), dim3(256), 0, (hipStream_t)stream,
                       part, (f16*)z, z_pitch, gate, q_pitch, T, n_q_heads, n_kv_heads, pairs);
    return fl::check_launch("attn_decode_paged merge");
}

}  // extern "C"
