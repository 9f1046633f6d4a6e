// Causal attention of chunks of new tokens over the paged KV cache (attn_paged.hpp says
// what is computed), several sequences a call.
//
// A row tile is 256 (token, q head) rows of one kv head of one sequence, token-major, 64
// a wave; a wave's tile of 32 cache rows is attn_r64.hpp's: S^T = K Q^T with Q in
// registers, the softmax with a query column a lane pair, O^T += V^T P^T in AGPRs, K and V
// copied HBM -> LDS three tiles ahead. What is this file's own:
//   * a tile's rows come from the pages of its two 16-row halves: a wave copies 8 rows of
//     one half, so its copies have one scalar base. Rows that no query of the row tile
//     sees (past its last token, before its window, on absent pages) are copied from a row
//     of zeros: p is 0 there, and 0 times whatever a page holds must stay 0;
//   * a row tile walks the tiles of the first `sinks` rows and those from its window on;
//   * the masks are bits, formed only for tiles that some query does not see whole;
//   * workgroups are persistent, one a CU, over a host-made plan for the whole batch:
//     either a list of whole row tiles each (CUT false), or equal runs of all row tiles'
//     walks laid end to end, cut wherever the cuts fall (CUT): an uncut row tile of a run
//     goes to z, a cut one leaves partials that paged_piece_merge_kernel combines.
// Over int8 pools the visible rows are first copied to fp16 in the work buffer, K as the bytes
// and V as f16(byte scale), absent and unwritten rows as zeros, and the same kernel walks that
// copy (DENSE): K's block scales go onto the partial scores in fp32 (put_steps) and P goes in as
// two fp16 terms, so that V's rounding is the only one of the products and z is off by 1.4 times
// its own rounding, as over fp16 pools and in the int8 decode. (With f16(byte scale) for K as
// well and P in one term it is 1.8 times, in two thirds of the time; K exact alone 1.7.)
//
// Bound by a wave's own chain, one wave a SIMD: 8192 fresh tokens at 24 q and 4 kv heads 842 us,
// 1.0 PFLOP/s of the 1.3 that a large fp16 product reaches, the matrix cores busy 40 % of the
// cycles; the softmax between the two products of a tile and a row tile's start and end
// (ITEM_COST) are the difference. Four chunks of 1024 with a window 450 - 470 us (0.8: short
// walks). Over int8 pools a tile has half again the products and 256 multiplications for the
// steps, 3.2 us where it has 2.0: 8192 fresh tokens 1300 us, six of 1 - 1024 tokens at 0 - 60k
// 1.88 ms (0.55), 117 us of it the copy (6.3 TB/s).
// The wave's registers are nearly all taken (233, over int8 pools 247 of 256, beside O's). A
// spill is not only slow but wrong here: the O accumulators are written by inline-asm MFMAs,
// whose hazards the compiler does not see when it stores them. Its resource report has to say
// 0 spilled VGPRs.
#include "attn_paged.hpp"
#include "attn_r64.hpp"

#include <algorithm>
#include <mutex>
#include <new>
#include <queue>
#include <string.h>
#include <type_traits>
#include <vector>

using fl::R64_BQ;

namespace {

constexpr int MAX_SEQS = FL_PAGED_MAX_SEQS_PREFILL;
constexpr int THREADS = 256;
constexpr int OUT_ROWS = 8;    // rows whose gates are in flight when a row tile ends (4, 8: 852,
                               // 842 us for 8192 fresh tokens; 16 spills)

// Packed chunks: sequence b's tokens are start[b] .. start[b + 1] - 1, the first at
// position pos0[b], its row tiles tile0[b] .. tile0[b + 1] - 1; dense[b]: its first row in
// the fp16 copy (DENSE).
struct Chunks {
    int n;
    int start[MAX_SEQS + 1];
    int tile0[MAX_SEQS + 1];
    int pos0[MAX_SEQS];
    int dense[MAX_SEQS];
};

// What a row tile walks: the rows [lo, hi) and [0, min(sinks, hi)) of its sequence as
// tiles, the first s ones, then those from a on, n in all.
struct Walk {
    int lo, hi, s, a, n;
    __host__ __device__ __forceinline__ int row0(int j) const {
        return R64_BK * (j < s ? j : a + j - s);
    }
};
__host__ __device__ __forceinline__ Walk make_walk(int p_first, int p_last, const Sight& sight) {
    Walk w;
    w.hi = p_last + 1;
    w.lo = sight.window > 0 && p_first >= sight.window ? p_first - sight.window + 1 : 0;
    w.a = w.lo / R64_BK;
    const int sk = sight.sinks < w.hi ? sight.sinks : w.hi;
    const int st = (int)(((unsigned)sk + R64_BK - 1) / R64_BK);
    w.s = st < w.a ? st : w.a;
    w.n = w.s + (int)(((unsigned)w.hi + R64_BK - 1) / R64_BK) - w.a;
    return w;
}

// The plan of a call, alike for every kv head. CUT: run r goes from row tile tile[r], tile
// j[r] of its walk, to those of r + 1; its first partial's slot is slot[r]. Else run r has
// the row tiles list[at[r]] .. list[at[r + 1] - 1].
constexpr int MAX_RUNS = 256;
constexpr int LIST_MAX = 1024;
struct Plan {
    int runs;
    union {
        struct {
            uint32_t j[MAX_RUNS + 1];
            uint16_t tile[MAX_RUNS + 1];
            uint16_t slot[MAX_RUNS];
        } cut;
        struct {
            uint16_t at[MAX_RUNS + 1];
            uint16_t list[LIST_MAX];
        } whole;
    };
};

// The partials: O unnormalised [slot][256 rows][256], its maximum (log2 units) and sum
// [slot][256]; kv head h's slots start at h n.
struct Parts {
    float* pacc;
    float* pm;
    float* pd;
    int n;
};

__device__ const u32x4 zero_row[ROW_B / 16] = {};

// Over int8 pools the copy's K are the bytes, exact in fp16, and a score is formed block by block
// in place, S <- (S + product of block b) t_b with t_b = s_b / s_(b + 1) for b < 7 and t_7 = s_7:
// sum_b s_b q.k_b, K not rounded, in no more registers than S. t is in LDS behind the stages, for
// this tile and the next, [tile & 1][block][row]; ahead of it the scales as they come, a stage's
// by the waves that copy them: [wave][pair of blocks][row of its 8], a dword two blocks' scales
// of a row (the other half of a wave's part takes what its lanes 32 - 63 copy, the same again).
constexpr int SCALE_W = 256;                 // bytes a wave
constexpr int SCALE_STAGE = 4 * SCALE_W;
constexpr int STEP_AT = R64_LDS + R64_NST * SCALE_STAGE;
constexpr int STEP_B = 8 * R64_BK * 4;
constexpr int DENSE_LDS = STEP_AT + 2 * STEP_B;
__device__ __forceinline__ void copy4_v(const char* vptr, uint32_t lds) {   // copy16_v, 4 bytes a lane
    asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(vptr), "{m0}"(lds));
}
// t of this wave's 8 rows of a tile from its scales, a (block, row) a lane. (A scale of 0, whose
// block's copy is 0: any other does.)
__device__ __forceinline__ void put_steps(char* smem, int stage, int tile, int w, int lane) {
    asm volatile("" : "+v"(lane));   // (its addresses are not worth registers across the tile loop)
    const int blk = lane >> 3, row = lane & 7;
    const char* sc = smem + R64_LDS + stage * SCALE_STAGE + w * SCALE_W;
    auto scale = [&](int b) {
        const float x = (float)*(const f16*)(sc + 32 * (b >> 1) + 4 * row + 2 * (b & 1));
        return x == 0.f ? 0x1p-24f : x;
    };
    const float own = scale(blk), next = scale(min(blk + 1, 7));
    *(float*)(smem + STEP_AT + (tile & 1) * STEP_B + 4 * (R64_BK * blk + 8 * w + row)) =
        blk < 7 ? own * __builtin_amdgcn_rcpf(next) : own;
}

// Softmax of one 32-column block of a tile (a query column a lane pair, 16 of its 32
// scores a lane: score r is row 8 (r / 4) + 4 hh + r % 4), `see` the column's visible rows
// from 4 hh on; the lazy rescale of this block's O^T; P in fp16 as the PV operand, TWO: and
// what that leaves of it in another fp16 (pl).
template <bool TWO>
__device__ __forceinline__ void softmax_block(f32x16& s, bool whole, uint32_t see, float sl2,
                                              float& m_run, float& l_run, f32x16 (&o)[8],
                                              f16x8 (&pk)[2], f16x8 (&pl)[2]) {
    if (!whole) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
            s[r] = see & (1u << (8 * (r >> 2) + (r & 3))) ? s[r] : -INFINITY;
    }
    float mt = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) mt = __builtin_elementwise_maximum(mt, s[r]);
    mt = pair32_max(mt) * sl2;
    if (__any(mt > m_run + P_TOP)) {   // always on a wave's first tile, rarely after
        const float m_new = fmaxf(m_run, mt - P_BELOW);
        const float corr = fast_exp2(m_run - m_new);
        m_run = m_new;
        l_run *= corr;
        acc_scale(o, corr);
    }
    float psum = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        s[r] = fast_exp2(fmaf(s[r], sl2, -m_run));
        psum += s[r];
    }
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
        const f32x8 p = {s[8 * ks],     s[8 * ks + 1], s[8 * ks + 2], s[8 * ks + 3],
                         s[8 * ks + 4], s[8 * ks + 5], s[8 * ks + 6], s[8 * ks + 7]};
        pk[ks] = __builtin_convertvector(p, f16x8);
        if (TWO) pl[ks] = __builtin_convertvector(p - __builtin_convertvector(pk[ks], f32x8), f16x8);
    }
    l_run += pair32_sum(psum);
}

// Copy 8 rows of a tile's K and V (this wave's) into its stage: two rows an instruction,
// loff[n] this lane's source offset, swizzled (attn_prefill's layout).
__device__ __forceinline__ void copy_rows(uint32_t d0, const char* kr, const char* vr,
                                          const uint32_t (&loff)[4]) {
    copy16_at<0 * ROW_B>(kr, loff[0], d0);
    copy16_at<2 * ROW_B>(kr, loff[1], d0);
    copy16_at<4 * ROW_B>(kr, loff[2], d0);
    copy16_at<6 * ROW_B>(kr, loff[3], d0);
    copy16_at<R64_TILE + 0 * ROW_B>(vr, loff[0], d0);
    copy16_at<R64_TILE + 2 * ROW_B>(vr, loff[1], d0);
    copy16_at<R64_TILE + 4 * ROW_B>(vr, loff[2], d0);
    copy16_at<R64_TILE + 6 * ROW_B>(vr, loff[3], d0);
}

// DENSE: kc and vc are the copy, [row][n_kv][256], ksc the pool's scales of K; else the pools.
template <bool DENSE, bool CUT>
__global__ void __launch_bounds__(THREADS)
paged_prefill_kernel(const f16* __restrict__ q, int q_pitch, const char* __restrict__ kc,
                     const char* __restrict__ vc, const char* __restrict__ ksc, const Pages pg,
                     const Chunks ch, f16* __restrict__ z, int z_pitch, int gated, int n_q_heads,
                     int n_kv, float sl2,
                     const Sight sight, const Plan plan, Parts parts) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    // Workgroups go to the 8 XCDs round-robin, each with an L2 of its own: where the kv
    // heads divide 8, XCDs 8 / n_kv h .. take all of kv head h.
    int h, run;
    {
        const int id = blockIdx.x;
        if (8 % n_kv == 0 && gridDim.x % 8 == 0) {
            const int xcd = id & 7, per = 8 / n_kv;
            h = xcd / per;
            run = (id >> 3) * per + xcd % per;
        } else {
            h = id % n_kv;
            run = id / n_kv;
        }
    }
    if (run >= plan.runs) return;
    const int tid = threadIdx.x, lane = tid & 63;
    const int w = uni(tid >> 6);
    const int ql = lane & 31, hh = lane >> 5;
    const int G = n_q_heads / n_kv;
    const uint32_t rsb = (uint32_t)n_kv * ROW_B;
    const char* kb = uniform_ptr(kc + (size_t)h * ROW_B);
    const char* vb = uniform_ptr(vc + (size_t)h * ROW_B);
    uint32_t loff[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        const int r = 2 * n + (lane >> 5);   // row from 8 w
        loff[n] = r * rsb + 16 * ((lane & 31) ^ sw(8 * w + r));
    }
    const uint32_t lds_base = (uint32_t)(uintptr_t)((__attribute__((address_space(3))) char*)smem);
    // K operand of k-step ks: tile row ql, chunk 16 hh + ks, at 16 hh + (ks ^ sw(ql)); DENSE:
    // chunk 2 ks + hh, at (2 ks) ^ hh ^ sw(ql), so that two k-steps are a 32-dim block
    const uint32_t koff = ql * ROW_B + (DENSE ? 16 * (hh ^ sw(ql)) : 256 * hh + 16 * sw(ql));
    const int tr_r = (lane & 15) >> 2;
    const int tr_d = 16 * ((lane & 31) >> 4) + 4 * (lane & 3);
    uint32_t troff[8];
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2)
            troff[2 * u + s2] = (4 * hh + tr_r + 8 * s2) * ROW_B + 64 * (u ^ tr_r) +
                                16 * ((tr_d >> 3) ^ (hh + 2 * s2)) + 2 * (tr_d & 7);

    const int item0 = uni(CUT ? plan.cut.tile[run] : plan.whole.at[run]);
    const int item1 = uni(CUT ? plan.cut.tile[run + 1] : plan.whole.at[run + 1]);
    const int j_first = CUT ? uni(plan.cut.j[run]) : 0, j_last = CUT ? uni(plan.cut.j[run + 1]) : 0;
    int slot = CUT ? uni(plan.cut.slot[run]) : 0;
    const int n_items = item1 - item0 + (j_last > 0 ? 1 : 0);
    int seq = 0;
    for (int it = 0; it < n_items; ++it) {
        const int tile = CUT ? item0 + it : uni(plan.whole.list[item0 + it]);
        if (!CUT) seq = 0;
        while (tile >= ch.tile0[seq + 1]) ++seq;   // (scalar)
        if (it > 0) tile_done();   // every wave is done with the previous row tile's stages
        const int pos0 = ch.pos0[seq], start = ch.start[seq];
        const int RT = (ch.start[seq + 1] - start) * G;
        const int R0 = (tile - ch.tile0[seq]) * R64_BQ;
        // this lane's two query rows (columns of the two MFMA blocks)
        int t[2], g[2], qpos[2];
        bool rvalid[2];
#pragma unroll
        for (int nb = 0; nb < 2; ++nb) {
            const int row = R0 + 64 * w + 32 * nb + ql;
            rvalid[nb] = row < RT;
            t[nb] = rvalid[nb] ? row / G : 0;
            g[nb] = rvalid[nb] ? row - t[nb] * G : 0;
            qpos[nb] = rvalid[nb] ? pos0 + t[nb] : -1;
        }
        const int wfirst = R0 + 64 * w, wlast = min(wfirst + 63, RT - 1);
        const int wqmax = uni(wlast >= wfirst ? pos0 + wlast / G : -1);
        const int wqmin = uni(pos0 + wfirst / G);
        const Walk walk = make_walk(uni(pos0 + R0 / G), uni(pos0 + min(R0 + R64_BQ - 1, RT - 1) / G),
                                    sight);
        const int j_lo = CUT && it == 0 ? j_first : 0;
        const int j_hi = CUT && it == n_items - 1 && j_last > 0 ? j_last : walk.n;
        const int n_tiles = j_hi - j_lo;
        if (CUT && n_tiles <= 0) continue;   // (uniform)

        // in the copy a sequence's rows before its first window's are left out
        int dense_cut = 0, dense_skip = 0;
        if constexpr (DENSE) {
            const Walk all = make_walk(pos0, pos0, sight);
            dense_cut = R64_BK * all.s;
            dense_skip = R64_BK * (all.a - all.s);
        }
        auto ids = page_ids(pg, seq, j_lo, j_hi - 1, 0, [&](int j) { return walk.row0(j); });
        // copy tile j into the stage at dst; the pages of its halves
        auto issue = [&](int stage, int j, int& id0, int& id1) {
            const uint32_t d0 = uni(lds_base + stage * R64_STAGE + 8 * w * ROW_B);
            const int r0 = walk.row0(j);
            ids.at(j, id0, id1);
            const int id = w >> 1 ? id1 : id0, r = r0 + 8 * w;   // this wave's page, first row
            const long long at = ((long long)max(id, 0) << pg.shift) + (r & ((1 << pg.shift) - 1));
            if constexpr (DENSE) {
                const long long row = ch.dense[seq] + (r0 < dense_cut ? r0 : r0 - dense_skip) + 8 * w;
                // (of an absent page page 0's: its scores are masked)
                int l = lane;
                asm volatile("" : "+v"(l));   // (as in put_steps)
                copy4_v(uniform_ptr(ksc + (at * n_kv + h) * 16) + (16 * (l & 7) * n_kv + 4 * (l >> 3 & 3)),
                        uni(lds_base + R64_LDS + stage * SCALE_STAGE + w * SCALE_W));
                copy_rows(d0, kb + row * rsb, vb + row * rsb, loff);
                return;
            }
            const char* kr = kb + at * rsb;
            const char* vr = vb + at * rsb;
            if (id >= 0 && r + 8 <= walk.hi && (r >= walk.lo || r + 8 <= sight.sinks)) {
                copy_rows(d0, kr, vr, loff);
            } else {
                const char* zero = (const char*)zero_row + 16 * (lane & 31);
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const int row = r + 2 * n + (lane >> 5);
                    const bool on = id >= 0 && row < walk.hi && (row >= walk.lo || row < sight.sinks);
                    copy16_v(on ? kr + loff[n] : zero, d0 + 2 * n * ROW_B);
                    copy16_v(on ? vr + loff[n] : zero, d0 + R64_TILE + 2 * n * ROW_B);
                }
            }
        };
        // pages of the tiles in flight, tile j's at j % 4
        int id0[R64_NST], id1[R64_NST];
#pragma unroll
        for (int d = 0; d < R64_DIST; ++d)
            if (d < n_tiles) issue(d, j_lo + d, id0[d], id1[d]);

        // Q[row nb][128 hh + 8 ks + 0..7], DENSE [16 ks + 8 hh + 0..7] (a lane past the rows
        // reads token 0's; its column is never stored)
        f16x8 qreg[2][16];
#pragma unroll
        for (int nb = 0; nb < 2; ++nb) {
            const f16* qrow =
                q + ((size_t)(start + t[nb]) * n_q_heads + h * G + g[nb]) * q_pitch + (DENSE ? 8 : 128) * hh;
#pragma unroll
            for (int ks = 0; ks < 16; ++ks) qreg[nb][ks] = *(const f16x8*)(qrow + (DENSE ? 16 : 8) * ks);
        }
        WAIT_VMCNT(0);   // the first tiles, and Q, pinned here: a later wait would drain the copies
        if constexpr (DENSE) {
            asm volatile("" ::: "memory");
            put_steps(smem, 0, 0, w, lane);
        }
#pragma unroll
        for (int nb = 0; nb < 2; ++nb)
#pragma unroll
            for (int ks = 0; ks < 16; ++ks) asm volatile("" : "+v"(qreg[nb][ks]));

        f32x16 o[2][8];
        f16x8 zero = (f16x8)(0);
        asm volatile("" : "+v"(zero));   // (not four registers across the row tiles)
#pragma unroll
        for (int nb = 0; nb < 2; ++nb)
#pragma unroll
            for (int mb = 0; mb < 8; ++mb) acc_zero(o[nb][mb], zero);
        float m_run[2] = {-1e30f, -1e30f}, l_run[2] = {0.f, 0.f};

        typedef __attribute__((address_space(3))) const f16x8 lds_f16x8;
        typedef __attribute__((address_space(3))) const char lds_char;
        constexpr int COPIES = R64_COPIES + DENSE;   // a wave's of a tile
        int st = 0;   // stage of tile j
        for (int j = 0; j < n_tiles; ++j) {
            // tile j landed: the copies of the min(DIST - 1, n_tiles - 1 - j) tiles issued
            // after it may still be in flight
            const int ahead = min(R64_DIST - 1, n_tiles - 1 - j);
            if (ahead == 2) WAIT_VMCNT(2 * COPIES);
            else if (ahead == 1) WAIT_VMCNT(COPIES);
            else WAIT_VMCNT(0);
            tile_done();   // every wave is past tile j - 1: its stage can be refilled
            const int p0 = id0[0], p1 = id1[0];
            id0[0] = id0[1], id1[0] = id1[1];
            id0[1] = id0[2], id1[1] = id1[2];
            if (j + R64_DIST < n_tiles) {
                const int sn = st == 0 ? R64_NST - 1 : st - 1;   // (j + DIST) % NST == (j - 1) % NST
                issue(sn, j_lo + j + R64_DIST, id0[2], id1[2]);
            }
            const int kv0 = walk.row0(j_lo + j);
            if (kv0 <= wqmax) {
                const uint32_t kst = koff + st * R64_STAGE;
                f32x16 s[2] = {(f32x16)(0.f), (f32x16)(0.f)};
                if constexpr (DENSE) {
                    // (the two column blocks alternate: one's products run under the other's steps)
                    auto frag = [&](int ks) {
                        return *(lds_f16x8*)((lds_char*)smem + (kst ^ (32 * ks)));
                    };
                    typedef __attribute__((address_space(3))) const f32x4 lds_f32x4;
                    lds_char* steps = (lds_char*)smem + (STEP_AT + (j & 1) * STEP_B + 16 * hh);
                    f16x8 ka[4] = {frag(0), frag(1), frag(2), frag(3)};
                    f32x4 t[4];   // of rows 8 r4 + 4 hh ..
                    auto product = [&](int nb, int ks) {
                        s[nb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka[ks & 3], qreg[nb][ks], s[nb], 0, 0, 0);
                        __builtin_amdgcn_sched_barrier(0);
                    };
                    auto step = [&](int nb, int r4) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[nb][4 * r4 + e] *= t[r4][e];
                    };
                    // one column block's products alternate with the other's steps
#pragma unroll
                    for (int b = 0; b < 8; ++b) {
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            product(0, 2 * b + k);
#pragma unroll
                            for (int r4 = 2 * k; r4 < 2 * k + 2; ++r4) {   // the last block's step,
                                if (b > 0) step(1, r4);                    // then this one's t
                                t[r4] = *(lds_f32x4*)(steps + 4 * R64_BK * b + 32 * r4);
                            }
                            __builtin_amdgcn_sched_barrier(0);
                        }
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            product(1, 2 * b + k);
                            if (b < 6) ka[(2 * b + k) & 3] = frag(2 * b + 4 + k);
                            step(0, 2 * k), step(0, 2 * k + 1);
                            __builtin_amdgcn_sched_barrier(0);
                        }
                    }
#pragma unroll
                    for (int r4 = 0; r4 < 4; ++r4) step(1, r4);
                } else {
                    constexpr int KPF = R64_KPF;
                    f16x8 ka[KPF];
#pragma unroll
                    for (int ks = 0; ks < KPF; ++ks)
                        ka[ks] = *(lds_f16x8*)((lds_char*)smem + (kst ^ (16 * ks)));
#pragma unroll
                    for (int ks = 0; ks < 16; ++ks) {
                        const f16x8 a = ka[ks % KPF];
                        if (ks + KPF < 16)
                            ka[ks % KPF] = *(lds_f16x8*)((lds_char*)smem + (kst ^ (16 * (ks + KPF))));
                        s[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qreg[0][ks], s[0], 0, 0, 0);
                        s[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qreg[1][ks], s[1], 0, 0, 0);
                        __builtin_amdgcn_sched_barrier(0);   // keep the reads ahead
                    }
                }
                // whole: every query of the wave sees every row (uniform)
                const TileMask mask(kv0, p0, p1, sight.sinks);
                auto low = [&](int p) {
                    return sight.window > 0 && p >= sight.window ? p - sight.window + 1 : 0;
                };
                const bool whole = mask.all(low(wqmax), wqmin + 1);
                f16x8 pk[2][2], pl[2][2];
#pragma unroll
                for (int nb = 0; nb < 2; ++nb) {
                    uint32_t see = 0;
                    if (!whole) see = mask.rows(low(qpos[nb]), qpos[nb] + 1) >> (4 * hh);
                    softmax_block<DENSE>(s[nb], whole, see, sl2, m_run[nb], l_run[nb], o[nb], pk[nb], pl[nb]);
                }
                const char* vt = smem + st * R64_STAGE + R64_TILE;
                auto operand = [](const s16x4& lo, const s16x4& hi) {
                    const f16x4 lf = __builtin_bit_cast(f16x4, lo), hf = __builtin_bit_cast(f16x4, hi);
                    return (f16x8){lf[0], lf[1], lf[2], lf[3], hf[0], hf[1], hf[2], hf[3]};
                };
                if constexpr (DENSE) {
                    // O^T += V^T P^T, 16 fragments with 2 blocks x 2 terms each, VPF fragments read ahead
                    constexpr int VPF = 4;
                    s16x4 vf[VPF][2];
                    auto read = [&](int i) {   // fragment i: rows 16 (i / 8) .., dim block 4 (i / 4 % 2) + i % 4
                        const int imm = 16 * ROW_B * (i >> 3) + 256 * (i >> 2 & 1);
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            vf[i % VPF][e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                (lds_s16x4*)(vt + troff[2 * (i & 3) + e] + imm));
                    };
#pragma unroll
                    for (int i = 0; i < VPF; ++i) read(i);
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const f16x8 av = operand(vf[i % VPF][0], vf[i % VPF][1]);
                        const int mb = i & 7, kq = i >> 3;
                        acc_mfma(o[0][mb], av, pk[0][kq]);
                        acc_mfma(o[1][mb], av, pk[1][kq]);
                        acc_mfma(o[0][mb], av, pl[0][kq]);
                        acc_mfma(o[1][mb], av, pl[1][kq]);
                        if (i + VPF < 16) read(i + VPF);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                } else {
                    // O^T += V^T P^T: 4 steps (kq, dim half) of 4 fragments x 2 blocks, the next
                    // step's fragments read under this step's MFMAs
                    s16x4 vf[2][8];
                    r64_vfrags(vf[0], vt, troff, 0);
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        if (n + 1 < 4) r64_vfrags(vf[(n + 1) & 1], vt, troff, n + 1);
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            const f16x8 av = operand(vf[n & 1][2 * u], vf[n & 1][2 * u + 1]);
                            acc_mfma(o[0][4 * (n & 1) + u], av, pk[0][n >> 1]);
                            acc_mfma(o[1][4 * (n & 1) + u], av, pk[1][n >> 1]);
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
            st = st == R64_NST - 1 ? 0 : st + 1;
            if (DENSE && j + 1 < n_tiles) {
                // the next tile's steps: its scales were copied ahead of its rows, those of the
                // tiles after it may still be in flight
                const int later = min(R64_DIST - 1, n_tiles - 2 - j);
                if (later == 2) WAIT_VMCNT(2 * COPIES + R64_COPIES);
                else if (later == 1) WAIT_VMCNT(COPIES + R64_COPIES);
                else WAIT_VMCNT(R64_COPIES);
                asm volatile("" ::: "memory");
                put_steps(smem, st, j + 1, w, lane);
            }
        }

        // O leaves through LDS, a 32-row block at a time in this wave's quarter of the
        // stages, so that rows are written (and gates read) whole: chunk c (4 dims) of row r
        // at c ^ 2 r. A cut row tile's rows go to its partial, a whole one's to z.
        acc_settle(o[0]);
        acc_settle(o[1]);
        tile_done();   // every wave is past its last tile
        const bool part = CUT && n_tiles < walk.n;
        char* ob = smem + w * (R64_LDS / 4);
        int oq = ql, ol = lane;   // (opaque: the addresses below would be hoisted out of the tile
        asm volatile("" : "+v"(oq), "+v"(ol));   // loop and held in registers that it needs)
        const int first = R0 + 64 * w, rows = min(64, RT - first);   // this wave's rows (uniform)
        // the (token, q head) row of its rows, one after the other; past the last the last
        int tt = uni(first / G), gg = first - tt * G, left = rows;
        auto next_row = [&] {
            const size_t rh = (size_t)(start + tt) * n_q_heads + h * G + gg;
            if (--left > 0 && ++gg == G) gg = 0, ++tt;
            return rh;
        };
        const size_t slot0 = (size_t)(slot + h * parts.n) * R64_BQ + 64 * w;
        // gates are requested OUT_ROWS rows ahead of their use (no gate: one that is open)
        f16x4 g_next[OUT_ROWS] = {};   // (undefined ones would hold registers through the tile loop)
        size_t rh_next[OUT_ROWS] = {};
        auto request = [&] {
#pragma unroll
            for (int i = 0; i < OUT_ROWS; ++i) {
                rh_next[i] = next_row();
                g_next[i] = (f16x4)((f16)65504.f);
            }
            if (gated && !part) {
#pragma unroll
                for (int i = 0; i < OUT_ROWS; ++i)
                    g_next[i] = *(const f16x4*)(q + rh_next[i] * q_pitch + PF_HD + 4 * ol);
            }
        };
        if (rows > 0) request();
#pragma unroll
        for (int nb = 0; nb < 2; ++nb) {
            const int n = min(32, rows - 32 * nb);   // (uniform)
            if (n <= 0) break;
#pragma unroll
            for (int mb = 0; mb < 8; ++mb)
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4)
                    *(f32x4*)(ob + 1024 * oq + 16 * ((8 * mb + 2 * r4 + hh) ^ (2 * oq))) =
                        (f32x4){o[nb][mb][4 * r4], o[nb][mb][4 * r4 + 1], o[nb][mb][4 * r4 + 2],
                                o[nb][mb][4 * r4 + 3]};
            if (part && lane < n) {   // (lanes 0 .. 31 hold the columns)
                parts.pm[slot0 + 32 * nb + lane] = m_run[nb];
                parts.pd[slot0 + 32 * nb + lane] = l_run[nb];
            }
#pragma unroll 1
            for (int r0 = 0; r0 < n; r0 += OUT_ROWS) {
                f32x4 v[OUT_ROWS];
                float l[OUT_ROWS];
#pragma unroll
                for (int i = 0; i < OUT_ROWS; ++i) {
                    const int r = min(r0 + i, n - 1);   // (past the last row: the last once more)
                    v[i] = *(const f32x4*)(ob + 1024 * r + 16 * (ol ^ (2 * r)));
                    l[i] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(l_run[nb]), r));
                }
                if (part) {
#pragma unroll
                    for (int i = 0; i < OUT_ROWS; ++i)
                        *(f32x4*)(parts.pacc + (slot0 + 32 * nb + min(r0 + i, n - 1)) * PF_HD + 4 * ol) = v[i];
                    continue;
                }
                f16x4 gv[OUT_ROWS];
                size_t rh[OUT_ROWS];
#pragma unroll
                for (int i = 0; i < OUT_ROWS; ++i) gv[i] = g_next[i], rh[i] = rh_next[i];
                request();
#pragma unroll
                for (int i = 0; i < OUT_ROWS; ++i) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {   // O / l sigmoid(g) = O / (l + l e^-g)
                        const float x = fast_exp2(fmaf((float)gv[i][e], -FL_LOG2E, 0.f));
                        v[i][e] *= __builtin_amdgcn_rcpf(fmaf(l[i], x, l[i]));
                    }
                    *(f16x4*)(z + rh[i] * z_pitch + 4 * ol) = f16_sat4(v[i]);
                }
            }
            // queries that see no row give 0, whatever their gates and the rows that others
            // see hold: rare, so written over what was formed above
            if (!part)
                for (uint32_t blind = (uint32_t)__ballot(lane < n && l_run[nb] == 0.f); blind;
                     blind &= blind - 1) {
                    const int row = first + 32 * nb + __builtin_ctz(blind), tb = row / G;
                    const size_t at = (size_t)(start + tb) * n_q_heads + h * G + row - tb * G;
                    *(f16x4*)(z + at * z_pitch + 4 * ol) = (f16x4)(0);
                }
        }
        if (part) ++slot;
    }
}

// The cut row tiles of a plan: row tile `tile`'s partials are slots first .. + n - 1.
struct CutTiles {
    int n;
    uint16_t tile[MAX_RUNS], first[MAX_RUNS], count[MAX_RUNS];
};

// z of the cut row tiles: a wave a row, lane l holding dims 4 l .. + 3, the partials in
// batches whose loads are all issued before any is used, against one running maximum.
constexpr int PM_BATCH = 8;
__global__ void __launch_bounds__(256)
paged_piece_merge_kernel(const Parts in, const Chunks ch, const CutTiles cut, f16* __restrict__ z,
                         int z_pitch, const f16* __restrict__ gate, int g_pitch, int n_q_heads, int n_kv) {
    const int lane = threadIdx.x & 63, h = blockIdx.y, G = n_q_heads / n_kv;
    const int c = uni(blockIdx.x / (R64_BQ / 4)), r = uni(4 * (blockIdx.x % (R64_BQ / 4)) + (threadIdx.x >> 6));
    const int tile = cut.tile[c], ns = cut.count[c];
    int seq = 0;
    while (tile >= ch.tile0[seq + 1]) ++seq;
    const int row = (tile - ch.tile0[seq]) * R64_BQ + r;
    if (row >= (ch.start[seq + 1] - ch.start[seq]) * G) return;   // (wave-uniform)
    const int t = row / G;
    const size_t rh = (size_t)(ch.start[seq] + t) * n_q_heads + h * G + row - t * G;
    f16x4 gv = (f16x4)(0);
    if (gate != nullptr) gv = *(const f16x4*)(gate + rh * g_pitch + 4 * lane);
    const size_t p0 = (size_t)(h * in.n + cut.first[c]) * R64_BQ + r;
    f32x4 num = (f32x4)(0.f);
    float den = 0.f, M = -1e30f;
    for (int s = 0; s < ns; s += PM_BATCH) {
        float mv[PM_BATCH], dv[PM_BATCH];
        f32x4 av[PM_BATCH];
#pragma unroll
        for (int k = 0; k < PM_BATCH; ++k) {
            if (s + k >= ns) break;   // uniform
            const size_t at = p0 + (size_t)(s + k) * R64_BQ;
            mv[k] = in.pm[at];
            dv[k] = in.pd[at];
            av[k] = *(const f32x4*)(in.pacc + at * PF_HD + 4 * lane);
        }
        float bm = M;
#pragma unroll
        for (int k = 0; k < PM_BATCH; ++k)
            if (s + k < ns) bm = fmaxf(bm, mv[k]);
        const float corr = fast_exp2(M - bm);
        num *= corr;
        den *= corr;
        M = bm;
#pragma unroll
        for (int k = 0; k < PM_BATCH; ++k) {
            if (s + k >= ns) break;
            const float e = fast_exp2(mv[k] - M);
            num += e * av[k];
            den = fmaf(e, dv[k], den);
        }
    }
    const float inv = 1.f / den;
    f16x4 out;
#pragma unroll
    for (int e = 0; e < 4; ++e)   // (no row seen: 0)
        out[e] = den == 0.f ? (f16)0.f
                            : f16_sat(num[e] * (gate != nullptr ? inv * fast_sigmoid((float)gv[e]) : inv));
    *(f16x4*)(z + rh * z_pitch + 4 * lane) = out;
}

// ---------------------------------------------------------------------------
// host: chunks, plan, launch
// ---------------------------------------------------------------------------

int make_chunks(const int* Ts, const int* pos0s, int B, int G, long long capacity, Chunks& ch) {
    FL_REQUIRE(Ts && pos0s, "null pointer");
    FL_REQUIRE(B >= 1 && B <= MAX_SEQS, "1 <= B <= FL_PAGED_MAX_SEQS_PREFILL");
    memset(&ch, 0, sizeof(ch));
    ch.n = B;
    long long at = 0, tiles = 0;
    for (int b = 0; b < B; ++b) {
        FL_REQUIRE(Ts[b] >= 0 && pos0s[b] >= 0, "T, pos0 >= 0");
        FL_REQUIRE((long long)pos0s[b] + Ts[b] <= capacity, "pos0 + T <= max_pages * page_size");
        ch.pos0[b] = pos0s[b];
        at += Ts[b];
        tiles += ((long long)Ts[b] * G + R64_BQ - 1) / R64_BQ;
        FL_REQUIRE(tiles < 65536, "sum of T n_q_heads / n_kv_heads under 2^24 a call");
        ch.start[b + 1] = (int)at;
        ch.tile0[b + 1] = (int)tiles;
    }
    return FL_OK;
}

// The rows of a sequence in the fp16 copy: those of the union of its row tiles' walks.
int dense_rows(int T, int pos0, const Sight& sight) {
    return T == 0 ? 0 : R64_BK * make_walk(pos0, pos0 + T - 1, sight).n;
}

// The plan's costs, in tiles' time (2.0 us: 8192 fresh tokens are 387 tiles a CU and three row
// tiles' ends). They are chosen by the plans they give, not fitted: a row tile's start and end are
// 16 - 20 us, 448 partials' merge 34 us where the rule says 13 tiles.
constexpr int ITEM_COST = 12;   // a row tile's (Q, pipeline fill, z); 5, 8, 10, 12, 14: 856, 845,
                                // 842, 842, 839 us for 8192 fresh tokens, 61.6, 55.4, 60.6, 57.0,
                                // 61.0 for 1024
constexpr int PIECE_COST = 8;   // a piece's (its 256 KiB partial)
constexpr int PIECE_MIN = 2;    // tiles a piece, at least
constexpr int RUN_MIN = 6;      // a run's cost, at least; 20, 8, 6, 3: 70, 57, 56, 56 us for 1024
                                // fresh tokens, 61, 41, 40, 38 for 37 at 3001
constexpr int MERGE_COST = 2;        // the merge's launch
constexpr int SLOTS_PER_TILE = 40;   // partials the merge reads in a tile's time

struct CallPlan {
    bool cut;
    int slots;
    Plan plan;
    CutTiles tiles;
};

void walks(const Chunks& ch, int G, const Sight& sight, std::vector<int>& n) {
    n.clear();
    for (int b = 0; b < ch.n; ++b) {
        const int RT = (ch.start[b + 1] - ch.start[b]) * G;
        for (int R0 = 0; R0 < RT; R0 += R64_BQ)
            n.push_back(make_walk(ch.pos0[b] + R0 / G,
                                  ch.pos0[b] + std::min(R0 + R64_BQ - 1, RT - 1) / G, sight).n);
    }
}

// The cut plan over at most `most` runs, and its cost (the longest run and the merge).
long long cut_plan(const std::vector<int>& n, int n_kv, int most, CallPlan& cp) {
    const int N = (int)n.size();
    long long total = 0;
    for (int x : n) total += x + ITEM_COST;
    const int runs = (int)std::max<long long>(
        1, std::min<long long>(most, total / RUN_MIN));
    Plan& p = cp.plan;
    p.runs = runs;
    int tile = 0;
    long long before = 0;   // cost of the row tiles ahead of `tile`
    for (int r = 0; r <= runs; ++r) {
        const long long u = r == runs ? total : total * r / runs;
        while (tile < N && before + n[tile] + ITEM_COST <= u) before += n[tile++] + ITEM_COST;
        int j = tile < N ? (int)std::max<long long>(0, u - before - ITEM_COST) : 0;
        int t = tile;
        if (j < PIECE_MIN) j = 0;
        else if (n[t] - j < PIECE_MIN) ++t, j = 0;
        p.cut.tile[r] = (uint16_t)t;
        p.cut.j[r] = (uint32_t)j;
    }
    // slots of the cut row tiles' pieces, in stream order
    cp.slots = 0;
    cp.tiles.n = 0;
    long long longest = 0;
    int open = -1;   // the cut row tile that the last partial belongs to
    for (int r = 0; r < runs; ++r) {
        p.cut.slot[r] = (uint16_t)cp.slots;
        const int t0 = p.cut.tile[r], t1 = p.cut.tile[r + 1];
        const int j0 = (int)p.cut.j[r], j1 = (int)p.cut.j[r + 1];
        long long cost = 0;
        for (int t = t0; t < t1 + (j1 > 0 ? 1 : 0); ++t) {
            const int lo = t == t0 ? j0 : 0, hi = t == t1 ? j1 : n[t];
            if (hi == lo) continue;
            const bool part = hi - lo < n[t];
            cost += hi - lo + (part ? PIECE_COST : ITEM_COST);
            if (!part) continue;
            if (open != t) {
                cp.tiles.tile[cp.tiles.n] = (uint16_t)t;
                cp.tiles.first[cp.tiles.n] = (uint16_t)cp.slots;
                cp.tiles.count[cp.tiles.n++] = 0;
                open = t;
            }
            ++cp.tiles.count[cp.tiles.n - 1];
            ++cp.slots;
        }
        longest = std::max(longest, cost);
    }
    return longest + (cp.slots ? MERGE_COST + cp.slots * n_kv / SLOTS_PER_TILE : 0);
}

// The plan of whole row tiles, the heaviest first to the lightest run, then moves and swaps
// off the heaviest run while they shorten it (8192 fresh tokens 0.89 -> 0.83 ms; 0.1 ms of
// host time for their 192 row tiles, up to 2.4 for a thousand unlike ones, once for the layers
// of a step); and its cost, 0 where its list does not fit.
long long whole_plan(const std::vector<int>& n, int most, Plan& p) {
    const int N = (int)n.size();
    if (N > LIST_MAX) return 0;
    const int runs = std::min(most, N);
    std::vector<int> order(N), run_of(N);
    for (int t = 0; t < N; ++t) order[t] = t;
    std::stable_sort(order.begin(), order.end(), [&](int a, int b) { return n[a] > n[b]; });
    typedef std::pair<long long, int> Load;
    std::priority_queue<Load, std::vector<Load>, std::greater<Load>> light;
    for (int r = 0; r < runs; ++r) light.push({0, r});
    std::vector<std::vector<int>> list(runs);
    std::vector<long long> load(runs, 0);
    long long total = 0;
    for (int t : order) {
        Load l = light.top();
        light.pop();
        list[l.second].push_back(t);
        load[l.second] = l.first += n[t] + ITEM_COST;
        total += n[t] + ITEM_COST;
        light.push(l);
    }
    for (int round = 0; round < 4 * N; ++round) {
        const int hi = (int)(std::max_element(load.begin(), load.end()) - load.begin());
        if (load[hi] * runs <= total + total / 256) break;   // even to 0.4 %
        long long best = load[hi];
        int bx = -1, by = -1, bl = -1;   // list[hi][bx] to run bl, for list[bl][by] (by < 0: for none)
        for (int lo = 0; lo < runs; ++lo) {
            if (lo == hi) continue;
            for (int x = 0; x < (int)list[hi].size(); ++x)
                for (int y = -1; y < (int)list[lo].size(); ++y) {
                    const long long d =
                        n[list[hi][x]] - (y < 0 ? -ITEM_COST : n[list[lo][y]]);
                    const long long m = std::max(load[hi] - d, load[lo] + d);
                    if (d > 0 && m < best) best = m, bx = x, by = y, bl = lo;
                }
        }
        if (bl < 0) break;
        const int t = list[hi][bx];
        const long long d = n[t] - (by < 0 ? -ITEM_COST : n[list[bl][by]]);
        load[hi] -= d;
        load[bl] += d;
        if (by < 0) {
            list[hi].erase(list[hi].begin() + bx);
            list[bl].push_back(t);
        } else {
            std::swap(list[hi][bx], list[bl][by]);
        }
    }
    const long long longest = *std::max_element(load.begin(), load.end());
    p.runs = runs;
    int k = 0;
    for (int r = 0; r < runs; ++r) {
        p.whole.at[r] = (uint16_t)k;
        for (int t : list[r]) p.whole.list[k++] = (uint16_t)t;
    }
    p.whole.at[runs] = (uint16_t)k;
    return longest;
}

void make_plan(const Chunks& ch, int G, int n_kv, const Sight& sight, int n_cu, CallPlan& cp) {
    std::vector<int> n;
    walks(ch, G, sight, n);
    const int most = std::min(MAX_RUNS, std::max(1, n_cu / n_kv));
    const long long cut = cut_plan(n, n_kv, most, cp);
    Plan whole;
    const long long w = whole_plan(n, most, whole);
    // (whole / cut, us: 8192 fresh tokens 842 / 921, 130 fresh 31.2 / 32.4, four chunks of 1024
    // with a window 545 / 455, 1024 at 30000 1841 / 813, 37 at 3001 197 / 40)
    cp.cut = w == 0 || cut < w;
    if (!cp.cut) {
        cp.plan = whole;
        cp.slots = cp.tiles.n = 0;
    }
}

// ... kept for the last few calls (the layers of a step ask the same)
struct PlanEntry {
    bool used;
    Chunks ch;
    int G, n_kv, n_cu;
    Sight sight;
    CallPlan cp;
};
constexpr int PLAN_CACHE = 8;
std::mutex g_mu;
PlanEntry g_plans[PLAN_CACHE];
int g_next;

// FL_OK, or FL_ELAUNCH without host memory
int call_plan(const Chunks& ch, int G, int n_kv, const Sight& sight, int n_cu, CallPlan& cp) {
    {
        std::lock_guard<std::mutex> lock(g_mu);
        for (const PlanEntry& e : g_plans)
            if (e.used && e.G == G && e.n_kv == n_kv && e.n_cu == n_cu && e.sight.window == sight.window &&
                e.sight.sinks == sight.sinks && memcmp(&e.ch, &ch, sizeof(ch)) == 0) {
                cp = e.cp;
                return FL_OK;
            }
    }
    try {
        make_plan(ch, G, n_kv, sight, n_cu, cp);
    } catch (const std::bad_alloc&) {
        fl::set_error("attention_prefill_paged: no host memory for the plan");
        return FL_ELAUNCH;
    }
    std::lock_guard<std::mutex> lock(g_mu);
    PlanEntry& e = g_plans[g_next];
    e.used = true, e.ch = ch, e.G = G, e.n_kv = n_kv, e.n_cu = n_cu, e.sight = sight, e.cp = cp;
    g_next = (g_next + 1) % PLAN_CACHE;
    return FL_OK;
}

size_t parts_bytes(int slots, int n_kv) { return (size_t)slots * n_kv * R64_BQ * (PF_HD + 2) * 4; }

// The rows of the fp16 copy of an int8 call; ch.dense[] set.
long long lay_dense(Chunks& ch, const Sight& sight) {
    long long at = 0;
    for (int b = 0; b < ch.n; ++b) {
        ch.dense[b] = (int)at;
        at += dense_rows(ch.start[b + 1] - ch.start[b], ch.pos0[b], sight);
        if (at > INT_MAX / 2) return -1;
    }
    return at;
}
size_t dense_bytes(long long rows, int n_kv) { return 2 * (size_t)rows * n_kv * ROW_B; }

// The sequences of an int8 call whose copies fit GROUP_BYTES together, from `b` on (one at
// least): the call runs a group after the other over the same work, so that a batch of long
// contexts does not ask for tens of GB (4 KiB a row at 4 kv heads).
constexpr size_t GROUP_BYTES = (size_t)1 << 30;
int group_end(const int* Ts, const int* pos0s, int B, int b, int n_kv, const Sight& sight) {
    size_t bytes = 0;
    int e = b;
    for (; e < B; ++e) {
        const long long rows = dense_rows(Ts[e], pos0s[e], sight);
        bytes += dense_bytes(rows, n_kv);
        if (e > b && bytes > GROUP_BYTES) break;
    }
    return e;
}

// Dynamic LDS above the default limit, raised once per device.
int raise_lds() {
    static std::atomic<bool> done[64];
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) {
        fl::set_error("attention_prefill_paged: no current device below index 64");
        return FL_ELAUNCH;
    }
    if (done[dev].load()) return FL_OK;
    const void* fns[] = {(const void*)paged_prefill_kernel<false, false>,
                         (const void*)paged_prefill_kernel<false, true>,
                         (const void*)paged_prefill_kernel<true, false>,
                         (const void*)paged_prefill_kernel<true, true>};
    for (const void* f : fns)
        if (hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, DENSE_LDS) != hipSuccess) {
            fl::set_error("attention_prefill_paged: cannot raise the dynamic LDS limit to %d bytes",
                          DENSE_LDS);
            return FL_ELAUNCH;
        }
    done[dev].store(true);
    return FL_OK;
}

int too_little_work(size_t have, size_t need) {
    fl::set_error("work: %zu bytes, fl_attention_prefill_paged_work_bytes asks %zu", have, need);
    return FL_ESCRATCH;
}

// The fp16 copy, K as the bytes (a block of scale 0 as zeros) and V as f16(byte scale): row i of
// sequence b's part is the row of the union of its walks; a wave a row, 8 dims (both of K and V)
// a lane and step. Rows past the sequence and of absent pages are zeros.
__global__ void __launch_bounds__(256)
paged_stage_kernel(const char* __restrict__ kp, const char* __restrict__ vp, const Pages pg,
                   const Chunks ch, const Sight sight, f16x8* __restrict__ ko, f16x8* __restrict__ vo,
                   long long rows, int n_kv) {
    const long long i = (long long)blockIdx.x * 4 + uni(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (i >= rows) return;   // (wave-uniform)
    int seq = ch.n - 1;
    while (seq > 0 && i < ch.dense[seq]) --seq;
    const int p0 = ch.pos0[seq], end = p0 + ch.start[seq + 1] - ch.start[seq];
    const Walk first = make_walk(p0, p0, sight);
    const int k = (int)(i - ch.dense[seq]);
    const int pos = k < R64_BK * first.s ? k : k + R64_BK * (first.a - first.s);
    const bool seen = pos < end && (pos >= first.lo || pos < sight.sinks);
    const long long row = seen ? fl::page_row(pg, seq, pos) : -1;
    const int chunks = n_kv * (PF_HD / 8);
    const size_t scales = (((size_t)pg.n_pages << pg.shift) * n_kv) * PF_HD;
    for (int c = lane; c < chunks; c += 64) {
        f16x8 kx = (f16x8)(0), vx = (f16x8)(0);
        if (row >= 0) {
            const size_t at = (size_t)row * chunks + c;
            auto get = [&](const char* pool, f16 s) {
                const u32x2 b = *(const u32x2*)(pool + 8 * at);
                const f16x4 lo = q8_deq4(b.x, (f16x2){s, s}), hi = q8_deq4(b.y, (f16x2){s, s});
                return (f16x8){lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            };
            // (a block of scale 0 is 0 whatever its bytes)
            kx = get(kp, ((const f16*)(kp + scales))[at >> 2] != (f16)0.f ? (f16)1.f : (f16)0.f);
            vx = get(vp, ((const f16*)(vp + scales))[at >> 2]);
        }
        ko[(size_t)i * chunks + c] = kx;
        vo[(size_t)i * chunks + c] = vx;
    }
}

}  // namespace

extern "C" {

size_t fl_attention_prefill_paged_work_bytes(const int* Ts, const int* pos0s, int B, int n_q_heads,
                                             int n_kv_heads, int head_dim, int window, int sinks,
                                             int q8) {
    if (n_kv_heads < 1 || n_q_heads < 1 || n_q_heads % n_kv_heads || head_dim != PF_HD || window < 0 ||
        sinks < 0)
        return 0;
    const int G = n_q_heads / n_kv_heads;
    const Sight sight = {window, sinks};
    Chunks ch;
    if (make_chunks(Ts, pos0s, B, G, INT_MAX - 1024, ch)) return 0;
    size_t most = 0;
    for (int b = 0, e; b < B; b = e) {
        e = q8 ? group_end(Ts, pos0s, B, b, n_kv_heads, sight) : B;
        CallPlan cp;
        if (make_chunks(Ts + b, pos0s + b, e - b, G, INT_MAX - 1024, ch)) return 0;
        if (ch.start[e - b] == 0) continue;
        if (call_plan(ch, G, n_kv_heads, sight, cu_count(), cp)) return 0;
        const long long rows = q8 ? lay_dense(ch, sight) : 0;
        if (rows < 0) return 0;
        most = std::max(most, up16(parts_bytes(cp.slots, n_kv_heads)) + dense_bytes(rows, n_kv_heads));
    }
    return most;
}

int fl_attention_prefill_paged(const void* q, int q_pitch, const void* kpool, const void* vpool,
                               int q8, int n_pages, int page_size, const int* pages, int max_pages,
                               long long pages_stride, const int* Ts, const int* pos0s, int B,
                               int n_q_heads, int n_kv_heads, int head_dim, float scale, int window,
                               int sinks, int gated, void* z, int z_pitch, void* work,
                               size_t work_bytes, fl_stream_t stream_) {
    Pages pg;
    int rc = fl::make_pages(kpool, vpool, q8, n_pages, page_size, pages, max_pages, pages_stride, B,
                            n_kv_heads, head_dim, pg);
    if (rc) return rc;
    rc = check_heads(q, q_pitch, z, z_pitch, gated, n_q_heads, n_kv_heads, scale, window, sinks);
    if (rc) return rc;
    Chunks ch;
    const int G = n_q_heads / n_kv_heads;
    rc = make_chunks(Ts, pos0s, B, G, (long long)max_pages * page_size, ch);
    if (rc) return rc;
    if (ch.start[B] == 0) return FL_OK;
    const Sight sight = {window, sinks};
    if (q8 && group_end(Ts, pos0s, B, 0, n_kv_heads, sight) < B) {
        const size_t need = fl_attention_prefill_paged_work_bytes(Ts, pos0s, B, n_q_heads, n_kv_heads,
                                                                  head_dim, window, sinks, q8);
        if (work == nullptr || work_bytes < need) return too_little_work(work_bytes, need);
        for (int b = 0, e; b < B; b = e) {
            e = group_end(Ts, pos0s, B, b, n_kv_heads, sight);
            const size_t row = (size_t)ch.start[b] * n_q_heads;
            rc = fl_attention_prefill_paged((const f16*)q + row * q_pitch, q_pitch, kpool, vpool, q8,
                                            n_pages, page_size, pages + b * pages_stride, max_pages,
                                            pages_stride, Ts + b, pos0s + b, e - b, n_q_heads,
                                            n_kv_heads, head_dim, scale, window, sinks, gated,
                                            (f16*)z + row * z_pitch, z_pitch, work, work_bytes, stream_);
            if (rc) return rc;
        }
        return FL_OK;
    }
    const int n_cu = cu_count();
    CallPlan cp;
    rc = call_plan(ch, G, n_kv_heads, sight, n_cu, cp);
    if (rc) return rc;
    const long long rows = q8 ? lay_dense(ch, sight) : 0;
    FL_REQUIRE(rows >= 0, "too many cached rows for one int8 call");
    const size_t part_b = up16(parts_bytes(cp.slots, n_kv_heads));
    const size_t need = part_b + dense_bytes(rows, n_kv_heads);
    if (need > 0) {
        if (work == nullptr || work_bytes < need) return too_little_work(work_bytes, need);
        FL_REQUIRE(aligned16(work), "16-byte aligned work");
    }
    rc = raise_lds();
    if (rc) return rc;
    const hipStream_t stream = (hipStream_t)stream_;
    const size_t part_rows = (size_t)cp.slots * n_kv_heads * R64_BQ;
    Parts parts = {(float*)work, nullptr, nullptr, cp.slots};
    parts.pm = parts.pacc + part_rows * PF_HD;
    parts.pd = parts.pm + part_rows;
    const char *kc = (const char*)kpool, *vc = (const char*)vpool, *ksc = nullptr;
    if (q8) {
        ksc = kc + (((size_t)n_pages << pg.shift) * n_kv_heads) * PF_HD;
        char* copy = (char*)work + part_b;
        char* copy_v = copy + dense_bytes(rows, n_kv_heads) / 2;
        hipLaunchKernelGGL(paged_stage_kernel, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, stream, kc,
                           vc, pg, ch, sight, (f16x8*)copy, (f16x8*)copy_v, rows, n_kv_heads);
        rc = fl::check_launch("attention_prefill_paged int8 copy");
        if (rc) return rc;
        kc = copy;
        vc = copy_v;
    }
    auto kernel = q8 ? (cp.cut ? paged_prefill_kernel<true, true> : paged_prefill_kernel<true, false>)
                     : (cp.cut ? paged_prefill_kernel<false, true> : paged_prefill_kernel<false, false>);
    // a whole number of workgroups an XCD, so that its kv head's rows stay in one L2
    const int per = 8 % n_kv_heads == 0 ? 8 / n_kv_heads : 1;
    const int runs = (cp.plan.runs + per - 1) / per * per;
    hipLaunchKernelGGL(kernel, dim3(runs * n_kv_heads), dim3(THREADS), q8 ? DENSE_LDS : R64_LDS, stream,
                       (const f16*)q, q_pitch, kc, vc, ksc, pg, ch, (f16*)z, z_pitch, gated, n_q_heads,
                       n_kv_heads, scale * FL_LOG2E, sight, cp.plan, parts);
    rc = fl::check_launch("attention_prefill_paged");
    if (rc || cp.tiles.n == 0) return rc;
    hipLaunchKernelGGL(paged_piece_merge_kernel, dim3(cp.tiles.n * (R64_BQ / 4), n_kv_heads), dim3(256), 0,
                       stream, parts, ch, cp.tiles, (f16*)z, z_pitch,
                       gated ? (const f16*)q + PF_HD : nullptr, q_pitch, n_q_heads, n_kv_heads);
    return fl::check_launch("attention_prefill_paged merge");
}

}  // extern "C"
