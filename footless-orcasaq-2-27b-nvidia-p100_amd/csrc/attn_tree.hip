// Attention of trees of drafted tokens over the paged KV cache (attn_paged.hpp, tree.hpp).
//
// Token i of a sequence, at position p = pos0 + depth(i), sees the context's rows r < pos0 with
// r > p - window or r < sinks, and of the tree's rows pos0 + j those of its ancestors and its own
// whose position pos0 + depth(j) is in sight alike. The rest is the decode's:
//   z = f16_sat(sum_r e^(scale q.k_r - m) v_r / sum_r e^(scale q.k_r - m) * sigmoid(gate)).
//
// The T G query rows of a kv head are columns. A workgroup has 16 of them on each of its 4, 8 or 12
// waves, and walks tiles of 32 cache rows that its waves share through LDS:
//   S^T (32 rows x 16 columns) = K Q^T        16x16x32 MFMAs, Q in registers
//   softmax                                   a lane holds column i's rows 4 g + e of both halves
//   O^T (256 dims x 16 columns) += V^T P^T    P as it lies: k slot (g, e) is row 4 g + e of half
//                                             e / 4; V^T by transposed LDS reads
// The tiles that the sequences' trees see make one stream a kv head and group of columns, cut into
// equal runs, one a workgroup, wherever the cuts fall; the runs are found from pos0 on the device, so
// that a captured call follows it. A sequence that lies in one run is finished there; a cut one leaves
// a partial a piece, which the merge weighs.
//
// Measured, from a graph: a tree of 16 on 500 rows 17 us, 8 of them on 8192 62 us (4.4 TB/s, int8 73 us), 16 of 8
// tokens on 16384 195 us (5.5 TB/s, int8 175), 4 of 63 on 20000 to 60000 282 us (0.82 PFLOP/s; 291 on another card),
// 12 of 5 to 26 on 100 to 32768 int8 rows 117 us. Small trees are bound by the cache's bytes, and by what comes ahead of the first
// tile and behind the last (a sequence's tree, plan and first rows 10 us one behind another, the partials' merge
// 4 to 12); a large one's tile of 32 rows and 192 columns takes 3100 clocks (int8 5000), of which MFMAs are 1540
// (2300) and LDS reads as many: a tile's waves are in step and use both at once. Scores of the next tile under the
// softmax, two tiles a barrier, an int8 tile's conversion under the products with V, and waves that convert
// ahead of their products beside waves that do behind them were all built, and none was faster.
#include "attn_paged.hpp"
#include "tree.hpp"

#include <algorithm>

using fl::Pages;
using fl::PAGED_HD;

namespace {

constexpr int TT = 32;                  // rows a tile
constexpr int ROW_B = 2 * PAGED_HD;     // bytes a row in LDS
constexpr int TILE_B = TT * ROW_B;
constexpr int STAGE_B = 2 * TILE_B;     // K | V
// Tiles a run, at least: with one a tree of 16 on 2000 rows takes 25 us in place of 23 (more partials), with
// six 4 trees of 32 on 1000 rows 42 us in place of 34 (CUs without work).
constexpr int RUN_MIN = 3;
// What a sequence's start costs in tiles, where there are several (its tree, plan, Q and first rows come one
// behind another): counted as 2, 8 trees of 16 on 8192 rows take 68 us in place of 61, and 12 of 26 on ragged
// int8 rows 141 us in place of 121; 12 is no better.
constexpr int SEQ_COST = 8;

// The chunk swizzle of tile row r: 16-byte chunk c lies at c ^ sw(r). A read of 16 bytes a lane takes
// lanes 0 - 3, 12 - 15, 20 - 27 together, then 4 - 11, 16 - 19, 28 - 31, ...: 16 rows of K at chunk c
// and, of other rows, at c + 1; one of V^T's 8 bytes a lane takes 8 rows' pairs of chunks together. With
// these values both meet every bank once (with r / 4 in place of -r / 4 half of the LDS cycles are conflicts).
__device__ __forceinline__ int sw(int r) { return ((r & 3) << 2) | (-(r >> 2) & 3); }

// What a sequence's tokens see at most, as tiles: the first s ones, then those from a on, n in all.
struct Walk {
    int ctx, hi;        // context rows [0, ctx); rows behind the last token's
    int lo0, lo1;       // the window's first row of a token at depth 0 and T - 1
    int s, a, n;
    __device__ __forceinline__ int row0(int j) const { return TT * (j < s ? j : a + j - s); }
};
__device__ __forceinline__ int window_from(int pos0, int depth, int window) {
    if (window <= 0) return 0;
    const long long lo = (long long)pos0 + depth - window + 1;
    return lo < 0 ? 0 : lo > INT_MAX ? INT_MAX : (int)lo;
}
__device__ __forceinline__ Walk make_walk(int pos0, int T, const Sight& sight, int cap) {
    Walk w = {};
    if (pos0 < 0) return w;
    w.ctx = min(pos0, cap);
    w.hi = (int)min((long long)pos0 + T, (long long)cap);
    w.lo0 = window_from(pos0, 0, sight.window);
    w.lo1 = window_from(pos0, T - 1, sight.window);
    w.a = min(w.lo0, w.ctx) / TT;
    w.s = sight.window > 0 ? min((int)(((unsigned)min(sight.sinks, w.hi) + TT - 1) / TT), w.a) : 0;
    w.n = w.s + (w.hi + TT - 1) / TT - w.a;
    return w;
}

struct Parts {
    int2* meta;      // [B]: a cut sequence's first slot and its number of partials; 0: finished, -1: no rows
    float* pm;       // [slot][n_kv][R], log2 units
    float* pd;
    float* pacc;     // [slot][n_kv][R][256], unnormalised
};

// inclusive sum over the lanes 0 .. l (DPP row shifts, then the rows' totals)
__device__ __forceinline__ int lanes_sum(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, true);
    return x;
}

// A workgroup's run of its stream: runs are `per` units long, a sequence `cost` units and its tiles.
struct TreeRun {
    int run, per, u, u_end;   // u .. u_end: what is left
    int b, su, cost;          // the sequence that u lies in, and where it starts
    bool any;
    __device__ __forceinline__ TreeRun(const int* pos0, int B, int T, int run_, int runs, int run_min,
                                       const Sight& sight, int cap) {
        const int lane = threadIdx.x & 63;
        run = run_;
        cost = B > 1 ? SEQ_COST : 1;   // (not 0: a sequence without rows has its place too)
        auto units = [&](int s) { return make_walk(pos0[s], T, sight, cap).n + cost; };
        int total = 0, scan = 0, un = 0;   // (of the last 64 sequences: the first ones if B <= 64)
        for (int b0 = 0; b0 < B; b0 += 64) {
            un = b0 + lane < B ? units(b0 + lane) : 0;
            scan = lanes_sum(un);
            total += __builtin_amdgcn_readlane(scan, 63);
        }
        // (a little over total / runs: no run is left over)
        per = max((int)((float)total * (1.0001f / (float)runs)) + 1, run_min);
        any = (long long)run * per < total;
        if (!any) return;
        u = run * per;
        u_end = (int)min((long long)u + per, (long long)total);
        b = su = 0;
        for (int b0 = 0; b0 < B; b0 += 64) {
            if (B > 64) {
                un = b0 + lane < B ? units(b0 + lane) : 0;
                scan = lanes_sum(un);
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
};

__device__ const u32x4 zero_row[ROW_B / 16] = {};

// 8 bytes as the integers they are, exact in fp16: 1024 + (byte + 128) by its bits, less 1152
__device__ __forceinline__ f16x8 bytes_as_ints(uint32_t a, uint32_t b) {
    u32x4 r;
    const uint32_t ua = a ^ 0x80808080u, ub = b ^ 0x80808080u;
    r[0] = __builtin_amdgcn_perm(0x64646464u, ua, 0x04010400u);
    r[1] = __builtin_amdgcn_perm(0x64646464u, ua, 0x04030402u);
    r[2] = __builtin_amdgcn_perm(0x64646464u, ub, 0x04010400u);
    r[3] = __builtin_amdgcn_perm(0x64646464u, ub, 0x04030402u);
    return __builtin_bit_cast(f16x8, r) - (f16x8)((f16)1152.f);
}

// O^T lives in accumulation registers and is touched by the asm below alone: with the compiler's own
// MFMAs it got a second set of registers and was moved back on every tile. What the compiler cannot see
// in asm: an operand written by a VALU instruction right ahead of an MFMA needs two wait states (s_nop 1
// in front of each), and a result must have left the matrix pipeline before it is read (acc_settle).
// A spill of an accumulator would read it too early: there must be none.
__device__ __forceinline__ void acc_mfma(f32x4& acc, const f16x8& a, const f16x8& b) {
    asm("s_nop 1\n\tv_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(acc) : "v"(a), "v"(b));
}
__device__ __forceinline__ void acc_settle(f32x4 (&o)[16]) {
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7"
                 : "+a"(o[0]), "+a"(o[1]), "+a"(o[2]), "+a"(o[3]), "+a"(o[4]), "+a"(o[5]), "+a"(o[6]), "+a"(o[7]));
    asm volatile(""
                 : "+a"(o[8]), "+a"(o[9]), "+a"(o[10]), "+a"(o[11]), "+a"(o[12]), "+a"(o[13]), "+a"(o[14]),
                   "+a"(o[15]));
}
__device__ __forceinline__ void acc_scale(f32x4 (&o)[16], float c) {
    acc_settle(o);
#pragma unroll
    for (int n = 0; n < 16; ++n) {
        float x[4] = {o[n][0], o[n][1], o[n][2], o[n][3]}, t0, t1;
#pragma unroll
        for (int e = 0; e < 4; e += 2)
            asm volatile(
                "v_accvgpr_read_b32 %2, %0\n\t"
                "v_accvgpr_read_b32 %3, %1\n\t"
                "v_mul_f32 %2, %2, %4\n\t"
                "v_mul_f32 %3, %3, %4\n\t"
                "s_nop 2\n\t"
                "v_accvgpr_write_b32 %0, %2\n\t"
                "v_accvgpr_write_b32 %1, %3"
                : "+a"(x[e]), "+a"(x[e + 1]), "=&v"(t0), "=&v"(t1)
                : "v"(c));
        o[n] = (f32x4){x[0], x[1], x[2], x[3]};
    }
}

constexpr int STAGES_F16 = 4, AHEAD = STAGES_F16 - 1;   // tiles in LDS and copied ahead
constexpr int PLAN = 64;                                // tiles planned at a time
constexpr int KPF = 3, VPF = 3;                         // K and V^T operands read ahead of their products

// Over int8 pools a tile's bytes come to LDS as they are, RAW_AHEAD tiles ahead, a wave's rows of K, of
// V and their scales behind each other; the same wave turns them into rows of the fp16 stage, K as the
// integers they are and V as f16(byte scale), while the stage before it is in use.
constexpr int STAGES_Q8 = 2, RAW_STAGES = 4, RAW_AHEAD = RAW_STAGES - 1;
constexpr int RAW_ROW = PAGED_HD + 16;   // bytes a row and its scales
__device__ __forceinline__ void copy4_v(const char* vptr, uint32_t dst) {   // copy16_v, 4 bytes a lane
    asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(vptr), "{m0}"(dst));
}

// W waves, of which COPY only copy and convert tiles (0: the first ones do, beside their columns).
template <int W, bool Q8, int COPY = 0>
__global__ void __launch_bounds__(64 * W)
tree_attn_kernel(const f16* __restrict__ qg, int q_pitch, const char* __restrict__ kp,
                 const char* __restrict__ vp, const Pages pg, const int* __restrict__ pos0s,
                 const int* __restrict__ parents, int B, int T, int n_q, int n_kv, int groups, int runs,
                 int run_min, float sl2, const Sight sight, f16* __restrict__ z, int z_pitch, int gated,
                 const Parts parts) {
    constexpr int STAGES = Q8 ? STAGES_Q8 : STAGES_F16;
    constexpr int COLW = W - COPY;                            // waves with columns
    constexpr int CW = COPY ? COPY : W < 8 ? W : 8;           // waves that copy: C0 ..
    constexpr int C0 = COPY ? COLW : 0;
    constexpr int ROWS = TT / CW;                             // a copying wave's rows of a tile
    constexpr int RAW_WAVE = 2 * ROWS * RAW_ROW;
    constexpr int COPIES = Q8 ? ROWS / 2 + 1 : ROWS;          // its copy instructions a tile
    __shared__ __attribute__((aligned(16))) char s_tile[STAGES * STAGE_B];
    __shared__ __attribute__((aligned(16))) char s_raw[Q8 ? RAW_STAGES * CW * RAW_WAVE : 16];
    // the steps of K's blocks, [stage][block][row] (int8)
    __shared__ __attribute__((aligned(16))) float s_step[Q8 ? STAGES : 1][8][Q8 ? TT : 4];
    __shared__ uint2 s_line[TREE_MAX];   // a token's rows in sight, of the tree's
    __shared__ int s_lo[TREE_MAX];       // and the first of the context's
    // of 64 tiles and the next 64: the pool rows of their halves (of an absent page: row 0), the rows on
    // pages, those of them that some token sees, and the tiles that every token sees whole
    __shared__ int2 s_rows[2 * PLAN];
    __shared__ uint32_t s_here[2 * PLAN], s_seen[2 * PLAN];
    __shared__ uint64_t s_whole[2];
    const int tid = threadIdx.x, lane = tid & 63, w = uni(tid >> 6);
    const int col = lane & 15, g = lane >> 4, cw = w - C0;
    const bool copies = cw >= 0 && cw < CW;
    const int G = n_q / n_kv, R = T * G;
    const int cap = pg.max_pages << pg.shift;
    // Workgroups go to the 8 XCDs round-robin: the groups and kv heads of a run go to one of them, for
    // its L2 (the groups read the same rows), the runs to all.
    int hg, run_id;
    {
        const int id = blockIdx.x, n = n_kv * groups;
        const bool even = runs % 8 == 0;
        const int at = even ? id >> 3 : id;
        hg = at % n;
        run_id = even ? at / n * 8 + (id & 7) : at / n;
    }
    const int h = hg / groups, grp = hg - h * groups;
    TreeRun run(pos0s, B, T, run_id, runs, run_min, sight, cap);
    if (!run.any) return;   // (the whole workgroup)

    // this lane's query row: of token t, or none
    const int c0 = w < COLW ? (grp * COLW + w) * 16 : R, r_mine = c0 + col;
    const int t = r_mine < R ? r_mine / G : -1;
    const int qrow = r_mine < R ? t * n_q + h * G + r_mine - t * G : 0;
    const uint32_t rsb = (Q8 ? PAGED_HD : ROW_B) * n_kv;   // bytes a pool row
    const char* kb = uniform_ptr(kp + (size_t)h * (Q8 ? PAGED_HD : ROW_B));
    const char* vb = uniform_ptr(vp + (size_t)h * (Q8 ? PAGED_HD : ROW_B));
    const size_t values = ((size_t)pg.n_pages << pg.shift) * n_kv * PAGED_HD;   // ahead of the scales
    const uint32_t lds = (uint32_t)(uintptr_t)((__attribute__((address_space(3))) char*)s_tile);
    // K operand of k step ks: row col (+ 16), chunk 4 ks + g, at koff ^ 64 ks; V^T operand of dims 16 n ..:
    // this lane points at row 4 g + col / 4 (+ 16), dims 16 n + 4 (col % 4), at voff ^ 32 n (bit 8 of both
    // is not swizzled: an immediate)
    const uint32_t koff = col * ROW_B + 16 * (g ^ sw(col));
    const int vr = 4 * g + (col >> 2);
    const uint32_t voff = vr * ROW_B + 16 * ((col >> 1 & 1) ^ sw(vr)) + 8 * (col & 1);

    for (;;) {
        const int b = uni(run.b), pos0 = uni(pos0s[b]);
        const Walk walk = make_walk(pos0, T, sight, cap);
        const int cost = run.cost, eu = run.su + walk.n + cost;
        const int j0 = max(0, run.u - run.su - cost), j1 = max(0, min(run.u_end, eu) - run.su - cost);
        // pieces of a cut sequence: slot 2 r where a run's first piece, 2 r + 1 where another
        const bool whole_seq = j0 == 0 && j1 == walk.n;
        const int slot = 2 * run.run + (run.u != run.run * run.per);
        if (run.u == run.su && hg == 0 && tid == 0) {
            // (its first tile may be the first of the next run)
            const int first = (run.su + cost) / run.per, count = (eu - 1) / run.per - first + 1;
            parts.meta[b] = make_int2(2 * first + (run.su > first * run.per),
                                      walk.n == 0 ? -1 : count > 1 ? count : 0);
        }
        __syncthreads();   // (the last piece's reads of s_line, s_lo and the stages)
        // Q, ahead of the tree and the plan: a wait for it later would drain the copies
        f16x8 q[8];
        const f16* q_row = qg + ((size_t)b * T * n_q + qrow) * q_pitch + 8 * g;
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) q[ks] = t >= 0 ? *(const f16x8*)(q_row + 32 * ks) : (f16x8)(0);
        uint64_t present = 0;   // (wave 0's)
        // Tiles j0 + 64 c ..: a tile a lane of wave 0, so that the copies and masks of one cost no more than a
        // look at its entry (a page's lookup on the scalar unit, which a SIMD's waves share, held them all up).
        auto row_of = [&](int c) { return walk.row0(min(j0 + PLAN * c + lane, j1 - 1)); };
        auto ids_of = [&](int c) {   // (in the table, also behind its last page)
            const int *row = pg.table + (size_t)b * pg.stride, r0 = row_of(c), top = pg.max_pages - 1;
            return make_int2(row[min(r0 >> pg.shift, top)], row[min((r0 + 16) >> pg.shift, top)]);
        };
        auto plan = [&](int c, int2 ids) {
            const int r0 = row_of(c), at = PLAN * (c & 1) + lane;
            auto row = [&](int r, int id) {
                return r < cap && (unsigned)id < (unsigned)pg.n_pages
                           ? (id << pg.shift) + (r & ((1 << pg.shift) - 1)) : -1;
            };
            const int a = row(r0, ids.x), e = row(r0 + 16, ids.y);
            const uint32_t here = (a < 0 ? 0u : 0xFFFFu) | (e < 0 ? 0u : 0xFFFF0000u);
            uint32_t seen = low_bits(walk.ctx - r0) & (~low_bits(walk.lo0 - r0) | low_bits(sight.sinks - r0));
            const int d = r0 - pos0;   // of the tree's
            if (d > -TT && d < 64) seen |= (uint32_t)(d < 0 ? present << -d : present >> d) & low_bits(walk.hi - r0);
            s_rows[at] = make_int2(max(a, 0), max(e, 0));
            s_here[at] = here;
            s_seen[at] = seen & here;
            const uint64_t whole =
                __ballot(here == ~0u && r0 + TT <= walk.ctx && (r0 >= walk.lo1 || r0 + TT <= sight.sinks));
            if (lane == 0) s_whole[c & 1] = whole;
        };
        if (w == 0) {
            const int parent = parents[(size_t)b * T + min(lane, T - 1)];
            const int2 ids = j1 > j0 ? ids_of(0) : make_int2(0, 0);
            const Node node = tree_node<false>(parent, T);
            present = __ballot(node.here());
            // a path's tokens are numbered upwards: out of the window are its first ones, but those
            // that count as first rows of the sequence
            uint64_t line = (uint64_t)node.hi << 32 | node.lo, kept = 0;
            if (sight.window > 0) {
                const int depth = node.depth();
                uint64_t rest = line;
                for (int e = 0; __any(e <= depth - sight.window); ++e) {
                    const uint64_t bit = rest & -rest;
                    if (e <= depth - sight.window) {
                        if (pos0 < sight.sinks - e) kept |= bit;
                        rest &= ~bit;
                    }
                }
                line = rest | kept;
            }
            s_line[lane] = make_uint2((uint32_t)line, (uint32_t)(line >> 32));
            s_lo[lane] = node.here() ? window_from(pos0, node.depth(), sight.window) : INT_MAX;
            if (j1 > j0) plan(0, ids);
        }
        __syncthreads();
        // (a padded batch's waves without a token have no products; wave-uniform)
        const bool busy = __any(t >= 0 && s_lo[max(t, 0)] != INT_MAX);
        if (j1 > j0) {
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) {   // (beside O, as far as there is room at three waves a SIMD)
                if (ks < 5) asm volatile("" : "+a"(q[ks]));
                else asm volatile("" : "+v"(q[ks]));
            }
            f32x4 o[16];
#pragma unroll
            for (int n = 0; n < 16; ++n) {
                o[n] = (f32x4)(0.f);
                asm volatile("" : "+a"(o[n]));
            }
            float m_run = -1e30f, l_run = 0.f;
            auto tree_bits = [&](uint2 l, int r) {
                const int d = r - pos0;
                const uint64_t x = (uint64_t)l.y << 32 | l.x;
                return d <= -32 || d >= 64 ? 0u : (uint32_t)(d < 0 ? x << -d : x >> d);
            };
            uint64_t whole_bits = 0;
            // scores, softmax and product with V of tile j0 + j, in a stage
            auto tile = [&](int stage, int j) {
                if (!busy) return;
                if ((j & (PLAN - 1)) == 0) {
                    const uint64_t x = s_whole[j / PLAN & 1];
                    whole_bits = (uint64_t)(uint32_t)uni((int)(x >> 32)) << 32 | (uint32_t)uni((int)x);
                }
                uint32_t ko = koff, vo = voff;
                asm volatile("" : "+v"(ko), "+v"(vo));   // (its swizzled forms are not worth registers across tiles)
                auto k_frag = [&](int i) {   // k step i % 8 of rows 16 (i / 8) ..
                    return *(const f16x8*)(s_tile + stage * STAGE_B + (ko ^ (64 * (i & 3))) + 256 * (i >> 2 & 1) +
                                           16 * ROW_B * (i >> 3));
                };
                s16x4 vf[VPF][2];
                auto v_frag = [&](int n) {
                    const char* at = s_tile + stage * STAGE_B + TILE_B + (vo ^ (32 * (n & 7))) + 256 * (n >> 3);
                    vf[n % VPF][0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at);
                    vf[n % VPF][1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + 16 * ROW_B));
                };
                f32x4 s[2];
                f16x8 ka[KPF];
                // the two halves' products alternate: one's are a chain
                auto product = [&](int i, f32x4 c) {
                    return __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[i % KPF], q[i >> 1], c, 0, 0, 0);
                };
                auto frag_of = [](int i) { return (i & 1) << 3 | i >> 1; };
#pragma unroll
                for (int i = 0; i < KPF; ++i) ka[i] = k_frag(frag_of(i));
                if constexpr (Q8) {
                    // a k step is a block: its step goes onto its product, under the next one
                    f32x4 p[2], step[2];
                    auto block = [&](int i) {
                        step[i & 1] = *(const f32x4*)&s_step[stage][i >> 1][16 * (i & 1) + 4 * g];
                        p[i & 1] = product(i, (f32x4)(0.f));
                        if (i + KPF < 16) ka[i % KPF] = k_frag(frag_of(i + KPF));
                        __builtin_amdgcn_sched_barrier(0);
                    };
                    block(0);
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        if (i + 1 < 16) block(i + 1);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            s[i & 1][e] = i < 2 ? step[i & 1][e] * p[i & 1][e]
                                                : fmaf(step[i & 1][e], p[i & 1][e], s[i & 1][e]);
                        asm volatile("" : "+v"(s[i & 1]));   // (here: sunk behind the masks, all products would be held)
                        __builtin_amdgcn_sched_barrier(0);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        s[i & 1] = product(i, i < 2 ? (f32x4)(0.f) : s[i & 1]);
                        if (i + KPF < 16) ka[i % KPF] = k_frag(frag_of(i + KPF));
                        __builtin_amdgcn_sched_barrier(0);   // (keeps the reads ahead)
                    }
                }
#pragma unroll
                for (int n = 0; n < VPF; ++n) v_frag(n);
                __builtin_amdgcn_sched_barrier(0);
                if (!(whole_bits >> (j & (PLAN - 1)) & 1)) {   // (uniform)
                    int mine = t;
                    asm volatile("" : "+v"(mine));   // (nor are the entries' addresses)
                    const int lo = mine >= 0 ? s_lo[mine] : INT_MAX, r0 = walk.row0(j0 + j);
                    const uint2 line = mine >= 0 ? s_line[mine] : make_uint2(0, 0);
                    uint32_t see = low_bits(walk.ctx - r0) & (~low_bits(lo - r0) | low_bits(sight.sinks - r0));
                    see = lo == INT_MAX ? 0u : see | (tree_bits(line, r0) & low_bits(walk.hi - r0));
                    see = (see & s_here[j & (2 * PLAN - 1)]) >> (4 * g);
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        s[e >> 2][e & 3] = see & (1u << (16 * (e >> 2) + (e & 3))) ? s[e >> 2][e & 3] : -INFINITY;
                }
                f32x8 p;
                float sum;
                auto weights = [&] {
#pragma unroll
                    for (int e = 0; e < 8; ++e) p[e] = fast_exp2(fmaf(s[e >> 2][e & 3], sl2, -m_run));
                    sum = ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
                };
                weights();
                // A sum past 2^P_TOP: a score may be that far above the column's reference. On a piece's first
                // tile, rarely after, so the maximum is looked for only then.
                if (__any(sum > 32768.f)) {
                    float mt = s[0][0];
#pragma unroll
                    for (int e = 1; e < 8; ++e) mt = __builtin_elementwise_maximum(mt, s[e >> 2][e & 3]);
                    mt *= sl2;
                    mt = fmaxf(mt, lane_xor(mt, 16));
                    mt = pair32_max(mt);
                    const float m_new = mt > m_run + P_TOP ? mt - P_BELOW : m_run;
                    const float corr = fast_exp2(m_run - m_new);
                    m_run = m_new;
                    l_run *= corr;
                    if (j > 0) acc_scale(o, corr);   // (O is 0 till then)
                    weights();
                }
                l_run += sum;
                // Into the product with V in fp16, as in the decode: over fp16 pools one term (z 2.9e-4 off, 2.1e-4 of it
                // its own rounding; a second term, 2.1e-4, takes 343 us for 282, 4 trees of 63 on 20000 to 60000)
                const f16x8 p_hi = __builtin_convertvector(p, f16x8);
                f16x8 p_lo;
                if (Q8) p_lo = __builtin_convertvector(p - __builtin_convertvector(p_hi, f32x8), f16x8);
#pragma unroll
                for (int n = 0; n < 16; ++n) {
                    const f16x4 va = __builtin_bit_cast(f16x4, vf[n % VPF][0]);
                    const f16x4 vc = __builtin_bit_cast(f16x4, vf[n % VPF][1]);
                    const f16x8 a = {va[0], va[1], va[2], va[3], vc[0], vc[1], vc[2], vc[3]};
                    acc_mfma(o[n], a, p_hi);
                    if (Q8) acc_mfma(o[n], a, p_lo);
                    if (n + VPF < 16) v_frag(n + VPF);
                    __builtin_amdgcn_sched_barrier(0);
                }
            };
            const int n_tiles = j1 - j0;
            // a copying wave's entry of the tile that it copies next: its first row in the pool, and those of the
            // tile's rows that some token sees
            int e_row = 0;
            uint32_t e_seen = 0;
            auto look = [&](int j) {
                if (!copies) return;
                const int at = min(j, n_tiles - 1) & (2 * PLAN - 1);
                e_row = ROWS * cw >= 16 ? s_rows[at].y : s_rows[at].x;
                e_seen = s_seen[at];
            };
            auto pool_row = [&] { return (long long)uni(e_row) + (ROWS * cw & 15); };
            // between two tiles: the plan of the next 64
            auto ahead = [&](int j) {
                if (w == 0 && (j & (PLAN - 1)) == 0 && j + PLAN < n_tiles) plan(j / PLAN + 1, ids_of(j / PLAN + 1));
            };
            if constexpr (!Q8) {
                uint32_t loff[ROWS / 2];
#pragma unroll
                for (int n = 0; n < ROWS / 2; ++n) {
                    const int r = 2 * n + (lane >> 5);
                    loff[n] = r * rsb + 16 * ((lane & 31) ^ sw(ROWS * cw + r));
                }
                auto issue = [&](int j) {   // tile j0 + j, whose entry look() fetched
                    if (!copies) return;
                    const long long at = pool_row() * rsb;
                    const char *kr = uniform_ptr(kb + at), *vr = uniform_ptr(vb + at);
                    const uint32_t d0 = uni(lds + (j & 3) * STAGE_B + ROWS * cw * ROW_B);
                    // rows that no token sees may hold anything, and 0 x NaN is a NaN: zeros
                    const uint32_t on = (uint32_t)uni((int)e_seen) >> (ROWS * cw);
                    look(j + 1);
                    if ((on & ((1u << ROWS) - 1)) == (1u << ROWS) - 1) {
#pragma unroll
                        for (int n = 0; n < ROWS / 2; ++n) copy16(kr, loff[n], d0 + 2 * n * ROW_B);
#pragma unroll
                        for (int n = 0; n < ROWS / 2; ++n) copy16(vr, loff[n], d0 + TILE_B + 2 * n * ROW_B);
                    } else {
                        const char* zero = (const char*)zero_row + 16 * (lane & 31);
#pragma unroll
                        for (int n = 0; n < ROWS / 2; ++n) {
                            const bool ok = on >> (2 * n + (lane >> 5)) & 1;
                            copy16_v(ok ? kr + loff[n] : zero, d0 + 2 * n * ROW_B);
                            copy16_v(ok ? vr + loff[n] : zero, d0 + TILE_B + 2 * n * ROW_B);
                        }
                    }
                };
                look(0);
#pragma unroll 1
                for (int d = 0; d < min(AHEAD, n_tiles); ++d) issue(d);
                for (int j = 0; j < n_tiles; ++j) {
                    // tile j landed; those issued after it may still be in flight
                    const int later = min(AHEAD - 1, n_tiles - 1 - j);
                    if (later == 2) WAIT_VMCNT(2 * COPIES);
                    else if (later == 1) WAIT_VMCNT(COPIES);
                    else WAIT_VMCNT(0);
                    tile_done();   // every wave is past tile j - 1: its stage can be refilled
                    if (j + AHEAD < n_tiles) issue(j + AHEAD);
                    ahead(j);
                    tile(j & 3, j);
                }
            } else {
                const uint32_t raw0 =
                    (uint32_t)(uintptr_t)((__attribute__((address_space(3))) char*)s_raw) + cw * RAW_WAVE;
                auto issue = [&](int j) {   // tile j0 + j, whose entry look() fetched
                    if (!copies) return;
                    const long long at = pool_row();
                    look(j + 1);
                    int l = lane;
                    asm volatile("" : "+v"(l));   // (what follows is not worth registers across tiles)
                    const uint32_t xo = (l >> 4) * rsb + 16 * (l & 15);
                    // scales: a row's on 4 lanes, K's rows on the first 4 ROWS lanes, V's on the next
                    const uint32_t so = ((l >> 2) & (ROWS - 1)) * (rsb >> 4) + 4 * (l & 3);
                    const char *kr = uniform_ptr(kb + at * rsb), *vr = uniform_ptr(vb + at * rsb);
                    const uint32_t d0 = uni(raw0 + (j % RAW_STAGES) * (CW * RAW_WAVE));
#pragma unroll
                    for (int n = 0; n < ROWS / 4; ++n) {
                        copy16(kr, xo + 4 * n * rsb, d0 + 4 * n * PAGED_HD);
                        copy16(vr, xo + 4 * n * rsb, d0 + (ROWS + 4 * n) * PAGED_HD);
                    }
                    const char* scales = ((l & (4 * ROWS)) == 0 ? kp : vp) + values + (at * n_kv + h) * 16;
                    if (lane < 8 * ROWS) copy4_v(scales + so, d0 + 2 * ROWS * PAGED_HD);
                };
                auto convert = [&](int j) {   // this wave's rows of tile j0 + j to its stage
                    if (!copies) return;
                    const char* raw = s_raw + (j % RAW_STAGES) * (CW * RAW_WAVE) + cw * RAW_WAVE;
                    const uint32_t on = s_seen[j & (2 * PLAN - 1)];
                    const int stage = j & 1;
                    int l = lane;
                    asm volatile("" : "+v"(l));   // (as in issue)
                    const int g = l >> 4, col = l & 15;
#pragma unroll
                    for (int n = 0; n < ROWS / 4; ++n) {
                        const f16* sc = (const f16*)(raw + 2 * ROWS * PAGED_HD) + 8 * (4 * n + g) + (col >> 1);
                        const u32x4 kx = *(const u32x4*)(raw + 1024 * n + 16 * l);
                        const u32x4 vx = *(const u32x4*)(raw + ROWS * PAGED_HD + 1024 * n + 16 * l);
                        const f16 ks = sc[0], vs = sc[8 * ROWS];
                        const int r = ROWS * cw + 4 * n + g;
                        // rows that no token sees may hold any scale: theirs is 0
                        const f16 v = on >> r & 1 ? vs : (f16)0.f;
                        char* at = s_tile + stage * STAGE_B + r * ROW_B;
                        const int a0 = 16 * ((2 * col) ^ sw(r)), a1 = 16 * ((2 * col + 1) ^ sw(r));
                        auto values8 = [&](uint32_t x, uint32_t y) {
                            const f16x4 a = q8_deq4(x, (f16x2){v, v}), c = q8_deq4(y, (f16x2){v, v});
                            return (f16x8){a[0], a[1], a[2], a[3], c[0], c[1], c[2], c[3]};
                        };
                        *(f16x8*)(at + a0) = bytes_as_ints(kx.x, kx.y);
                        *(f16x8*)(at + a1) = bytes_as_ints(kx.z, kx.w);
                        *(f16x8*)(at + TILE_B + a0) = values8(vx.x, vx.y);
                        *(f16x8*)(at + TILE_B + a1) = values8(vx.z, vx.w);
                        if ((col & 1) == 0) s_step[stage][col >> 1][r] = (float)ks;
                    }
                };
                look(0);
#pragma unroll 1
                for (int d = 0; d < min(RAW_AHEAD, n_tiles); ++d) issue(d);
                auto landed = [&](int j) {   // tile j did; those issued after it may still be in flight
                    const int later = min(RAW_AHEAD - 1, n_tiles - 1 - j);
                    if (later == 2) WAIT_VMCNT(2 * COPIES);
                    else if (later == 1) WAIT_VMCNT(COPIES);
                    else WAIT_VMCNT(0);
                    asm volatile("" ::: "memory");
                };
                landed(0);
                convert(0);
                for (int j = 0; j < n_tiles; ++j) {
                    // stage j % 2 is written, and the other one done with
                    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
                    if (j + RAW_AHEAD < n_tiles) issue(j + RAW_AHEAD);
                    ahead(j);
                    tile(j & 1, j);
                    if (j + 1 < n_tiles) {
                        landed(j + 1);
                        convert(j + 1);
                    }
                }
            }
            if (c0 < R) {
                acc_settle(o);
                float l = l_run;
                l += lane_xor(l, 16);
                l = pair32_sum(l);
                if (t >= 0) {
                    // a place without a token, in tiles that all others see: its partial weighs nothing, whatever
                    // its q made of m (an infinite one would be the merge's maximum)
                    if (s_lo[t] == INT_MAX) l = 0.f, m_run = -1e30f;
                    if (!whole_seq) {
                        const size_t part = ((size_t)slot * n_kv + h) * R + r_mine;
                        float* dst = parts.pacc + part * PAGED_HD + 4 * g;
#pragma unroll
                        for (int n = 0; n < 16; ++n) *(f32x4*)(dst + 16 * n) = o[n];
                        if (g == 0) parts.pm[part] = m_run, parts.pd[part] = l;
                    } else {
                        const size_t rh = (size_t)b * T * n_q + qrow;
                        const f16* gate = qg + rh * q_pitch + PAGED_HD + 4 * g;
                        const float inv = 1.f / l;
#pragma unroll
                        for (int n = 0; n < 16; ++n) {
                            f32x4 v = o[n] * inv;
                            if (gated) {
                                const f16x4 gv = *(const f16x4*)(gate + 16 * n);
#pragma unroll
                                for (int e = 0; e < 4; ++e) v[e] *= fast_sigmoid((float)gv[e]);
                            }
                            // (no row seen: 0, whatever the gate holds)
                            *(f16x4*)(z + rh * z_pitch + 16 * n + 4 * g) = l == 0.f ? (f16x4)(0) : f16_sat4(v);
                        }
                    }
                }
            }
        }
        run.u = run.su = eu;
        ++run.b;
        if (run.u >= run.u_end) return;
    }
}

// z of the cut sequences' queries from their partials, and 0 where a sequence has no rows at all: a
// wave a (token, q head), lane l holding dims 4 l .. + 3, batches of partials whose loads are all
// issued before any is used.
constexpr int MERGE_BATCH = 4;
__global__ void __launch_bounds__(256)
tree_merge_kernel(const Parts in, f16* __restrict__ z, int z_pitch, const f16* __restrict__ gate, int g_pitch,
                  int T, int n_q, int n_kv, int n_rows) {
    const int lane = threadIdx.x & 63, rh = blockIdx.x * 4 + uni(threadIdx.x >> 6);
    if (rh >= n_rows) return;
    const int i = rh / n_q, head = rh - i * n_q, b = i / T, G = n_q / n_kv, h = head / G, R = T * G;
    const int2 meta = in.meta[b];
    f16* out = z + (size_t)rh * z_pitch + 4 * lane;
    if (meta.y <= 0) {
        if (meta.y < 0) *(f16x4*)out = (f16x4)(0);
        return;
    }
    f16x4 gv = (f16x4)(0);
    if (gate != nullptr) gv = *(const f16x4*)(gate + (size_t)rh * g_pitch + 4 * lane);
    const size_t row = (size_t)(i - b * T) * G + head - h * G;
    // its first piece's slot, then the first one of every further run
    auto at = [&](int s) { return ((size_t)(s == 0 ? meta.x : (meta.x >> 1) * 2 + 2 * s) * n_kv + h) * R + row; };
    f32x4 num = (f32x4)(0.f);
    float den = 0.f, M = -1e30f;
    for (int s = 0; s < meta.y; s += MERGE_BATCH) {
        float mv[MERGE_BATCH], dv[MERGE_BATCH];
        f32x4 av[MERGE_BATCH];
#pragma unroll
        for (int k = 0; k < MERGE_BATCH; ++k) {
            const size_t p = at(min(s + k, meta.y - 1));
            mv[k] = in.pm[p];
            dv[k] = in.pd[p];
            av[k] = *(const f32x4*)(in.pacc + p * PAGED_HD + 4 * lane);
        }
        float bm = M;
#pragma unroll
        for (int k = 0; k < MERGE_BATCH; ++k) {
            const bool ok = s + k < meta.y;
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
        for (int k = 0; k < MERGE_BATCH; ++k) {
            const float e = fast_exp2(mv[k] - M);
#pragma unroll
            for (int c = 0; c < 4; ++c) num[c] = fmaf(e, av[k][c], num[c]);
            den = fmaf(e, dv[k], den);
        }
    }
    const float inv = 1.f / den;
    f16x4 v;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const float x = num[c] * inv;
        v[c] = den == 0.f ? (f16)0.f : f16_sat(gate != nullptr ? x * fast_sigmoid((float)gv[c]) : x);
    }
    *(f16x4*)out = v;
}

// How a call is cut: groups of 16 `waves` columns, runs a kv head and group.
struct TreeCut {
    int waves, groups, runs, run_min;
};
// Waves, of 16 columns each: as many as share a tile's copies without more registers than there are. (4 of
// 63 on 20000 to 60000 rows: 287 us with twelve, 325 with eight; 96 columns on eight: 67 us, on twelve 75; 48 on
// four: 192, on eight 206.) Over int8 pools four more waves copy and convert where there is room for them (48
// columns on 16384 rows: 174 us, with waves that do both 227, with eight more 183; 96 on 8192: 73, 85). Of 193 to 256
// columns (two groups of twelve: 198 on 20000 rows 133 us, 192 in one group 107) two groups of eight were not timed.
TreeCut tree_cut(int T, int n_q, int n_kv) {
    const int R = T * (n_q / n_kv);
    TreeCut c;
    c.waves = R <= 64 ? 4 : R <= 128 ? 8 : 12;
    c.groups = (R + 16 * c.waves - 1) / (16 * c.waves);
    c.runs = std::max(1, cu_count() / (n_kv * c.groups));
    c.run_min = RUN_MIN;
    return c;
}

size_t tree_parts(int B, int T, int n_q, int runs, char* work, Parts& p) {
    const size_t rows = (size_t)2 * runs * T * n_q, m = up16((size_t)B * sizeof(int2)), f = up16(rows * 4);
    p = {(int2*)work, (float*)(work + m), (float*)(work + m + f), (float*)(work + m + 2 * f)};
    return m + 2 * f + rows * PAGED_HD * 4;
}

bool tree_sizes(int B, int T, int n_q, int n_kv, int head_dim) {
    return B >= 1 && B <= FL_PAGED_MAX_SEQS && T >= 1 && T <= FL_TREE_MAX && n_kv >= 1 && n_q >= 1 && n_q <= 4096 &&
           n_q % n_kv == 0 && head_dim == PAGED_HD;
}

}  // namespace

extern "C" {

size_t fl_attn_tree_paged_work_bytes(int B, int T, int n_q_heads, int n_kv_heads, int head_dim) {
    if (!tree_sizes(B, T, n_q_heads, n_kv_heads, head_dim)) return 0;
    Parts p;
    return tree_parts(B, T, n_q_heads, tree_cut(T, n_q_heads, n_kv_heads).runs, nullptr, p);
}

int fl_attn_tree_paged(const void* qg, int q_pitch, const void* kpool, const void* vpool, int q8, int n_pages,
                       int page_size, const int* pages, int max_pages, long long pages_stride, const int* pos0,
                       const int* parents, int B, int T, int n_q_heads, int n_kv_heads, int head_dim, float scale,
                       int window, int sinks, int gated, void* z, int z_pitch, void* work, size_t work_bytes,
                       fl_stream_t stream) {
    Pages pg;
    int rc = fl::make_pages(kpool, vpool, q8, n_pages, page_size, pages, max_pages, pages_stride, B, n_kv_heads,
                            head_dim, pg);
    if (rc) return rc;
    rc = check_heads(qg, q_pitch, z, z_pitch, gated, n_q_heads, n_kv_heads, scale, window, sinks);
    if (rc) return rc;
    FL_REQUIRE(pos0 && parents, "null pointer");
    FL_REQUIRE(tree_sizes(B, T, n_q_heads, n_kv_heads, head_dim), "1 <= T <= FL_TREE_MAX");
    // (tiles and starts of all sequences in 32 bits, with TreeRun's 1.0001)
    FL_REQUIRE((((long long)max_pages << pg.shift) / TT + 16) * B <= INT_MAX - INT_MAX / 1024,
               "B * max_pages * page_size < 0.999 * 2^36");
    const TreeCut cut = tree_cut(T, n_q_heads, n_kv_heads);
    Parts parts;
    if (tree_parts(B, T, n_q_heads, cut.runs, (char*)work, parts) > work_bytes || !work) {
        fl::set_error("work: smaller than fl_attn_tree_paged_work_bytes");
        return FL_ESCRATCH;
    }
    FL_REQUIRE(aligned16(work), "16-byte aligned work");
    const int rows = B * T * n_q_heads;
    const size_t need = tree_parts(B, T, n_q_heads, cut.runs, (char*)work, parts);
    const size_t pool = ((size_t)n_pages << pg.shift) * n_kv_heads * (q8 ? PAGED_HD + PAGED_HD / 16 : 2 * PAGED_HD);
    const RowsOf out = {z, (size_t)rows, 2 * (size_t)z_pitch, ROW_B};
    const RowsOf in = {qg, (size_t)rows, 2 * (size_t)q_pitch, (gated ? 2u : 1u) * ROW_B};
    auto clear_of = [&](const void* p, size_t n) { return !meet(z, out.bytes(), p, n) && !meet(work, need, p, n); };
    FL_REQUIRE(!meet(out, in) && !meet(work, need, qg, in.bytes()) && !meet(work, need, z, out.bytes()) &&
                   clear_of(kpool, pool) && clear_of(vpool, pool) && clear_of(pos0, 4 * (size_t)B) &&
                   clear_of(parents, 4 * (size_t)B * T) &&
                   clear_of(pages, 4 * ((B - 1) * (size_t)pages_stride + max_pages)),
               "z or work overlaps another buffer");
    const int copy = q8 && cut.waves < 12 ? 4 : 0;
    auto kernel = cut.waves == 4   ? (q8 ? tree_attn_kernel<8, true, 4> : tree_attn_kernel<4, false>)
                  : cut.waves == 8 ? (q8 ? tree_attn_kernel<12, true, 4> : tree_attn_kernel<8, false>)
                                   : (q8 ? tree_attn_kernel<12, true> : tree_attn_kernel<12, false>);
    hipLaunchKernelGGL(kernel, dim3(cut.runs * n_kv_heads * cut.groups), dim3(64 * (cut.waves + copy)), 0,
                       (hipStream_t)stream, (const f16*)qg, q_pitch, (const char*)kpool, (const char*)vpool, pg, pos0,
                       parents, B, T, n_q_heads, n_kv_heads, cut.groups, cut.runs, cut.run_min, scale * FL_LOG2E,
                       Sight{window, sinks}, (f16*)z, z_pitch, gated, parts);
    rc = fl::check_launch("attn_tree_paged");
    if (rc) return rc;
    hipLaunchKernelGGL(tree_merge_kernel, dim3((rows + 3) / 4), dim3(256), 0, (hipStream_t)stream, parts, (f16*)z,
                       z_pitch, gated ? (const f16*)qg + PAGED_HD : nullptr, q_pitch, T, n_q_heads, n_kv_heads, rows);
    return fl::check_launch("attn_tree_paged merge");
}

}  // extern "C"
