// Attention of trees of drafted tokens over the paged KV cache (attn_paged.hpp, tree.hpp).
//
// Token i of a sequence, at position p = pos0 + depth(i), sees the context's rows r < pos0 with
// r > p - window or r < sinks, and of the tree's rows pos0 + j those of its ancestors and its own
// whose position pos0 + depth(j) is in sight alike. The rest is the decode's:
//   z = f16_sat(sum_r e^(scale q.k_r - m) v_r / sum_r e^(scale q.k_r - m) * sigmoid(gate)).
//
// The T G query rows of a kv head are columns. A workgroup has 64 CB of them, 16 CB a wave, and
// walks tiles of 32 cache rows that its four waves share through LDS:
//   S^T (32 rows x 16 columns) = K Q^T        16x16x32 MFMAs, Q in registers
//   softmax                                   a lane holds column i's rows 4 g + e of both halves
//   O^T (256 dims x 16 columns) += V^T P^T    P as it lies: k slot (g, e) is row 4 g + e of half
//                                             e / 4; V^T by transposed LDS reads
// The tiles that the sequences' trees see make one stream a kv head and group of columns, cut into
// equal runs, one a workgroup, wherever the cuts fall; the runs are found from pos0 on the device, so
// that a captured call follows it. A sequence that lies in one run is finished there; a cut one leaves
// a partial a piece, which the merge weighs.
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
constexpr int W = 4;                    // waves
constexpr int MAX_CB = 2;
constexpr int RUN_MIN = 4;              // tiles a run, at least
constexpr int SEQ_COST = 2;             // a further piece's fixed cost in tiles

// the chunk swizzle of tile row r: 16-byte chunk c lies at c ^ sw(r)
__device__ __forceinline__ int sw(int r) { return ((r & 3) << 2) | ((r >> 2) & 3); }

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

constexpr int STAGES_F16 = 4, AHEAD = STAGES_F16 - 1;   // tiles in LDS and copied ahead
constexpr int COPIES = 8;                               // copy instructions a wave a tile
constexpr int STAGES_Q8 = 2;

// A wave's 8 rows of an int8 tile in flight: bytes [row 4 n + g][16 i .. + 15] of K and V, and the
// scales of those 16 dims' blocks.
struct Bytes {
    u32x4 k[2], v[2];
    f16 ks[2], vs[2];
};

template <int CB, bool Q8>
__global__ void __launch_bounds__(64 * W)
tree_attn_kernel(const f16* __restrict__ qg, int q_pitch, const char* __restrict__ kp,
                 const char* __restrict__ vp, const Pages pg, const int* __restrict__ pos0s,
                 const int* __restrict__ parents, int B, int T, int n_q, int n_kv, int groups, int runs,
                 int run_min, float sl2, const Sight sight, f16* __restrict__ z, int z_pitch, int gated,
                 const Parts parts) {
    constexpr int STAGES = Q8 ? STAGES_Q8 : STAGES_F16;
    __shared__ __attribute__((aligned(16))) char s_tile[STAGES * STAGE_B];
    // the steps of K's blocks, [stage][block][row] (int8)
    __shared__ __attribute__((aligned(16))) float s_step[Q8 ? STAGES : 1][8][Q8 ? TT : 4];
    __shared__ uint2 s_line[TREE_MAX];   // a token's rows in sight, of the tree's
    __shared__ int s_lo[TREE_MAX];       // and the first of the context's
    const int tid = threadIdx.x, lane = tid & 63, w = uni(tid >> 6);
    const int col = lane & 15, g = lane >> 4;
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

    // this lane's query rows: of token t[cb], or none
    int t[CB];
    size_t qrow[CB];
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
        const int r = (grp * W + w) * 16 * CB + 16 * cb + col;
        t[cb] = r < R ? r / G : -1;
        qrow[cb] = r < R ? (size_t)(r / G) * n_q + h * G + r % G : 0;
    }
    const bool busy = (grp * W + w) * 16 * CB < R;   // (wave-uniform)
    const uint32_t rsb = (Q8 ? PAGED_HD : ROW_B) * n_kv;   // bytes a pool row
    const char* kb = uniform_ptr(kp + (size_t)h * (Q8 ? PAGED_HD : ROW_B));
    const char* vb = uniform_ptr(vp + (size_t)h * (Q8 ? PAGED_HD : ROW_B));
    const size_t values = ((size_t)pg.n_pages << pg.shift) * n_kv * PAGED_HD;   // ahead of the scales
    const uint32_t lds = (uint32_t)(uintptr_t)((__attribute__((address_space(3))) char*)s_tile);
    // K operand of k step ks: row col (+ 16), chunk 4 ks + g, at koff ^ 64 ks; V^T operand of dims 16 n ..:
    // this lane points at row 4 g + col / 4 (+ 16), dims 16 n + 4 (col % 4), at voff ^ 32 n
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
        uint64_t present;
        {
            double none = 0.;
            const Node node = tree_node(parents + (size_t)b * T, T, none);   // (every wave)
            present = __ballot(node.here());
            if (w == 0) {
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
            }
        }
        __syncthreads();
        if (j1 > j0) {
            f16x8 q[CB][8];
            f32x4 o[CB][16];
            float m_run[CB], l_run[CB];
            int lo[CB];
            uint2 line[CB];
#pragma unroll
            for (int cb = 0; cb < CB; ++cb) {
                const f16* row = qg + ((size_t)b * T * n_q + qrow[cb]) * q_pitch + 8 * g;
#pragma unroll
                for (int ks = 0; ks < 8; ++ks) q[cb][ks] = t[cb] >= 0 ? *(const f16x8*)(row + 32 * ks) : (f16x8)(0);
#pragma unroll
                for (int n = 0; n < 16; ++n) o[cb][n] = (f32x4)(0.f);
                m_run[cb] = -1e30f, l_run[cb] = 0.f;
                lo[cb] = t[cb] >= 0 ? s_lo[t[cb]] : INT_MAX;
                line[cb] = t[cb] >= 0 ? s_line[t[cb]] : make_uint2(0, 0);
            }
            auto ids = page_ids(pg, b, j0, j1 - 1, 0, [&](int j) { return walk.row0(j); });
            // the rows of [r, r + 32) that some token sees, were their pages there
            auto seen_rows = [&](int r) {
                uint32_t m = low_bits(walk.ctx - r) & (~low_bits(walk.lo0 - r) | low_bits(sight.sinks - r));
                const int d = r - pos0;   // of the tree's
                if (d > -32 && d < 64) m |= (uint32_t)(d < 0 ? present << -d : present >> d) & low_bits(walk.hi - r);
                return m;
            };
            auto tree_bits = [&](uint2 l, int r) {
                const int d = r - pos0;
                const uint64_t x = (uint64_t)l.y << 32 | l.x;
                return d <= -32 || d >= 64 ? 0u : (uint32_t)(d < 0 ? x << -d : x >> d);
            };
            // scores, softmax and product with V of the tile at row r0 in a stage; here: rows on pages
            auto tile = [&](int stage, int r0, uint32_t here) {
                if (!busy) return;
                const char *kt = s_tile + stage * STAGE_B, *vt = kt + TILE_B;
                f32x4 s[CB][2];
#pragma unroll
                for (int rb = 0; rb < 2; ++rb) {
#pragma unroll
                    for (int cb = 0; cb < CB; ++cb) s[cb][rb] = (f32x4)(0.f);
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks) {
                        const f16x8 a = *(const f16x8*)(kt + 16 * rb * ROW_B + (koff ^ (64 * ks)));
                        if constexpr (Q8) {
                            const f32x4 step = *(const f32x4*)&s_step[stage][ks][16 * rb + 4 * g];
#pragma unroll
                            for (int cb = 0; cb < CB; ++cb) {
                                const f32x4 p = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, q[cb][ks], (f32x4)(0.f), 0, 0, 0);
#pragma unroll
                                for (int e = 0; e < 4; ++e) s[cb][rb][e] = fmaf(step[e], p[e], s[cb][rb][e]);
                            }
                        } else {
#pragma unroll
                            for (int cb = 0; cb < CB; ++cb)
                                s[cb][rb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, q[cb][ks], s[cb][rb], 0, 0, 0);
                        }
                    }
                }
                // whole: every token sees every row (uniform)
                const bool whole = here == ~0u && r0 + TT <= walk.ctx && (r0 >= walk.lo1 || r0 + TT <= sight.sinks);
                f16x8 p_hi[CB], p_lo[CB];
#pragma unroll
                for (int cb = 0; cb < CB; ++cb) {
                    float x[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = s[cb][e >> 2][e & 3];
                    if (!whole) {
                        uint32_t see = low_bits(walk.ctx - r0) & (~low_bits(lo[cb] - r0) | low_bits(sight.sinks - r0));
                        see = lo[cb] == INT_MAX ? 0u : here & (see | (tree_bits(line[cb], r0) & low_bits(walk.hi - r0)));
                        see >>= 4 * g;
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[e] = see & (1u << (16 * (e >> 2) + (e & 3))) ? x[e] : -INFINITY;
                    }
                    float mt = x[0];
#pragma unroll
                    for (int e = 1; e < 8; ++e) mt = __builtin_elementwise_maximum(mt, x[e]);
                    mt *= sl2;
                    if (__any(mt > m_run[cb] + P_TOP)) {
                        mt = fmaxf(mt, lane_xor(mt, 16));
                        mt = pair32_max(mt);
                        const float m_new = mt > m_run[cb] + P_TOP ? mt - P_BELOW : m_run[cb];
                        const float corr = fast_exp2(m_run[cb] - m_new);
                        m_run[cb] = m_new;
                        l_run[cb] *= corr;
#pragma unroll
                        for (int n = 0; n < 16; ++n) o[cb][n] *= corr;
                    }
                    f32x8 p;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        p[e] = fast_exp2(fmaf(x[e], sl2, -m_run[cb]));
                        l_run[cb] += p[e];
                    }
                    p_hi[cb] = __builtin_convertvector(p, f16x8);
                    if (Q8) p_lo[cb] = __builtin_convertvector(p - __builtin_convertvector(p_hi[cb], f32x8), f16x8);
                }
#pragma unroll
                for (int n = 0; n < 16; ++n) {
                    const char* at = vt + (voff ^ (32 * n));
                    const f16x4 va = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at));
                    const f16x4 vc = __builtin_bit_cast(
                        f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + 16 * ROW_B)));
                    const f16x8 a = {va[0], va[1], va[2], va[3], vc[0], vc[1], vc[2], vc[3]};
#pragma unroll
                    for (int cb = 0; cb < CB; ++cb) {
                        o[cb][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, p_hi[cb], o[cb][n], 0, 0, 0);
                        if (Q8) o[cb][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, p_lo[cb], o[cb][n], 0, 0, 0);
                    }
                }
            };
            const int n_tiles = j1 - j0;
            auto pages_here = [](int id0, int id1) { return (id0 < 0 ? 0u : 0xFFFFu) | (id1 < 0 ? 0u : 0xFFFF0000u); };
            // the pool row of this wave's first row of a tile (of an absent page: page 0's)
            auto pool_row = [&](int r0, int id0, int id1) {
                const int id = w >> 1 ? id1 : id0;
                return ((long long)max(id, 0) << pg.shift) + ((r0 + 8 * w) & ((1 << pg.shift) - 1));
            };
            if constexpr (!Q8) {
                uint32_t loff[4];
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const int r = 2 * n + (lane >> 5);
                    loff[n] = r * rsb + 16 * ((lane & 31) ^ sw(8 * w + r));
                }
                auto issue = [&](int stage, int j, uint32_t& here) {
                    int id0, id1;
                    ids.at(j, id0, id1);
                    const int r0 = walk.row0(j);
                    here = pages_here(id0, id1);
                    const long long at = pool_row(r0, id0, id1) * rsb;
                    const char *kr = uniform_ptr(kb + at), *vr = uniform_ptr(vb + at);
                    const uint32_t d0 = uni(lds + stage * STAGE_B + 8 * w * ROW_B);
                    // rows that no token sees may hold anything, and 0 x NaN is a NaN: zeros
                    const uint32_t on = (seen_rows(r0) & here) >> (8 * w) & 0xFF;
                    if (on == 0xFF) {
#pragma unroll
                        for (int n = 0; n < 4; ++n) copy16(kr, loff[n], d0 + 2 * n * ROW_B);
#pragma unroll
                        for (int n = 0; n < 4; ++n) copy16(vr, loff[n], d0 + TILE_B + 2 * n * ROW_B);
                    } else {
                        const char* zero = (const char*)zero_row + 16 * (lane & 31);
#pragma unroll
                        for (int n = 0; n < 4; ++n) {
                            const bool ok = on >> (2 * n + (lane >> 5)) & 1;
                            copy16_v(ok ? kr + loff[n] : zero, d0 + 2 * n * ROW_B);
                            copy16_v(ok ? vr + loff[n] : zero, d0 + TILE_B + 2 * n * ROW_B);
                        }
                    }
                };
                uint32_t here[STAGES_F16] = {};
#pragma unroll
                for (int d = 0; d < AHEAD; ++d)
                    if (d < n_tiles) issue(d, j0 + d, here[d]);
                int st = 0;
                for (int j = 0; j < n_tiles; ++j) {
                    // tile j landed; those issued after it may still be in flight
                    const int later = min(AHEAD - 1, n_tiles - 1 - j);
                    if (later == 2) WAIT_VMCNT(2 * COPIES);
                    else if (later == 1) WAIT_VMCNT(COPIES);
                    else WAIT_VMCNT(0);
                    tile_done();   // every wave is past tile j - 1: its stage can be refilled
                    const uint32_t now = here[0];
                    here[0] = here[1], here[1] = here[2];
                    if (j + AHEAD < n_tiles) issue(st == 0 ? STAGES_F16 - 1 : st - 1, j0 + j + AHEAD, here[2]);
                    tile(st, walk.row0(j0 + j), now);
                    st = st == STAGES_F16 - 1 ? 0 : st + 1;
                }
            } else {
                const uint32_t xo = g * rsb + 16 * col, so = (g * rsb >> 4) + (col & ~1);
                auto load = [&](Bytes& x, int j, uint32_t& here) {
                    int id0, id1;
                    ids.at(j, id0, id1);
                    here = pages_here(id0, id1);
                    const long long at = pool_row(walk.row0(j), id0, id1);
                    const gptr k0 = uni_global(kb + at * rsb), v0 = uni_global(vb + at * rsb);
                    const gptr k1 = uni_global(kp + values + (at * n_kv + h) * 16), v1 = uni_global(vp + values + (at * n_kv + h) * 16);
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        x.k[n] = load_g<u32x4>(k0, xo + 4 * n * rsb);
                        x.v[n] = load_g<u32x4>(v0, xo + 4 * n * rsb);
                        x.ks[n] = load_g<f16>(k1, so + 4 * n * (rsb >> 4));
                        x.vs[n] = load_g<f16>(v1, so + 4 * n * (rsb >> 4));
                    }
                };
                auto put = [&](const Bytes& x, int stage, int r0, uint32_t here) {
                    const uint32_t on = seen_rows(r0) & here;
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        const int r = 8 * w + 4 * n + g;
                        // rows that no token sees may hold any scale: theirs is 0
                        const bool ok = on >> r & 1;
                        const f16 vs = ok ? x.vs[n] : (f16)0.f;
                        char* at = s_tile + stage * STAGE_B + r * ROW_B;
                        const int c0 = 16 * ((2 * col) ^ sw(r)), c1 = 16 * ((2 * col + 1) ^ sw(r));
                        *(f16x8*)(at + c0) = bytes_as_ints(x.k[n].x, x.k[n].y);
                        *(f16x8*)(at + c1) = bytes_as_ints(x.k[n].z, x.k[n].w);
                        const f16x4 a = q8_deq4(x.v[n].x, (f16x2){vs, vs}), c = q8_deq4(x.v[n].y, (f16x2){vs, vs});
                        const f16x4 e = q8_deq4(x.v[n].z, (f16x2){vs, vs}), f = q8_deq4(x.v[n].w, (f16x2){vs, vs});
                        *(f16x8*)(at + TILE_B + c0) = (f16x8){a[0], a[1], a[2], a[3], c[0], c[1], c[2], c[3]};
                        *(f16x8*)(at + TILE_B + c1) = (f16x8){e[0], e[1], e[2], e[3], f[0], f[1], f[2], f[3]};
                        if ((col & 1) == 0) s_step[stage][col >> 1][r] = (float)x.ks[n];
                    }
                };
                Bytes x[2];
                uint32_t here[2];
                load(x[0], j0, here[0]);
                put(x[0], 0, walk.row0(j0), here[0]);
                uint32_t now = here[0];
                load(x[0], min(j0 + 1, j1 - 1), here[0]);
                load(x[1], min(j0 + 2, j1 - 1), here[1]);
                __syncthreads();
                auto body = [&](int j, int buf) {
                    tile(j & 1, walk.row0(j0 + j), now);
                    if (j + 1 < n_tiles) {
                        put(x[buf], (j + 1) & 1, walk.row0(j0 + j + 1), here[buf]);
                        now = here[buf];
                        load(x[buf], min(j0 + j + 3, j1 - 1), here[buf]);
                    }
                    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
                };
                for (int j = 0; j < n_tiles; j += 2) {
                    body(j, 0);
                    if (j + 1 < n_tiles) body(j + 1, 1);
                }
            }
            if (busy) {
#pragma unroll
                for (int cb = 0; cb < CB; ++cb) {
                    float l = l_run[cb];
                    l += lane_xor(l, 16);
                    l = pair32_sum(l);
                    if (t[cb] < 0) continue;
                    if (lo[cb] == INT_MAX) l = 0.f;   // (a place without a token, in tiles that all others see)
                    const int r = (grp * W + w) * 16 * CB + 16 * cb + col;
                    if (!whole_seq) {
                        const size_t part = ((size_t)slot * n_kv + h) * R + r;
                        float* dst = parts.pacc + part * PAGED_HD + 4 * g;
#pragma unroll
                        for (int n = 0; n < 16; ++n) *(f32x4*)(dst + 16 * n) = o[cb][n];
                        if (g == 0) parts.pm[part] = m_run[cb], parts.pd[part] = l;
                        continue;
                    }
                    const size_t rh = (size_t)b * T * n_q + qrow[cb];
                    const f16* gate = qg + rh * q_pitch + PAGED_HD + 4 * g;
                    const float inv = 1.f / l;
#pragma unroll
                    for (int n = 0; n < 16; ++n) {
                        f32x4 v = o[cb][n] * inv;
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

// How a call is cut: groups of 64 CB columns, runs a kv head and group.
struct TreeCut {
    int cb, groups, runs, run_min;
};
TreeCut tree_cut(int T, int n_q, int n_kv) {
    const int R = T * (n_q / n_kv);
    TreeCut c;
    c.groups = (R + 64 * MAX_CB - 1) / (64 * MAX_CB);
    c.cb = ((R + c.groups - 1) / c.groups + 63) / 64;
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
    FL_REQUIRE((((long long)max_pages << pg.shift) / TT + 8) * B < INT_MAX, "B * max_pages * page_size < 2^36");
    const TreeCut cut = tree_cut(T, n_q_heads, n_kv_heads);
    Parts parts;
    if (tree_parts(B, T, n_q_heads, cut.runs, (char*)work, parts) > work_bytes || !work) {
        fl::set_error("work: smaller than fl_attn_tree_paged_work_bytes");
        return FL_ESCRATCH;
    }
    FL_REQUIRE(aligned16(work), "16-byte aligned work");
    auto kernel = cut.cb == 1 ? (q8 ? tree_attn_kernel<1, true> : tree_attn_kernel<1, false>)
                              : (q8 ? tree_attn_kernel<2, true> : tree_attn_kernel<2, false>);
    hipLaunchKernelGGL(kernel, dim3(cut.runs * n_kv_heads * cut.groups), dim3(64 * W), 0, (hipStream_t)stream,
                       (const f16*)qg, q_pitch, (const char*)kpool, (const char*)vpool, pg, pos0, parents, B, T,
                       n_q_heads, n_kv_heads, cut.groups, cut.runs, cut.run_min, scale * FL_LOG2E,
                       Sight{window, sinks}, (f16*)z, z_pitch, gated, parts);
    rc = fl::check_launch("attn_tree_paged");
    if (rc) return rc;
    const int rows = B * T * n_q_heads;
    hipLaunchKernelGGL(tree_merge_kernel, dim3((rows + 3) / 4), dim3(256), 0, (hipStream_t)stream, parts, (f16*)z,
                       z_pitch, gated ? (const f16*)qg + PAGED_HD : nullptr, q_pitch, T, n_q_heads, n_kv_heads, rows);
    return fl::check_launch("attn_tree_paged merge");
}

}  // extern "C"
