// The Gated DeltaNet layer over a tree of drafted tokens, and the state behind an accepted
// path.
//
// A token's conv window, decay and state follow its path through the tree, from the sequence's
// state S0 [V][K] (never written here) and conv frames. With alpha_i the decay, beta_i the rate,
// G_i the product of the alphas on the path to i (itself included), S_p the state of i's parent:
//   S_i = alpha_i S_p + u_i k_i^T,   u_i = beta_i (v_i - alpha_i S_p k_i),   o_i = s S_i q_i.
// Unrolled over the path, with j < i its ancestors (parents come before their children):
//   u_i = beta_i (v_i - G_i S0 k_i - sum_{j anc i} (G_i / G_j) (k_i . k_j) u_j)
//   o_i = s (G_i S0 q_i + sum_{j anc-or-self i} (G_i / G_j) (q_i . k_j) u_j),
// so no token's state is ever formed: the first line is (I + A) U = R with A strictly lower
// triangular, both need S0 only in products with all k_i and q_i. y_i is rmsnorm_gated of o_i.
// Everything is held in fp32 (fp64: the sums of log alpha, whose differences are the logarithms of
// G_i / G_j) and y is rounded once, where gdn_decode_normed rounds the conv's output, q, k and o to
// fp16 as the reference does. The operands of the products with S0 and among keys are two scaled fp16
// terms each, 22 bits: three 16x16x32 MFMAs of 16 clocks take the place of eight fp32 ones of 32. Their
// scales are a row's of S0 and a constant (|q|, |k| <= 1). The system's products are in fp32: a scale
// that tokens share would cost a small one its bits beside a large one that is not on its path.
//
// A workgroup has the v heads of a k head, up to three: their q, k and products are formed once. A wave
// has 16 or 32 of a head's state rows as the B operand, a row a column; the accumulators (register e of lane
// (g, c) is token 4 g + e of column c) are in turn B operands of the products with A and the q.k side,
// whose k slot g of step e is token 4 g + e. The 16-row diagonal blocks of I + A are inverted by
// substitution, a column a lane.
//
// Measured, from a graph, 16 k and 48 v heads: a tree of 16 8.2 us, 4 of 37 14.7, 16 of 16 16.4, 16 of 9 to 37
// 28.5, 8 of 64 34.9 us; a path of 4 committed 5.2 us, 16 of 7 22.3 us (4.5 TB/s of states read and written). The
// trees are bound by a workgroup's chain of phases, each between two barriers: of 43000 clocks (3 heads, 9 to 37
// tokens) 14000 until the tokens' rows are here and half of S0 is on its way, 9000 the conv, 2700 A and the q.k
// side, 9300 the products with S0, 2400 the system, 5600 the norm and the stores; VALU instructions are a fifth of
// it, MFMAs a tenth. S0's 50 MB alone would be 10 us.
#include "tree.hpp"

#include "gdn_gates.hpp"

#include <math.h>

namespace {

typedef float f32x8 __attribute__((ext_vector_type(8)));

constexpr int GT_K = 128;                // K = V
constexpr int ROW_H = GT_K + 8;          // terms a row of k and q
constexpr float QK_SCALE = 16384.f;      // of q and k, whose norms are at most 1
// Heads up to which a workgroup takes one, with 16 state rows a wave: a round of workgroups is the shorter one
// then (240 heads of 16 tokens 8.7 us, by threes 14.0; of 37 tokens 15.2 and 26.0), several are not (288 heads of 37
// tokens 27.9 and 26.2; 768 heads of 16 18.4 and 16.6, of 9 to 37 33.3 and 28.8) unless little LDS lets a CU have
// two at a time (288 heads of 16 tokens 12.4 and 14.2, which this number leaves at 14.2).
constexpr int GT_MANY = 256;
// State rows that a workgroup moves on (measured with the conv's input in registers yet, 16, 32, 64 and 128
// rows: 16 paths of 7 25.9, 26.9, 28.4 and 28.4 us; 2 of 40 16.0, 14.7, 13.4 and 18.8; one of 4 6.1, 6.2, 6.8, 8.2)
constexpr int GC_ROWS = 32;
constexpr int BLOCK_P = 20;              // floats a row of a 16 x 16 block

// Sum over the 16 lanes of a DPP row, on every one of them.
__device__ __forceinline__ float row16_sum(float v) {
    v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x128, 0xF, 0xF, true));   // row_ror 8
    v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x124, 0xF, 0xF, true));
    v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x122, 0xF, 0xF, true));
    v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x121, 0xF, 0xF, true));
    return v;
}

// log alpha, in (-1000, 0]: past that e^x is 0 in fp32 anyway, and differences of sums of these
// stay exact in fp64.
__device__ __forceinline__ float log_decay(float a_dt, float A) {
    const float sp = a_dt <= 20.f ? log1p_pos(hw_expf(a_dt)) : a_dt;
    const float l = -hw_expf(A) * sp;
    return l < -1000.f ? -1000.f : l;
}
// The product of the decays of which x is such a sum, or a difference of two, in log2 units
__device__ __forceinline__ float decayed(double x) { return fast_exp2((float)x); }

// Eight channels' conv: their taps, a channel's newest last.
struct Taps8 {
    f16x8 t[4];   // of two channels each
    __device__ __forceinline__ void load(const f16* conv_w, int ch) {
        const f16x8* w = (const f16x8*)(conv_w + 4 * ch);
        t[0] = w[0], t[1] = w[1], t[2] = w[2], t[3] = w[3];
    }
    // silu of the taps over x0 (the token's) and the three before it
    __device__ __forceinline__ void apply(f32x4& lo, f32x4& hi, f16x8 x3, f16x8 x2, f16x8 x1, f16x8 x0) {
        // (a mixed fma takes its halves as they are: they are neither converted here nor ahead of a loop)
        float zero = 0.f;
        asm("" : "+v"(t[0]), "+v"(t[1]), "+v"(t[2]), "+v"(t[3]), "+v"(zero));
        auto y = [&](int i) {
            const f16x8 w = t[i >> 1];
            const int at = 4 * (i & 1);
            float s = fmaf((float)w[at], (float)x3[i], zero);
            s = fmaf((float)w[at + 1], (float)x2[i], s);
            s = fmaf((float)w[at + 2], (float)x1[i], s);
            s = fmaf((float)w[at + 3], (float)x0[i], s);
            return s * __builtin_amdgcn_rcpf(1.f + hw_expf(-s));
        };
        lo = (f32x4){y(0), y(1), y(2), y(3)};
        hi = (f32x4){y(4), y(5), y(6), y(7)};
    }
};
// The sequence's last three frames ([channel][frame], oldest first; zero for a fresh sequence).
struct Frames8 {
    f16x8 f0, f1, f2;
    __device__ __forceinline__ void load(const f16* frames, bool fresh, int ch) {
        const f16x8* x = (const f16x8*)(frames + 3 * ch);
        const f16x8 x0 = x[0], x1 = x[1], x2 = x[2];
        f0 = (f16x8){x0[0], x0[3], x0[6], x1[1], x1[4], x1[7], x2[2], x2[5]};
        f1 = (f16x8){x0[1], x0[4], x0[7], x1[2], x1[5], x2[0], x2[3], x2[6]};
        f2 = (f16x8){x0[2], x0[5], x1[0], x1[3], x1[6], x2[1], x2[4], x2[7]};
        if (fresh) f0 = f1 = f2 = (f16x8)(0);
    }
};
// The row at `row`, or the frame n > 0 tokens ahead of a path's first: n = 1 is the newest. (By
// value: with the frames behind a reference the choice becomes one of addresses, in scratch.)
__device__ __forceinline__ f16x8 token(int n, const f16* row, f16x8 f0, f16x8 f1, f16x8 f2) {
    f16x8 r = n == 1 ? f2 : n == 2 ? f1 : f0;
    if (n <= 0) r = *(const f16x8*)row;
    return r;
}
__device__ __forceinline__ float sum_sq(f32x4 a, f32x4 b) {
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) s = fmaf(a[e], a[e], fmaf(b[e], b[e], s));
    return s;
}

struct TreeSeqs {
    const float* S[FL_MAX_SEQS];
    const f16* frames[FL_MAX_SEQS];
    int pos0[FL_MAX_SEQS];
};

__device__ __forceinline__ int ilogb_bits(float x) { return (int)(__float_as_uint(x) >> 23 & 255) - 127; }
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
// x s as two fp16 terms: 22 bits of it, down to 2^-24 (so s scales up). Two mixed fmas a number.
struct Terms {
    f16x8 hi, lo;
};
__device__ __forceinline__ Terms split8(f32x8 x, float s) {
    Terms r;
#pragma unroll
    for (int e = 0; e < 8; ++e) r.hi[e] = (f16)fmaf(x[e], s, 0.f);
    asm("" : "+v"(r.hi));   // (as it is packed: it would be formed twice)
#pragma unroll
    for (int e = 0; e < 8; ++e) r.lo[e] = (f16)fmaf(x[e], s, -(float)r.hi[e]);
    return r;
}
// The exponent that brings the largest of a column's entries to [2^14, 2^15) (to less where all are below
// 2^-98): the four lanes of a column have some each, the largest of which is `top`.
__device__ __forceinline__ int lift(float top) {
    top = fmaxf(top, lane_xor(top, 16));
    top = pair32_max(top);
    return 14 - min(max(ilogb_bits(top), -98), 127);
}
// c + a b for a 16 x 16 block: this lane has a's row `col`, columns 4 g .. + 3, and b's rows 4 g .. + 3.
__device__ __forceinline__ f32x4 mfma_block(f32x4 a, f32x4 b, f32x4 c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
}
// c + a b without the product of the two low terms (2^-22 of a b)
__device__ __forceinline__ f32x4 mfma_terms(const Terms& a, const Terms& b, f32x4 c) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.lo, b.hi, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.hi, b.lo, c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a.hi, b.hi, c, 0, 0, 0);
}
// What a wave wrote to LDS for itself, in another order.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// NB blocks of 16 tokens, HP v heads of one k head, TL tiles of 16 state rows a wave.
template <int NB, int HP, int TL>
__global__ void __launch_bounds__(512 * HP / TL)
gdn_tree_kernel(const f16* __restrict__ x, int x_stride, const f16* __restrict__ conv_w, const TreeSeqs seqs,
                const int* __restrict__ parents, const float* __restrict__ ga, const float* __restrict__ gb,
                int ab_stride, const float* __restrict__ A_log, const float* __restrict__ dt_bias,
                const f16* __restrict__ z, int z_pitch, const float* __restrict__ norm_w,
                f16* __restrict__ y, int y_pitch, int T, int n_kheads, int n_vheads, float out_scale,
                float l2eps, float norm_eps) {
    constexpr int HW = 8 / TL, WAVES = HP * HW, THREADS = 64 * WAVES;   // a head's waves
    constexpr int TP = 16 * NB, BLOCKS = NB * (NB + 1) / 2;
    constexpr int COLS = 16 * TL;                       // a wave's state rows
    constexpr int LT = 64 / (2 * TL), VR = (TP + LT - 1) / LT;   // its tokens at a time, 8 columns a lane
    constexpr int QT = THREADS / 32, QR = (TP + QT - 1) / QT;    // all waves' tokens of q and k at a time
    constexpr int RAW_P = COLS + 8, OUT_P = COLS + 4, OUT_ROWS = LT < TP ? LT : TP;
    constexpr int OWN_B = 4 * OUT_ROWS * OUT_P > 2 * (TP + 3) * RAW_P ? 4 * OUT_ROWS * OUT_P : 2 * (TP + 3) * RAW_P;
    typedef f16 Rows[TP][ROW_H];
    // (transposed while it waits to be inverted)
    typedef float Block[16][BLOCK_P];
    constexpr int MATS_B = 2 * HP * BLOCKS * sizeof(Block);
    constexpr int RAW_ROWS = TP + 3, RAW_B = 2 * RAW_ROWS * ROW_H * sizeof(f16);
    __shared__ __attribute__((aligned(16))) Rows s_q[2], s_k[2];   // hi, lo
    // q's and k's input rows behind three frames, then the heads' -A (inverses of I + A on the diagonal)
    // and q.k sides
    __shared__ __attribute__((aligned(16))) char s_mats[MATS_B > RAW_B ? MATS_B : RAW_B];
    // a wave's own: its columns' frames and input rows, later v and o on the way between two layouts
    __shared__ __attribute__((aligned(16))) char s_own[WAVES][OWN_B];
    __shared__ __attribute__((aligned(16))) float s_ss[HP][TP][HW];
    __shared__ double s_log[HP][64];
    __shared__ __attribute__((aligned(16))) float s_beta[HP][64], s_gain[HP][64];
    __shared__ uint2 s_line[64];
    __shared__ int4 s_up[64];            // the rows of the three tokens before it on its path; here
    __shared__ int s_n;
    auto s_raw = (f16(*)[RAW_ROWS][ROW_H])s_mats;
    auto s_a = (Block(*)[BLOCKS])s_mats, s_p = s_a + HP;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, g = lane >> 4;
    // Workgroups go to the 8 XCDs round-robin: neighbouring heads to one of them.
    const int group = n_vheads / n_kheads, units = n_vheads / HP;
    int at = blockIdx.x % units, b = blockIdx.x / units;
    if (units % 8 == 0) {
        const int per = units / 8, r = blockIdx.x >> 3;
        at = (blockIdx.x & 7) * per + r % per;
        b = r / per;
    }
    const int h = w / HW, hv = at * HP + h, hk = at * HP / group;   // the wave's head
    const int c0 = (w - h * HW) * COLS;                                 // and first state row
    const bool fresh = seqs.pos0[b] == 0;

    // Asked for first: what the tokens' conv needs. S0, which takes longest, follows once that is here.
    int parent = -2;
    float a_in = 0.f, b_in = 0.f, dt = 0.f, A = 0.f;
    if (w < HP) {   // the gates of head w
        const size_t token = (size_t)b * T + min(lane, T - 1);
        const int head = at * HP + w;
        parent = parents[token];
        a_in = ga[token * ab_stride + head], b_in = gb[token * ab_stride + head];
        dt = dt_bias[head], A = A_log[head];
    }
    const f16* xb = x + (size_t)b * T * x_stride;
    const int part = tid >> 4 & 1, ch8 = 8 * (tid & 15), v8 = 8 * (lane & (2 * TL - 1));
    const int ch_qk = (part == 0 ? hk : n_kheads + hk) * GT_K + ch8;
    const int ch_v = (2 * n_kheads + hv) * GT_K + c0 + v8;
    f16x8 x_qk[QR], x_v[VR];
#pragma unroll
    for (int n = 0; n < QR; ++n) x_qk[n] = *(const f16x8*)(xb + (size_t)min(tid / 32 + n * QT, T - 1) * x_stride + ch_qk);
#pragma unroll
    for (int n = 0; n < VR; ++n)
        x_v[n] = *(const f16x8*)(xb + (size_t)min(lane / (2 * TL) + n * LT, T - 1) * x_stride + ch_v);
    Taps8 conv, conv_v;
    conv.load(conv_w, ch_qk);
    conv_v.load(conv_w, ch_v);
    // the frames ahead of the rows, by two waves that have no gates to form
    Frames8 old;
    if (w == WAVES - 1 && lane < 32) {
        old.load(seqs.frames[b], fresh, ch_qk);
        f16* to = s_raw[part][0] + ch8;
        *(f16x8*)to = old.f0, *(f16x8*)(to + ROW_H) = old.f1, *(f16x8*)(to + 2 * ROW_H) = old.f2;
    }
    if (w == WAVES - 2 && lane < 16 * HP) {
        old.load(seqs.frames[b], fresh, (2 * n_kheads + at * HP) * GT_K + 8 * lane);
        f16* to = (f16*)s_own[8 * lane / COLS] + 8 * lane % COLS;
        *(f16x8*)to = old.f0, *(f16x8*)(to + RAW_P) = old.f1, *(f16x8*)(to + 2 * RAW_P) = old.f2;
    }
    // S0: rows c0 + 16 t + col, columns 32 c + 8 g .. + 7
    f32x8 s0[TL][4];
    const float* srow = seqs.S[b] + ((size_t)hv * GT_K + c0 + col) * GT_K + 8 * g;
    auto load_s0 = [&](int t) {
#pragma unroll
        for (int c = 0; c < 4; ++c) s0[t][c] = *(const f32x8*)(srow + 16 * t * GT_K + 32 * c);
    };
    // (half of it now where there is much of it: 16 trees of 16 17.0 us in place of 18.3; by one head a workgroup the
    // rows come sooner without, one tree of 16 8.5 us in place of 9.2)
    if (TL > 1) load_s0(0);

    if (w < HP) {
        double sum = lane < T ? (double)log_decay(a_in + dt, A) : 0.;
        const Node n = tree_node<true>(parent, T, &sum);
        // a place without a token has zeros everywhere: nothing of it reaches the others
        s_log[w][lane] = sum *= 1.4426950408889634;
        s_beta[w][lane] = n.here() ? gdn_beta(b_in) : 0.f;
        s_gain[w][lane] = n.here() ? decayed(sum) : 0.f;
        if (w == 0) {
            // (the n-th token ahead of the context: frame n, as -1 - n)
            const int p1 = n.parent < 0 ? -2 : n.parent;
            const int up1 = lane_of(n.parent, max(p1, 0));
            const int p2 = p1 < 0 ? p1 - 1 : up1 < 0 ? -2 : up1;
            const int up2 = lane_of(n.parent, max(p2, 0));
            const int p3 = p2 < 0 ? p2 - 1 : up2 < 0 ? -2 : up2;
            auto row = [](int p) { return p < 0 ? p + 4 : p + 3; };
            s_up[lane] = make_int4(row(p1), row(p2), row(p3), n.here());
            s_line[lane] = make_uint2(n.lo, n.hi);
            const uint64_t here = __ballot(n.here());
            if (lane == 0) s_n = here ? 64 - __builtin_clzll(here) : 0;
        }
    }
    f16(*own_x)[RAW_P] = (f16(*)[RAW_P])s_own[w];
    float(*own)[OUT_P] = (float(*)[OUT_P])s_own[w];
#pragma unroll
    for (int n = 0; n < QR; ++n)
        if (QR * QT == TP || tid / 32 + n * QT < TP) *(f16x8*)(s_raw[part][3 + tid / 32 + n * QT] + ch8) = x_qk[n];
#pragma unroll
    for (int n = 0; n < VR; ++n)
        if (VR * LT == TP || lane / (2 * TL) + n * LT < TP) *(f16x8*)(own_x[3 + lane / (2 * TL) + n * LT] + v8) = x_v[n];
    __syncthreads();
    const int n = __builtin_amdgcn_readfirstlane(s_n), nb = (n + 15) >> 4;   // tokens, blocks of them
#pragma unroll
    for (int t = TL > 1; t < TL; ++t) load_s0(t);

    auto conv_of = [&](Taps8& taps, const f16* at, int pitch, int i, f32x4& lo, f32x4& hi) {
        const int4 up = s_up[i];
        taps.apply(lo, hi, *(const f16x8*)(at + up.z * pitch), *(const f16x8*)(at + up.y * pitch),
                   *(const f16x8*)(at + up.x * pitch), *(const f16x8*)(at + (i + 3) * pitch));
    };
    for (int i = tid >> 5; i < 16 * nb; i += QT) {
        f32x4 lo, hi;
        const bool here = s_up[i].w;
        conv_of(conv, s_raw[part][0] + ch8, ROW_H, i, lo, hi);
        const float inv = QK_SCALE / sqrtf(row16_sum(sum_sq(lo, hi)) + l2eps);
        Terms t = split8(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7), inv);
        if (!here) t.hi = t.lo = (f16x8)(0);
        Rows* dst = part == 0 ? s_q : s_k;
        *(f16x8*)(dst[0][i] + ch8) = t.hi;
        *(f16x8*)(dst[1][i] + ch8) = t.lo;
    }
    // v: token 16 r + 4 g + e, state row c0 + 16 t + col
    f32x4 v[NB][TL];
    {
        f32x4 lo[VR], hi[VR];
#pragma unroll
        for (int k = 0; k < VR; ++k)
            if (k * LT < n) {
                const int i = VR * LT == TP ? lane / (2 * TL) + k * LT : min(lane / (2 * TL) + k * LT, TP - 1);
                conv_of(conv_v, own_x[0] + v8, RAW_P, i, lo[k], hi[k]);
                if (!s_up[i].w) lo[k] = hi[k] = (f32x4)(0.f);
            } else {
                lo[k] = hi[k] = (f32x4)(0.f);
            }
#pragma unroll
        for (int k = 0; k < VR; ++k) {
            wave_sync();
            if (OUT_ROWS == LT || lane / (2 * TL) < OUT_ROWS) {
                *(f32x4*)(own[lane / (2 * TL)] + v8) = lo[k];
                *(f32x4*)(own[lane / (2 * TL)] + v8 + 4) = hi[k];
            }
            wave_sync();
#pragma unroll
            for (int r = k * LT / 16; r < (k + 1) * LT / 16 && r < NB; ++r)
#pragma unroll
                for (int t = 0; t < TL; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[r][t][e] = own[16 * r - k * LT + 4 * g + e][16 * t + col];
        }
    }
    __syncthreads();
    auto terms = [&](const Rows* m, int row, int c) {
        return Terms{*(const f16x8*)(m[0][row] + 32 * c + 8 * g), *(const f16x8*)(m[1][row] + 32 * c + 8 * g)};
    };

    // -A and the q.k side, 16 x 16 blocks on and below the diagonal
    for (int job = w; job < nb * (nb + 1); job += WAVES) {
        const bool qk = job & 1;
        int r = 0, c = job >> 1;
        while (c > r) c -= ++r;
        f32x4 acc = (f32x4)(0.f);
#pragma unroll
        for (int s = 0; s < 4; ++s)
            acc = mfma_terms(terms(qk ? s_q : s_k, 16 * r + col, s), terms(s_k, 16 * c + col, s), acc);
        const int j = 16 * c + col, i0 = 16 * r + 4 * g;
        float f[4];
        bool anc[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint2 line = s_line[i0 + e];
            anc[e] = ((j < 32 ? line.x : line.y) >> (j & 31) & 1) && (qk || j != i0 + e);
            f[e] = anc[e] ? acc[e] * (1.f / (QK_SCALE * QK_SCALE)) : 0.f;
        }
#pragma unroll
        for (int m = 0; m < HP; ++m) {
            f32x4 beta = (f32x4)(1.f);
            if (!qk) beta = -*(const f32x4*)&s_beta[m][i0];
            const double lj = s_log[m][j];
            float a[4];
            double li[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) li[e] = s_log[m][i0 + e];
            asm("" : "+v"(li[0]), "+v"(li[1]), "+v"(li[2]), "+v"(li[3]));   // (here: a branch a number otherwise)
#pragma unroll
            for (int e = 0; e < 4; ++e)   // (others' decays may be anything)
                a[e] = f[e] * beta[e] * decayed(anc[e] ? li[e] - lj : 0.);
            Block& to = (qk ? s_p : s_a)[m][job >> 1];
            if (!qk && r == c) {
                *(f32x4*)&to[col][4 * g] = (f32x4){a[0], a[1], a[2], a[3]};
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) to[4 * g + e][col] = a[e];
            }
        }
    }
    __syncthreads();
    // the inverse of a diagonal block I + A, a column a lane
    if (w < HP * nb) {
        Block& m = s_a[w / nb][(w % nb) * (w % nb + 3) / 2];
        float xi[16];
        uint32_t at_m = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) xi[i] = i == col ? 1.f : 0.f;
#pragma unroll
        for (int i = 0; i < 15; ++i) {   // (a row of m is a column of -A: no chain but over the rows)
            // (no column before the sixth-last number is known: all at once are too many registers)
            if (i >= 6) asm("" : "+v"(at_m) : "v"(xi[i - 5]));
            f32x4 a[4];
#pragma unroll
            for (int q = (i + 1) / 4; q < 4; ++q) a[q] = *(const f32x4*)((const char*)&m[i][4 * q] + at_m);
#pragma unroll
            for (int q = i + 1; q < 16; ++q) xi[q] = fmaf(a[q >> 2][q & 3], xi[i], xi[q]);
        }
        if (g == 0)
#pragma unroll
            for (int i = 0; i < 16; ++i) m[i][col] = xi[i];
    }
    // The right side and o's first part, from S0 k_i and S0 q_i. With the largest number of a state row at
    // 2^14 or more the terms' 2^-25 is 2^-39 of it.
    Terms st[TL][4];
    float back[TL];   // from the products' units
#pragma unroll
    for (int t = 0; t < TL; ++t) {
        float top = 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(s0[t][c][e]));
        const int up = lift(top);
        const float unit = pow2(up);
#pragma unroll
        for (int c = 0; c < 4; ++c) st[t][c] = split8(s0[t][c], unit);
        back[t] = pow2(-up) * (1.f / QK_SCALE);
    }
    f32x4 u[NB][TL], o[NB][TL];
#pragma unroll
    for (int r = 0; r < NB; ++r) {
        if (r >= nb) continue;
        f32x4 wk[TL], wq[TL];
#pragma unroll
        for (int t = 0; t < TL; ++t) wk[t] = wq[t] = (f32x4)(0.f);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const Terms k = terms(s_k, 16 * r + col, c), q = terms(s_q, 16 * r + col, c);
#pragma unroll
            for (int t = 0; t < TL; ++t) {
                wk[t] = mfma_terms(k, st[t][c], wk[t]);
                wq[t] = mfma_terms(q, st[t][c], wq[t]);
            }
        }
        const f32x4 beta = *(const f32x4*)&s_beta[h][16 * r + 4 * g];
        const f32x4 gain = *(const f32x4*)&s_gain[h][16 * r + 4 * g];
#pragma unroll
        for (int t = 0; t < TL; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                u[r][t][e] = beta[e] * fmaf(-gain[e], wk[t][e] * back[t], v[r][t][e]);
                o[r][t][e] = gain[e] * (wq[t][e] * back[t]);
            }
    }
    // the output's gates, a token a row of 2 TL lanes (whose places are not worth registers until here)
    int l = lane;
    asm volatile("" : "+v"(l));
    const int row0 = l / (2 * TL), out8 = 8 * (l & (2 * TL - 1));
    f16x8 gate[VR];
#pragma unroll
    for (int k = 0; k < VR; ++k)
        gate[k] = *(const f16x8*)(z + ((size_t)b * T + min(row0 + k * LT, T - 1)) * z_pitch + hv * GT_K + c0 + out8);
    __syncthreads();

    // block by block of tokens
#pragma unroll
    for (int r = 0; r < NB; ++r) {
        if (r >= nb) continue;
        auto at = [&](const Block* m, int c) { return *(const f32x4*)&m[r * (r + 1) / 2 + c][col][4 * g]; };
#pragma unroll
        for (int c = 0; c < r; ++c) {
            const f32x4 a = at(s_a[h], c);
#pragma unroll
            for (int t = 0; t < TL; ++t) u[r][t] = mfma_block(a, u[c][t], u[r][t]);
        }
        const f32x4 inv = at(s_a[h], r);
#pragma unroll
        for (int t = 0; t < TL; ++t) u[r][t] = mfma_block(inv, u[r][t], (f32x4)(0.f));
#pragma unroll
        for (int c = 0; c <= r; ++c) {
            const f32x4 p = at(s_p[h], c);
#pragma unroll
            for (int t = 0; t < TL; ++t) o[r][t] = mfma_block(p, u[c][t], o[r][t]);
        }
    }
    // o scaled; squares of a row over this wave's columns, then over the head's waves
#pragma unroll
    for (int r = 0; r < NB; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float ss = 0.f;
#pragma unroll
            for (int t = 0; t < TL; ++t) {
                o[r][t][e] = r < nb ? o[r][t][e] * out_scale : 0.f;
                ss = fmaf(o[r][t][e], o[r][t][e], ss);
            }
            ss = row16_sum(ss);
            if (col == 0) s_ss[h][16 * r + 4 * g + e][w - h * HW] = ss;
        }
    __syncthreads();
    const f32x4 w0 = *(const f32x4*)(norm_w + c0 + out8), w1 = *(const f32x4*)(norm_w + c0 + out8 + 4);
#pragma unroll
    for (int k = 0; k < VR; ++k) {
        wave_sync();
#pragma unroll
        for (int r = k * LT / 16; r < (k + 1) * LT / 16 && r < NB; ++r)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int t = 0; t < TL; ++t) own[16 * r - k * LT + 4 * g + e][16 * t + col] = o[r][t][e];
        wave_sync();
        const int i = row0 + k * LT;
        if (i < T) {
            f16x8 out = (f16x8)(0);
            if (s_up[i].w) {
                const f32x4 a = *(const f32x4*)(own[row0] + out8), c = *(const f32x4*)(own[row0] + out8 + 4);
                float t[8] = {a[0], a[1], a[2], a[3], c[0], c[1], c[2], c[3]}, ss = 0.f;
#pragma unroll
                for (int m = 0; m < HW; m += 4) {
                    const f32x4 p = *(const f32x4*)&s_ss[h][i][m];
                    ss += (p[0] + p[1]) + (p[2] + p[3]);
                }
                const float inv = 1.f / sqrtf(ss / (float)GT_K + norm_eps);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float gz = (float)gate[k][e];
                    t[e] *= inv * (e < 4 ? w0[e] : w1[e - 4]) * (gz * __builtin_amdgcn_rcpf(1.f + hw_expf(-gz)));
                }
                out = f16_sat8(t);
            }
            *(f16x8*)(y + ((size_t)b * T + i) * y_pitch + hv * GT_K + c0 + out8) = out;
        }
    }
}

// ---------------------------------------------------------------------------
// The state and the conv frames behind an accepted path, token by token: ROWS state rows a workgroup,
// a row on 8 lanes (columns 4 l + 32 j .. + 3) in registers throughout, k and v of the path's tokens
// formed first. Reads and writes a state once: bound by that for a batch.
// ---------------------------------------------------------------------------
struct CommitSeqs {
    const float* S[FL_MAX_SEQS];
    float* S_out[FL_MAX_SEQS];
    const f16* frames[FL_MAX_SEQS];
    f16* frames_out[FL_MAX_SEQS];
    int pos0[FL_MAX_SEQS];
};

__device__ __forceinline__ float row8_sum(float v) {
    v += dpp_xor1(v);
    v += dpp_xor2(v);
    return v + __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x141, 0xF, 0xF, true));   // half mirror
}

// (five waves a SIMD: 22.6 us for 16 paths of 7, with the registers of four 23.5, six spill)
__global__ void __launch_bounds__(8 * GC_ROWS, 5)
gdn_commit_kernel(const f16* __restrict__ x, int x_stride, const f16* __restrict__ conv_w, const CommitSeqs seqs,
                  const int* __restrict__ path, const float* __restrict__ ga, const float* __restrict__ gb,
                  int ab_stride, const float* __restrict__ A_log, const float* __restrict__ dt_bias, int T, int D,
                  int n_kheads, int n_vheads, float l2eps) {
    constexpr int ROWS = GC_ROWS, THREADS = 8 * ROWS, PARTS = GT_K / ROWS, VL = ROWS / 8;   // lanes a token's v takes
    extern __shared__ __attribute__((aligned(16))) float s_kv[];            // [D][128] of k, [D][ROWS] of v,
    __shared__ float s_beta[TREE_MAX], s_alpha[TREE_MAX];                   // and their input's rows
    __shared__ int s_at[TREE_MAX], s_n;
    float(*s_k)[GT_K] = (float(*)[GT_K])s_kv;
    float(*s_v)[ROWS] = (float(*)[ROWS])(s_kv + D * GT_K);
    f16(*x_k)[GT_K] = (f16(*)[GT_K])(s_kv + D * (GT_K + ROWS));   // three frames, then the path's tokens
    f16(*x_v)[ROWS] = (f16(*)[ROWS])(x_k + D + 3);
    const int tid = threadIdx.x;
    const int part = blockIdx.x % PARTS, hv = blockIdx.x / PARTS % n_vheads, b = blockIdx.x / PARTS / n_vheads;
    const int group = n_vheads / n_kheads, hk = hv / group;
    const bool fresh = seqs.pos0[b] == 0;

    if (tid < 64) {   // the path's tokens, and their gates
        const int i = tid < D ? path[(size_t)b * D + tid] : -1;
        const int before = lane_of(i, max(tid - 1, 0));
        const uint64_t end = __ballot(!(i > (tid ? before : -1) && i < T));
        const int len = end ? __builtin_ctzll(end) : 64;
        if (tid == 0) s_n = len;
        if (tid < len) {
            const size_t at = ((size_t)b * T + i) * ab_stride + hv;
            s_at[tid] = i;
            s_alpha[tid] = gdn_decay(ga[at] + dt_bias[hv], A_log[hv]);
            s_beta[tid] = gdn_beta(gb[at]);
        }
    }
    const int k8 = 8 * (tid & 15), v8 = 8 * (tid & (VL - 1));   // k: a token on 16 lanes
    const int ch_k = (n_kheads + hk) * GT_K + k8, ch_v = (2 * n_kheads + hv) * GT_K + part * ROWS + v8;
    if (tid >= 64 && tid < 80) {
        Frames8 old;
        old.load(seqs.frames[b], fresh, ch_k);
        *(f16x8*)(x_k[0] + k8) = old.f0, *(f16x8*)(x_k[1] + k8) = old.f1, *(f16x8*)(x_k[2] + k8) = old.f2;
    }
    if (tid >= 128 && tid < 128 + VL) {
        Frames8 old;
        old.load(seqs.frames[b], fresh, ch_v);
        *(f16x8*)(x_v[0] + v8) = old.f0, *(f16x8*)(x_v[1] + v8) = old.f1, *(f16x8*)(x_v[2] + v8) = old.f2;
    }
    Taps8 tk, tv;
    tk.load(conv_w, ch_k);
    tv.load(conv_w, ch_v);
    __syncthreads();
    const int n = s_n;

    // the tokens' rows, then the state (row part ROWS + tid / 8): loads return in order
    const f16* xb = x + (size_t)b * T * x_stride;
    auto row_k = [&](int d) { return *(const f16x8*)(xb + (size_t)s_at[d] * x_stride + ch_k); };
    auto row_v = [&](int d) { return *(const f16x8*)(xb + (size_t)s_at[d] * x_stride + ch_v); };
    int dk = tid >> 4, dv = tid / VL;
    f16x8 rk, rv;
    if (dk < n) rk = row_k(dk);
    if (dv < n) rv = row_v(dv);
    const size_t srow = ((size_t)hv * GT_K + part * ROWS + (tid >> 3)) * GT_K + 4 * (tid & 7);
    f32x4 s[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) s[j] = *(const f32x4*)(seqs.S[b] + srow + 32 * j);
    if (dk < n) *(f16x8*)(x_k[dk + 3] + k8) = rk;
    if (dv < n) *(f16x8*)(x_v[dv + 3] + v8) = rv;
    while ((dk += THREADS / 16) < n) *(f16x8*)(x_k[dk + 3] + k8) = row_k(dk);
    while ((dv += THREADS / VL) < n) *(f16x8*)(x_v[dv + 3] + v8) = row_v(dv);
    __syncthreads();

    auto put_frames = [&](f16x8 x, f16x8 y, f16x8 z, int ch) {   // [channel][frame] of the last three
        f16x8* to = (f16x8*)(seqs.frames_out[b] + 3 * ch);
        to[0] = (f16x8){x[0], y[0], z[0], x[1], y[1], z[1], x[2], y[2]};
        to[1] = (f16x8){z[2], x[3], y[3], z[3], x[4], y[4], z[4], x[5]};
        to[2] = (f16x8){y[5], z[5], x[6], y[6], z[6], x[7], y[7], z[7]};
    };
    for (int d = tid >> 4; d < n; d += THREADS / 16) {
        f32x4 lo, hi;
        auto at = [&](int r) { return *(const f16x8*)(x_k[d + r] + k8); };
        tk.apply(lo, hi, at(0), at(1), at(2), at(3));
        const float inv = 1.f / sqrtf(row16_sum(sum_sq(lo, hi)) + l2eps);
        *(f32x4*)(s_k[d] + k8) = lo * inv;
        *(f32x4*)(s_k[d] + k8 + 4) = hi * inv;
    }
    for (int d = tid / VL; d < n; d += THREADS / VL) {
        f32x4 lo, hi;
        auto at = [&](int r) { return *(const f16x8*)(x_v[d + r] + v8); };
        tv.apply(lo, hi, at(0), at(1), at(2), at(3));
        *(f32x4*)(s_v[d] + v8) = lo;
        *(f32x4*)(s_v[d] + v8 + 4) = hi;
    }
    auto last = [&](int r) { return *(const f16x8*)(x_v[n + r] + v8); };
    if (tid < VL) put_frames(last(0), last(1), last(2), ch_v);
    if (hv == hk * group && part == 0) {   // the frames of q and k, once a k head
        auto last = [&](int r) { return *(const f16x8*)(x_k[n + r] + k8); };
        if (tid >= 64 && tid < 80) put_frames(last(0), last(1), last(2), ch_k);
        if (tid >= 128 && tid < 144) {
            const int ch = hk * GT_K + k8;
            Frames8 old;
            old.load(seqs.frames[b], fresh, ch);
            auto row = [&](int d) { return xb + (size_t)s_at[max(d, 0)] * x_stride + ch; };
            put_frames(token(3 - n, row(n - 3), old.f0, old.f1, old.f2),
                       token(2 - n, row(n - 2), old.f0, old.f1, old.f2),
                       token(1 - n, row(n - 1), old.f0, old.f1, old.f2), ch);
        }
    }
    __syncthreads();
    for (int d = 0; d < n; ++d) {
        f32x4 k[4];
        const float alpha = s_alpha[d];
        float m = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            k[j] = *(const f32x4*)(s_k[d] + 4 * (tid & 7) + 32 * j);
            s[j] *= alpha;
#pragma unroll
            for (int e = 0; e < 4; ++e) m = fmaf(s[j][e], k[j][e], m);
        }
        const float delta = s_beta[d] * (s_v[d][tid >> 3] - row8_sum(m));
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[j][e] = fmaf(delta, k[j][e], s[j][e]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) *(f32x4*)(seqs.S_out[b] + srow + 32 * j) = s[j];
}

bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int check_layer(const void* x, int x_stride, const void* conv_w, const void* const* cst_in, const int* pos0,
                const int* nodes, const float* a, const float* b, int ab_stride, const float* A_log,
                const float* dt_bias, const float* const* S, int B, int T, int n_kheads, int n_vheads, int K,
                int V, float l2eps) {
    FL_REQUIRE(x && conv_w && cst_in && pos0 && a && b && A_log && dt_bias && S, "null pointer");
    FL_REQUIRE(B >= 1 && B <= FL_MAX_SEQS, "1 <= B <= FL_MAX_SEQS");
    FL_REQUIRE(T >= 1 && T <= FL_TREE_MAX && nodes, "1 <= T <= FL_TREE_MAX, parents / path given");
    FL_REQUIRE(K == GT_K && V == GT_K, "K == V == 128");
    FL_REQUIRE(n_kheads >= 1 && n_vheads >= 1 && n_vheads <= 4096 && n_vheads % n_kheads == 0,
               "n_vheads % n_kheads");
    FL_REQUIRE(x_stride >= 2 * n_kheads * K + n_vheads * V && x_stride % 8 == 0 && al16(x) && al16(conv_w),
               "x_stride >= 2 n_kheads K + n_vheads V, % 8, 16-byte aligned x, conv_w");
    FL_REQUIRE(ab_stride >= n_vheads && l2eps >= 0.f, "ab_stride >= n_vheads, eps >= 0");
    for (int i = 0; i < B; ++i)
        FL_REQUIRE(S[i] && al16(S[i]) && cst_in[i] && al16(cst_in[i]) && pos0[i] >= 0,
                   "S, cst_in: null or not 16-byte aligned; pos0 >= 0");
    return FL_OK;
}

// Does an output overlap one of a layer's inputs (`nodes`: parents or path; the states and frames apart)?
bool meet_layer(const RowsOf& out, const void* x, int x_stride, const void* conv_w, const int* nodes, size_t n_nodes,
                const float* a, const float* b, int ab_stride, const float* A_log, const float* dt_bias, size_t rows,
                int n_kheads, int n_vheads) {
    const size_t dim = (2 * (size_t)n_kheads + n_vheads) * GT_K, gates = 4 * (size_t)n_vheads;
    auto flat = [&](const void* p, size_t n) { return meet(out.p, out.bytes(), p, n); };
    return meet(out, RowsOf{x, rows, 2 * (size_t)x_stride, 2 * dim}) ||
           meet(out, RowsOf{a, rows, 4 * (size_t)ab_stride, gates}) ||
           meet(out, RowsOf{b, rows, 4 * (size_t)ab_stride, gates}) || flat(conv_w, 8 * dim) || flat(nodes, 4 * n_nodes) ||
           flat(A_log, gates) || flat(dt_bias, gates);
}

}  // namespace

extern "C" {

int fl_gdn_tree_normed(const void* x, int x_stride, const void* conv_w, const void* const* cst_in,
                       const int* pos0, const int* parents, const float* a, const float* b, int ab_stride,
                       const float* A_log, const float* dt_bias, const float* const* S, const void* z,
                       int z_pitch, const float* norm_w, void* y, int y_pitch, int B, int T, int n_kheads,
                       int n_vheads, int K, int V, float out_scale, float l2eps, float norm_eps,
                       fl_stream_t stream) {
    const int rc = check_layer(x, x_stride, conv_w, cst_in, pos0, parents, a, b, ab_stride, A_log, dt_bias, S, B,
                               T, n_kheads, n_vheads, K, V, l2eps);
    if (rc) return rc;
    FL_REQUIRE(z && norm_w && y, "null pointer");
    FL_REQUIRE(z_pitch >= n_vheads * V && y_pitch >= n_vheads * V && z_pitch % 8 == 0 && y_pitch % 8 == 0 &&
                   al16(z) && al16(y) && al16(norm_w) && norm_eps >= 0.f,
               "z, y: pitch >= n_vheads V, % 8, 16-byte aligned; norm_w 16-byte aligned, eps >= 0");
    const size_t rows = (size_t)B * T, width = (size_t)n_vheads * V;
    const RowsOf out = {y, rows, 2 * (size_t)y_pitch, 2 * width};
    bool apart = !meet_layer(out, x, x_stride, conv_w, parents, rows, a, b, ab_stride, A_log, dt_bias, rows, n_kheads,
                             n_vheads) &&
                 !meet(out, RowsOf{z, rows, 2 * (size_t)z_pitch, 2 * width}) && !meet(y, out.bytes(), norm_w, 4 * (size_t)V);
    for (int i = 0; i < B; ++i)
        apart = apart && !meet(y, out.bytes(), S[i], 4 * width * K) &&
                !meet(y, out.bytes(), cst_in[i], 6 * (2 * (size_t)n_kheads * K + width));
    FL_REQUIRE(apart, "y overlaps an input");
    TreeSeqs seqs = {};
    for (int i = 0; i < B; ++i) {
        seqs.S[i] = S[i];
        seqs.frames[i] = (const f16*)cst_in[i];
        seqs.pos0[i] = pos0[i];
    }
    const int group = n_vheads / n_kheads;
    auto launch = [&](auto kernel, int heads, int threads) {
        hipLaunchKernelGGL(kernel, dim3(B * (n_vheads / heads)), dim3(threads), 0, (hipStream_t)stream, (const f16*)x,
                           x_stride, (const f16*)conv_w, seqs, parents, a, b, ab_stride, A_log, dt_bias,
                           (const f16*)z, z_pitch, norm_w, (f16*)y, y_pitch, T, n_kheads, n_vheads, out_scale,
                           l2eps, norm_eps);
    };
    const int nb = (T + 15) / 16;
    const bool many = B * n_vheads > GT_MANY;   // (beyond 48 tokens LDS holds one head's)
    if (nb <= 3 && many && group % 3 == 0)
        launch(nb == 1   ? gdn_tree_kernel<1, 3, 2>
               : nb == 2 ? gdn_tree_kernel<2, 3, 2>
                         : gdn_tree_kernel<3, 3, 2>, 3, 768);
    else if (nb <= 3 && many && group % 2 == 0)
        launch(nb == 1   ? gdn_tree_kernel<1, 2, 2>
               : nb == 2 ? gdn_tree_kernel<2, 2, 2>
                         : gdn_tree_kernel<3, 2, 2>, 2, 512);
    else
        launch(nb == 1   ? gdn_tree_kernel<1, 1, 1>
               : nb == 2 ? gdn_tree_kernel<2, 1, 1>
               : nb == 3 ? gdn_tree_kernel<3, 1, 1>
                         : gdn_tree_kernel<4, 1, 1>, 1, 512);
    return fl::check_launch("gdn_tree_normed");
}

int fl_gdn_tree_commit(const void* x, int x_stride, const void* conv_w, const void* const* cst_in,
                       void* const* cst_out, const int* pos0, const int* path, const float* a, const float* b,
                       int ab_stride, const float* A_log, const float* dt_bias, const float* const* S,
                       float* const* S_out, int B, int T, int D, int n_kheads, int n_vheads, int K, int V,
                       float l2eps, fl_stream_t stream) {
    const int rc = check_layer(x, x_stride, conv_w, cst_in, pos0, path, a, b, ab_stride, A_log, dt_bias, S, B, T,
                               n_kheads, n_vheads, K, V, l2eps);
    if (rc) return rc;
    FL_REQUIRE(cst_out && S_out, "null pointer");
    FL_REQUIRE(D >= 1 && D <= FL_TREE_MAX, "1 <= D <= FL_TREE_MAX");
    const size_t state = (size_t)n_vheads * V * K * 4, ring = ((size_t)2 * n_kheads * K + n_vheads * V) * 6;
    CommitSeqs seqs = {};
    for (int i = 0; i < B; ++i) {
        FL_REQUIRE(S_out[i] && al16(S_out[i]) && cst_out[i] && al16(cst_out[i]),
                   "S_out, cst_out: null or not 16-byte aligned");
        for (int j = 0; j < B; ++j) {
            FL_REQUIRE(!meet(cst_out[i], ring, cst_in[j], ring), "cst_out overlaps a cst_in: they must be distinct");
            FL_REQUIRE(j == i || (!meet(S_out[i], state, S_out[j], state) && !meet(cst_out[i], ring, cst_out[j], ring)),
                       "two sequences' S_out or cst_out overlap");
            FL_REQUIRE(!meet(S_out[i], state, S[j], state) || (i == j && S_out[i] == S[i]),
                       "S_out overlaps an S other than its own");
            FL_REQUIRE(!meet(S_out[i], state, cst_in[j], ring) && !meet(S_out[i], state, cst_out[j], ring) &&
                           !meet(cst_out[i], ring, S[j], state),
                       "states and frames overlap");
        }
        for (const RowsOf& out : {RowsOf{S_out[i], 1, state, state}, RowsOf{cst_out[i], 1, ring, ring}})
            FL_REQUIRE(!meet_layer(out, x, x_stride, conv_w, path, (size_t)B * D, a, b, ab_stride, A_log, dt_bias,
                                   (size_t)B * T, n_kheads, n_vheads),
                       "S_out or cst_out overlaps an input");
        seqs.S[i] = S[i];
        seqs.S_out[i] = S_out[i];
        seqs.frames[i] = (const f16*)cst_in[i];
        seqs.frames_out[i] = (f16*)cst_out[i];
        seqs.pos0[i] = pos0[i];
    }
    hipLaunchKernelGGL(gdn_commit_kernel, dim3(B * n_vheads * (GT_K / GC_ROWS)), dim3(8 * GC_ROWS),
                       (D * 6 + 6) * (GT_K + GC_ROWS), (hipStream_t)stream, (const f16*)x,
                       x_stride, (const f16*)conv_w, seqs, path, a, b, ab_stride, A_log, dt_bias, T, D, n_kheads,
                       n_vheads, l2eps);
    return fl::check_launch("gdn_tree_commit");
}

}  // extern "C"
