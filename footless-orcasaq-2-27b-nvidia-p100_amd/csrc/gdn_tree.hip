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
// Everything is fp32 (fp64: the sums of log alpha, whose differences are the logarithms of
// G_i / G_j) and y is rounded once, where gdn_decode_normed rounds the conv's output, q, k and o to
// fp16 as the reference does.
//
// A workgroup is a (sequence, v head); wave w has state rows 16 w .. + 15, held as the B operand of
// 16x16x4 fp32 MFMAs whose accumulators are in turn the B operands of the next product: D's
// register e of lane (g, c) is row 4 g + e of column c, and a k step takes k = 4 g + e from lane
// group g on both sides. The 16-row diagonal blocks of I + A are inverted by substitution, a
// column a lane; U is then a product a block.
#include "tree.hpp"

#include "gdn_gates.hpp"

#include <math.h>

namespace {

typedef float f32x8 __attribute__((ext_vector_type(8)));

constexpr int GT_K = 128;                // K = V
constexpr int GT_WAVES = 8;
constexpr int GT_THREADS = 64 * GT_WAVES;
constexpr int ROW_P = GT_K + 4;          // floats a row of v and o in LDS
constexpr int ROW_H = GT_K + 8;          // terms a row of k and q
constexpr float QK_SCALE = 16384.f;      // of q and k, whose norms are at most 1
constexpr int INV_P = 20;                // floats a row of an inverse block

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
// e^x of a difference of such sums
__device__ __forceinline__ float ratio(double x) { return fast_exp2((float)(x * 1.4426950408889634)); }

// Eight channels' conv: the taps and the sequence's last three frames ([channel][frame], oldest
// first; zero for a fresh sequence).
struct Conv8 {
    f16x8 w0, w1, w2, w3;   // a tap of all channels each, the newest last
    f16x8 f0, f1, f2;
    __device__ __forceinline__ void load(const f16* conv_w, const f16* frames, bool fresh, int ch) {
        const f16x8 *t = (const f16x8*)(conv_w + 4 * ch), *x = (const f16x8*)(frames + 3 * ch);
        const f16x8 a = t[0], b = t[1], c = t[2], d = t[3], x0 = x[0], x1 = x[1], x2 = x[2];
        w0 = (f16x8){a[0], a[4], b[0], b[4], c[0], c[4], d[0], d[4]};
        w1 = (f16x8){a[1], a[5], b[1], b[5], c[1], c[5], d[1], d[5]};
        w2 = (f16x8){a[2], a[6], b[2], b[6], c[2], c[6], d[2], d[6]};
        w3 = (f16x8){a[3], a[7], b[3], b[7], c[3], c[7], d[3], d[7]};
        f0 = (f16x8){x0[0], x0[3], x0[6], x1[1], x1[4], x1[7], x2[2], x2[5]};
        f1 = (f16x8){x0[1], x0[4], x0[7], x1[2], x1[5], x2[0], x2[3], x2[6]};
        f2 = (f16x8){x0[2], x0[5], x1[0], x1[3], x1[6], x2[1], x2[4], x2[7]};
        if (fresh) f0 = f1 = f2 = (f16x8)(0);
    }
    // silu of the taps over x0 (the token's) and the three before it
    __device__ __forceinline__ float channel(int c, f16x8 x3, f16x8 x2, f16x8 x1, f16x8 x0) const {
        float s = (float)w0[c] * (float)x3[c];
        s = fmaf((float)w1[c], (float)x2[c], s);
        s = fmaf((float)w2[c], (float)x1[c], s);
        s = fmaf((float)w3[c], (float)x0[c], s);
        return s * __builtin_amdgcn_rcpf(1.f + hw_expf(-s));
    }
    __device__ __forceinline__ void apply(f32x4& lo, f32x4& hi, f16x8 x3, f16x8 x2, f16x8 x1, f16x8 x0) const {
        auto y = [&](int c) { return channel(c, x3, x2, x1, x0); };
        lo = (f32x4){y(0), y(1), y(2), y(3)};
        hi = (f32x4){y(4), y(5), y(6), y(7)};
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

// x as two fp16 terms: 22 bits of it, and what lies 2^-24 below 1 (so x is scaled up first)
__device__ __forceinline__ void split(f32x8 x, f16x8& hi, f16x8& lo) {
    hi = __builtin_convertvector(x, f16x8);
    lo = __builtin_convertvector(x - __builtin_convertvector(hi, f32x8), f16x8);
}
__device__ __forceinline__ int ilogb_bits(float x) { return (int)(__float_as_uint(x) >> 23 & 255) - 127; }
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
struct Terms {
    f16x8 hi, lo;
};
// c + a b without the product of the two low terms (2^-22 of a b)
__device__ __forceinline__ f32x4 mfma_terms(const Terms& a, const Terms& b, f32x4 c) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.lo, b.hi, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.hi, b.lo, c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a.hi, b.hi, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma4(float a, float b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

template <int NB>
__global__ void __launch_bounds__(GT_THREADS)
gdn_tree_kernel(const f16* __restrict__ x, int x_stride, const f16* __restrict__ conv_w, const TreeSeqs seqs,
                const int* __restrict__ parents, const float* __restrict__ ga, const float* __restrict__ gb,
                int ab_stride, const float* __restrict__ A_log, const float* __restrict__ dt_bias,
                const f16* __restrict__ z, int z_pitch, const float* __restrict__ norm_w,
                f16* __restrict__ y, int y_pitch, int T, int n_kheads, int n_vheads, float out_scale,
                float l2eps, float norm_eps) {
    constexpr int TP = 16 * NB, MAT_P = TP + 4;
    // q and k (hi, lo each); v and then o take q's place
    __shared__ __attribute__((aligned(16))) f16 s_q[2][TP][ROW_H], s_k[2][TP][ROW_H];
    float(*s_v)[ROW_P] = (float(*)[ROW_P])s_q;
    static_assert(sizeof(float) * TP * ROW_P <= sizeof(s_q), "v over q");
    __shared__ __attribute__((aligned(16))) float s_a[TP][MAT_P], s_p[TP][MAT_P];   // -A; the q.k side
    __shared__ __attribute__((aligned(16))) float s_inv[NB][16][INV_P];
    __shared__ double s_log[64];
    __shared__ uint2 s_line[64];
    __shared__ int4 s_up[64];            // the three tokens before it on its path (-1 -n: a frame), here
    __shared__ float s_beta[64], s_gain[64];
    __shared__ int s_n;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, g = lane >> 4;
    // Workgroups go to the 8 XCDs round-robin: a k head's v heads to one of them.
    int hv = blockIdx.x % n_vheads, b = blockIdx.x / n_vheads;
    if (n_vheads % 8 == 0) {
        const int per = n_vheads / 8, r = blockIdx.x >> 3;
        hv = (blockIdx.x & 7) * per + r % per;
        b = r / per;
    }
    const int hk = hv / (n_vheads / n_kheads);

    // S0: row 16 w + col, columns 32 c + 8 g .. + 7
    f32x8 s0[4];
    const float* srow = seqs.S[b] + ((size_t)hv * GT_K + 16 * w + col) * GT_K + 8 * g;
#pragma unroll
    for (int c = 0; c < 4; ++c) s0[c] = *(const f32x8*)(srow + 32 * c);

    // the conv: a thread forms 8 channels of q or k, later of v, of tokens slot, slot + 16 (32), ...
    const bool fresh = seqs.pos0[b] == 0;
    const int part = tid >> 4 & 1, ch8 = 8 * (tid & 15);
    const f16* xb = x + (size_t)b * T * x_stride;
    const int ch_qk = (part == 0 ? hk : n_kheads + hk) * GT_K + ch8, ch_v = (2 * n_kheads + hv) * GT_K + ch8;
    Conv8 conv;
    conv.load(conv_w, seqs.frames[b], fresh, ch_qk);

    if (w == 0) {
        double sum = 0.;
        float beta = 0.f;
        if (lane < T) {
            const size_t at = ((size_t)b * T + lane) * ab_stride + hv;
            sum = (double)log_decay(ga[at] + dt_bias[hv], A_log[hv]);
            beta = gdn_beta(gb[at]);
        }
        const Node n = tree_node(parents + (size_t)b * T, T, sum);
        // (the n-th token ahead of the context: frame n, as -1 - n)
        const int p1 = n.parent < 0 ? -2 : n.parent;
        const int up1 = lane_of(n.parent, max(p1, 0));
        const int p2 = p1 < 0 ? p1 - 1 : up1 < 0 ? -2 : up1;
        const int up2 = lane_of(n.parent, max(p2, 0));
        const int p3 = p2 < 0 ? p2 - 1 : up2 < 0 ? -2 : up2;
        s_up[lane] = make_int4(p1, p2, p3, n.here());
        s_line[lane] = make_uint2(n.lo, n.hi);
        s_log[lane] = sum;
        s_beta[lane] = beta;
        s_gain[lane] = ratio(sum);
        const uint64_t here = __ballot(n.here());
        if (lane == 0) s_n = here ? 64 - __builtin_clzll(here) : 0;
    }
    __syncthreads();
    const int n = __builtin_amdgcn_readfirstlane(s_n), nb = (n + 15) >> 4;   // tokens, blocks of them

    auto conv_of = [&](const Conv8& cv, int i, int ch, f32x4& lo, f32x4& hi) {
        const int4 up = s_up[i];
        const f16* at = xb + ch;
        const f16x8 f0 = cv.f0, f1 = cv.f1, f2 = cv.f2;
        const f16x8 x0 = *(const f16x8*)(at + (size_t)i * x_stride);
        const f16x8 x1 = token(-1 - up.x, at + (size_t)max(up.x, 0) * x_stride, f0, f1, f2);
        const f16x8 x2 = token(-1 - up.y, at + (size_t)max(up.y, 0) * x_stride, f0, f1, f2);
        const f16x8 x3 = token(-1 - up.z, at + (size_t)max(up.z, 0) * x_stride, f0, f1, f2);
        cv.apply(lo, hi, x3, x2, x1, x0);
    };
    for (int i = tid >> 5; i < n; i += GT_THREADS / 32) {
        f32x4 lo, hi;
        conv_of(conv, i, ch_qk, lo, hi);
        const float inv = QK_SCALE / sqrtf(row16_sum(sum_sq(lo, hi)) + l2eps);
        f16x8 h, l;
        split(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7) * inv, h, l);
        f16(*dst)[TP][ROW_H] = part == 0 ? s_q : s_k;
        *(f16x8*)(dst[0][i] + ch8) = h;
        *(f16x8*)(dst[1][i] + ch8) = l;
    }
    conv.load(conv_w, seqs.frames[b], fresh, ch_v);
    __syncthreads();
    auto terms = [&](const f16 (*m)[TP][ROW_H], int row, int c) {
        return Terms{*(const f16x8*)(m[0][row] + 32 * c + 8 * g), *(const f16x8*)(m[1][row] + 32 * c + 8 * g)};
    };

    // -A and the q.k side, 16 x 16 blocks on and below the diagonal
    for (int job = w; job < nb * (nb + 1); job += GT_WAVES) {
        const bool qk = job & 1;
        int r = 0, c = job >> 1;
        while (c > r) c -= ++r;
        f32x4 acc = (f32x4)(0.f);
#pragma unroll
        for (int s = 0; s < 4; ++s)
            acc = mfma_terms(terms(qk ? s_q : s_k, 16 * r + col, s), terms(s_k, 16 * c + col, s), acc);
        const int j = 16 * c + col;
        const double lj = s_log[j];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = 16 * r + 4 * g + e;
            const uint2 line = s_line[i];
            const bool anc = ((j < 32 ? line.x : line.y) >> (j & 31) & 1) && (qk || j != i);
            const float m = acc[e] * (1.f / (QK_SCALE * QK_SCALE)) * ratio(s_log[i] - lj);
            (qk ? s_p : s_a)[i][j] = anc ? m * (qk ? 1.f : -s_beta[i]) : 0.f;
        }
    }
    __syncthreads();

    // the inverse of a diagonal block I + A, a column a lane
    if (w < nb) {
        float xi[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float s = i == col ? 1.f : 0.f;
#pragma unroll
            for (int m = 0; m < i; ++m) s = fmaf(s_a[16 * w + i][16 * w + m], xi[m], s);
            xi[i] = s;
        }
        if (g == 0)
#pragma unroll
            for (int i = 0; i < 16; ++i) s_inv[w][i][col] = xi[i];
    }
    // S0 k_i and S0 q_i: row 16 r + 4 g + e, state row 16 w + col. S0's terms are those of its rows with
    // their largest entries brought to [2^14, 2^15).
    float top = 0.f;
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(s0[c][e]));
    top = fmaxf(top, lane_xor(top, 16));
    top = fmaxf(top, lane_xor(top, 32));
    const int up = 14 - min(max(ilogb_bits(top), -100), 100);
    Terms st[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) split(s0[c] * pow2(up), st[c].hi, st[c].lo);
    const float down = pow2(-up) * (1.f / QK_SCALE);
    f32x4 wk[NB], wq[NB];
#pragma unroll
    for (int r = 0; r < NB; ++r) {
        wk[r] = wq[r] = (f32x4)(0.f);
        if (r < nb) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                wk[r] = mfma_terms(terms(s_k, 16 * r + col, c), st[c], wk[r]);
                wq[r] = mfma_terms(terms(s_q, 16 * r + col, c), st[c], wq[r]);
            }
            wk[r] *= down;
            wq[r] *= down;
        }
    }
    __syncthreads();
    for (int i = tid >> 4; i < n; i += GT_THREADS / 16) {
        f32x4 lo, hi;
        conv_of(conv, i, ch_v, lo, hi);
        *(f32x4*)(s_v[i] + ch8) = lo;
        *(f32x4*)(s_v[i] + ch8 + 4) = hi;
    }
    __syncthreads();

    f32x4 u[NB];
#pragma unroll
    for (int r = 0; r < NB; ++r) {
        u[r] = (f32x4)(0.f);
        if (r < nb) {
            f32x4 rhs, o;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = 16 * r + 4 * g + e;
                // (a place without a token adds nothing to others, whatever lies there)
                const bool here = s_up[i].w;
                const float gain = s_gain[i];
                rhs[e] = here ? s_beta[i] * (s_v[i][16 * w + col] - gain * wk[r][e]) : 0.f;
                o[e] = here ? gain * wq[r][e] : 0.f;
            }
#pragma unroll
            for (int c = 0; c < NB; ++c)
                if (c < r) {
                    const f32x4 av = *(const f32x4*)&s_a[16 * r + col][16 * c + 4 * g];
#pragma unroll
                    for (int e = 0; e < 4; ++e) rhs = mfma4(av[e], u[c][e], rhs);
                }
            const f32x4 iv = *(const f32x4*)&s_inv[r][col][4 * g];
#pragma unroll
            for (int e = 0; e < 4; ++e) u[r] = mfma4(iv[e], rhs[e], u[r]);
#pragma unroll
            for (int c = 0; c < NB; ++c)
                if (c <= r) {
                    const f32x4 pv = *(const f32x4*)&s_p[16 * r + col][16 * c + 4 * g];
#pragma unroll
                    for (int e = 0; e < 4; ++e) o = mfma4(pv[e], u[c][e], o);
                }
            // (this wave's columns of v, which no other wave reads)
#pragma unroll
            for (int e = 0; e < 4; ++e) s_v[16 * r + 4 * g + e][16 * w + col] = o[e] * out_scale;
        }
    }
    __syncthreads();

    // the gated norm of a row, 8 dims a lane of a DPP row
    const f32x4 w0 = *(const f32x4*)(norm_w + ch8), w1 = *(const f32x4*)(norm_w + ch8 + 4);
    for (int i = tid >> 4; i < T; i += GT_THREADS / 16) {
        const size_t row = (size_t)b * T + i;
        f16x8 out = (f16x8)(0);
        if (i < n && s_up[i].w) {
            const f16x8 gate = *(const f16x8*)(z + row * z_pitch + hv * GT_K + ch8);
            const f32x4 a = *(const f32x4*)(s_v[i] + ch8), c = *(const f32x4*)(s_v[i] + ch8 + 4);
            float o[8] = {a[0], a[1], a[2], a[3], c[0], c[1], c[2], c[3]}, ss = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) ss = fmaf(o[e], o[e], ss);
            const float inv = 1.f / sqrtf(row16_sum(ss) / (float)GT_K + norm_eps);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float gz = (float)gate[e];
                o[e] *= inv * (e < 4 ? w0[e] : w1[e - 4]) * (gz * __builtin_amdgcn_rcpf(1.f + hw_expf(-gz)));
            }
            out = f16_sat8(o);
        }
        *(f16x8*)(y + row * y_pitch + hv * GT_K + ch8) = out;
    }
}

// ---------------------------------------------------------------------------
// The state and the conv frames behind an accepted path, token by token: 32 state rows a
// workgroup, a row on 8 lanes (columns 4 l + 32 j .. + 3) in registers throughout, k and v of
// the path's tokens formed first. Reads and writes a state once: bound by that for a batch.
// ---------------------------------------------------------------------------
constexpr int GC_ROWS = 32, GC_THREADS = 256;

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

__global__ void __launch_bounds__(GC_THREADS)
gdn_commit_kernel(const f16* __restrict__ x, int x_stride, const f16* __restrict__ conv_w, const CommitSeqs seqs,
                  const int* __restrict__ path, const float* __restrict__ ga, const float* __restrict__ gb,
                  int ab_stride, const float* __restrict__ A_log, const float* __restrict__ dt_bias, int T, int D,
                  int n_kheads, int n_vheads, float l2eps) {
    __shared__ __attribute__((aligned(16))) float s_k[TREE_MAX][GT_K], s_v[TREE_MAX][GC_ROWS];
    __shared__ float s_beta[TREE_MAX], s_alpha[TREE_MAX];
    __shared__ int s_at[TREE_MAX], s_n;
    const int tid = threadIdx.x;
    constexpr int PARTS = GT_K / GC_ROWS;
    const int part = blockIdx.x % PARTS, hv = blockIdx.x / PARTS % n_vheads, b = blockIdx.x / PARTS / n_vheads;
    const int group = n_vheads / n_kheads, hk = hv / group;
    const bool fresh = seqs.pos0[b] == 0;

    // the state: row part GC_ROWS + tid / 8
    const size_t srow = ((size_t)hv * GT_K + part * GC_ROWS + (tid >> 3)) * GT_K + 4 * (tid & 7);
    f32x4 s[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) s[j] = *(const f32x4*)(seqs.S[b] + srow + 32 * j);

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
    __syncthreads();
    const int n = s_n;

    // Token d of the frames and the path as one row of tokens: d < 0 are frames.
    const f16* xb = x + (size_t)b * T * x_stride;
    auto row = [&](int d, int ch) { return xb + (size_t)s_at[max(d, 0)] * x_stride + ch; };
    auto put_frames = [&](f16x8 f0, f16x8 f1, f16x8 f2, int ch) {   // [channel][frame] of the last three
        const f16x8 x = token(3 - n, row(n - 3, ch), f0, f1, f2);
        const f16x8 y = token(2 - n, row(n - 2, ch), f0, f1, f2), z = token(1 - n, row(n - 1, ch), f0, f1, f2);
        f16x8* to = (f16x8*)(seqs.frames_out[b] + 3 * ch);
        to[0] = (f16x8){x[0], y[0], z[0], x[1], y[1], z[1], x[2], y[2]};
        to[1] = (f16x8){z[2], x[3], y[3], z[3], x[4], y[4], z[4], x[5]};
        to[2] = (f16x8){y[5], z[5], x[6], y[6], z[6], x[7], y[7], z[7]};
    };
    {   // k, a token on a DPP row
        const int ch8 = 8 * (tid & 15), ch = (n_kheads + hk) * GT_K + ch8;
        Conv8 c;
        c.load(conv_w, seqs.frames[b], fresh, ch);
        for (int d = tid >> 4; d < n; d += GC_THREADS / 16) {
            f32x4 lo, hi;
            const f16x8 x3 = token(3 - d, row(d - 3, ch), c.f0, c.f1, c.f2);
            const f16x8 x2 = token(2 - d, row(d - 2, ch), c.f0, c.f1, c.f2);
            const f16x8 x1 = token(1 - d, row(d - 1, ch), c.f0, c.f1, c.f2);
            c.apply(lo, hi, x3, x2, x1, *(const f16x8*)row(d, ch));
            const float inv = 1.f / sqrtf(row16_sum(sum_sq(lo, hi)) + l2eps);
            *(f32x4*)(s_k[d] + ch8) = lo * inv;
            *(f32x4*)(s_k[d] + ch8 + 4) = hi * inv;
        }
        if (hv == hk * group && part == 0 && tid < 32) {   // the frames of q and k, once a k head
            if (tid < 16) {
                put_frames(c.f0, c.f1, c.f2, ch);
            } else {
                c.load(conv_w, seqs.frames[b], fresh, hk * GT_K + ch8);
                put_frames(c.f0, c.f1, c.f2, hk * GT_K + ch8);
            }
        }
    }
    {   // this part's v, a token on 4 lanes
        const int ch8 = 8 * (tid & 3), ch = (2 * n_kheads + hv) * GT_K + part * GC_ROWS + ch8;
        Conv8 c;
        c.load(conv_w, seqs.frames[b], fresh, ch);
        for (int d = tid >> 2; d < n; d += GC_THREADS / 4) {
            f32x4 lo, hi;
            const f16x8 x3 = token(3 - d, row(d - 3, ch), c.f0, c.f1, c.f2);
            const f16x8 x2 = token(2 - d, row(d - 2, ch), c.f0, c.f1, c.f2);
            const f16x8 x1 = token(1 - d, row(d - 1, ch), c.f0, c.f1, c.f2);
            c.apply(lo, hi, x3, x2, x1, *(const f16x8*)row(d, ch));
            *(f32x4*)(s_v[d] + ch8) = lo;
            *(f32x4*)(s_v[d] + ch8 + 4) = hi;
        }
        if (tid < 4) put_frames(c.f0, c.f1, c.f2, ch);
    }
    __syncthreads();
    for (int d = 0; d < n; ++d) {
        f32x4 k[4];
        float m = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            k[j] = *(const f32x4*)(s_k[d] + 4 * (tid & 7) + 32 * j);
            s[j] *= s_alpha[d];
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

bool meet(const void* p, size_t np, const void* q, size_t nq) {
    return (uintptr_t)p < (uintptr_t)q + nq && (uintptr_t)q < (uintptr_t)p + np;
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
    TreeSeqs seqs = {};
    for (int i = 0; i < B; ++i) {
        seqs.S[i] = S[i];
        seqs.frames[i] = (const f16*)cst_in[i];
        seqs.pos0[i] = pos0[i];
    }
    auto kernel = T <= 16 ? gdn_tree_kernel<1> : T <= 32 ? gdn_tree_kernel<2> : T <= 48 ? gdn_tree_kernel<3>
                                                                                       : gdn_tree_kernel<4>;
    hipLaunchKernelGGL(kernel, dim3(B * n_vheads), dim3(GT_THREADS), 0, (hipStream_t)stream, (const f16*)x,
                       x_stride, (const f16*)conv_w, seqs, parents, a, b, ab_stride, A_log, dt_bias,
                       (const f16*)z, z_pitch, norm_w, (f16*)y, y_pitch, T, n_kheads, n_vheads, out_scale, l2eps,
                       norm_eps);
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
        }
        seqs.S[i] = S[i];
        seqs.S_out[i] = S_out[i];
        seqs.frames[i] = (const f16*)cst_in[i];
        seqs.frames_out[i] = (f16*)cst_out[i];
        seqs.pos0[i] = pos0[i];
    }
    hipLaunchKernelGGL(gdn_commit_kernel, dim3(B * n_vheads * (GT_K / GC_ROWS)), dim3(GC_THREADS), 0,
                       (hipStream_t)stream, (const f16*)x, x_stride, (const f16*)conv_w, seqs, path, a, b,
                       ab_stride, A_log, dt_bias, T, D, n_kheads, n_vheads, l2eps);
    return fl::check_launch("gdn_tree_commit");
}

}  // extern "C"
