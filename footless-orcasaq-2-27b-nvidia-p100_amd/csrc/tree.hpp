// Trees of drafted tokens: what the attention and the GDN kernels take from parents.
//
// Token i < T of a sequence has the parent parents[i], an earlier token or -1 (a child of
// the context). Any other entry is a place that holds no token, and so is one whose parent
// holds none.
#pragma once

#include "fl_common.hpp"

namespace {

constexpr int TREE_MAX = FL_TREE_MAX;

__device__ __forceinline__ int lane_of(int v, int from) {   // v of lane `from`
    return __builtin_amdgcn_ds_bpermute(from << 2, v);
}
__device__ __forceinline__ float lane_of(float v, int from) {
    return __int_as_float(lane_of(__float_as_int(v), from));
}
__device__ __forceinline__ double lane_of(double v, int from) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = lane_of((int)(uint32_t)u, from), hi = lane_of((int)(uint32_t)(u >> 32), from);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// Lane i's token: its parent (-1 where there is none), its ancestors and itself as bits (none
// where it holds no token).
struct Node {
    int parent;
    uint32_t lo, hi;
    __device__ __forceinline__ bool here() const { return (lo | hi) != 0; }
    __device__ __forceinline__ int depth() const { return __popc(lo) + __popc(hi) - 1; }
};

// Of a whole wave. Every round a token takes over what the token `up` has gathered and that
// one's own `up`: 2^r ancestors after r rounds, as many rounds as the tree is deep in bits.
// `sum`, if there is one, becomes its sum over the path to the token, itself included.
template <bool SUM>
__device__ __forceinline__ Node tree_node(int p, int T, double* sum = nullptr) {   // p: lane i's parents[i]
    const int i = threadIdx.x & 63;
    if (i >= T) p = -2;
    const bool ok = p >= -1 && p < i;
    Node n = {ok ? p : -1, i < 32 ? 1u << i : 0u, i < 32 ? 0u : 1u << (i - 32)};
    int up = n.parent, lost = !ok;
    while (__any(up >= 0)) {
        const int from = up >= 0 ? up : i;
        const uint32_t lo = lane_of((int)n.lo, from), hi = lane_of((int)n.hi, from);
        const int l = lane_of(lost, from), u = lane_of(up, from);
        double s = 0.;
        if constexpr (SUM) s = lane_of(*sum, from);
        if (up >= 0) {
            n.lo |= lo, n.hi |= hi, lost |= l, up = u;
            if constexpr (SUM) *sum += s;
        }
    }
    if (lost) n.lo = n.hi = 0, n.parent = -1;
    return n;
}

// Do np bytes at p and nq bytes at q have any in common? (on the host)
inline bool meet(const void* p, size_t np, const void* q, size_t nq) {
    return (uintptr_t)p < (uintptr_t)q + nq && (uintptr_t)q < (uintptr_t)p + np;
}
// Rows: n of `width` bytes, `pitch` apart. Rows of one pitch may lie between each other.
struct RowsOf {
    const void* p;
    size_t n, pitch, width;
    size_t bytes() const { return (n - 1) * pitch + width; }
};
inline bool meet(const RowsOf& a, const RowsOf& b) {
    if (!meet(a.p, a.bytes(), b.p, b.bytes())) return false;
    if (a.pitch != b.pitch) return true;
    const RowsOf &lo = (uintptr_t)a.p <= (uintptr_t)b.p ? a : b, &hi = &lo == &a ? b : a;
    const size_t at = ((uintptr_t)hi.p - (uintptr_t)lo.p) % lo.pitch;
    return at < lo.width || at + hi.width > lo.pitch;
}

}  // namespace
