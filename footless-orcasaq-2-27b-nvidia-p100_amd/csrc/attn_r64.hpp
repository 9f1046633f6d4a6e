// The pieces of the 64-query-rows-a-wave attention tile that the contiguous and the
// paged prefill kernels share: O^T accumulators in AGPRs, HBM -> LDS copies, the tile's
// swizzled layout and its V^T fragments.
#pragma once

#include "attn_pieces.hpp"
#include "fl_common.hpp"

namespace {

using fl::PF_HD;

constexpr int ROW_B = PF_HD * 2;       // bytes a K / V row
// A column's running max only moves when a tile's max exceeds it by more
// than this (log2 units): P = 2^(s - m) stays <= 256, exact in fp16 range,
// and the O / l rescale is skipped on almost every tile.
constexpr float RESCALE_LOG2 = 8.f;

// the chunk swizzle of tile row r: chunk c is stored at c ^ sw(r)
__device__ __forceinline__ int sw(int r) { return ((r & 3) << 2) | ((r >> 2) & 3); }

// The O^T accumulators live in AGPRs and are touched only through the asm
// below. With compiler-generated MFMAs O would be either in VGPRs (leaving no
// registers to read LDS ahead) or, in AGPRs, given a VGPR home because of the
// rare rescale and copied out of the accumulators on every tile. Hazards the
// compiler cannot see inside asm are covered here: s_nop 2 before each MFMA
// (a VALU write of an A / B operand needs two wait states before the MFMA
// reads it; without them the MFMA reads the register's previous contents),
// s_nop 2 between a VALU result and v_accvgpr_write of it, and acc_settle()
// before the accumulators are read (an MFMA result must leave the pipeline
// before v_accvgpr_read; 24 wait states cover the 8-pass MFMA). MFMAs that
// accumulate into the same registers back to back need no wait states.
__device__ __forceinline__ void acc_zero(f32x16& acc, const f16x8& zero) {
    asm volatile("s_nop 2\n\tv_mfma_f32_32x32x16_f16 %0, %1, %1, 0" : "=a"(acc) : "v"(zero));
}
__device__ __forceinline__ void acc_mfma(f32x16& acc, const f16x8& a, const f16x8& b) {
    asm("s_nop 2\n\tv_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+a"(acc) : "v"(a), "v"(b));
}
__device__ __forceinline__ void acc_settle(f32x16 (&o)[8]) {
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7"
                 : "+a"(o[0]), "+a"(o[1]), "+a"(o[2]), "+a"(o[3]), "+a"(o[4]), "+a"(o[5]),
                   "+a"(o[6]), "+a"(o[7]));
}
// a0..a3 *= c, on accumulator registers
__device__ __forceinline__ void scale4_acc(float& a0, float& a1, float& a2, float& a3, float c) {
    float t0, t1;
    asm volatile(
        "v_accvgpr_read_b32 %4, %0\n\t"
        "v_accvgpr_read_b32 %5, %1\n\t"
        "v_mul_f32 %4, %4, %6\n\t"
        "v_mul_f32 %5, %5, %6\n\t"
        "s_nop 2\n\t"
        "v_accvgpr_write_b32 %0, %4\n\t"
        "v_accvgpr_write_b32 %1, %5\n\t"
        "v_accvgpr_read_b32 %4, %2\n\t"
        "v_accvgpr_read_b32 %5, %3\n\t"
        "v_mul_f32 %4, %4, %6\n\t"
        "v_mul_f32 %5, %5, %6\n\t"
        "s_nop 2\n\t"
        "v_accvgpr_write_b32 %2, %4\n\t"
        "v_accvgpr_write_b32 %3, %5"
        : "+a"(a0), "+a"(a1), "+a"(a2), "+a"(a3), "=&v"(t0), "=&v"(t1)
        : "v"(c));
}
__device__ __forceinline__ void acc_scale(f32x16 (&o)[8], float c) {
    acc_settle(o);
#pragma unroll
    for (int mb = 0; mb < 8; ++mb)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            float x0 = o[mb][e], x1 = o[mb][e + 1], x2 = o[mb][e + 2], x3 = o[mb][e + 3];
            scale4_acc(x0, x1, x2, x3, c);
            o[mb][e] = x0;
            o[mb][e + 1] = x1;
            o[mb][e + 2] = x2;
            o[mb][e + 3] = x3;
        }
}

// One HBM -> LDS copy of 16 bytes a lane to LDS dst + IMM (+ 16 lane). m0 is
// set inside the asm from a wave-uniform base and an immediate, so the
// compiler keeps no per-copy LDS addresses in SGPRs (it would otherwise hoist
// all of them out of the tile loop); the asm declares m0 as its output, and that
// the s_add overwrites SCC: without that the compiler put a copy between the two
// halves of a 64-bit address add (s_add_u32 .. s_addc_u32) and the carry was
// lost, so a V cache whose rows cross a 4 GiB boundary of the address space was
// read 4 GiB below it (a memory fault, or another allocation's bytes).
template <int IMM>
__device__ __forceinline__ void copy16_at(const char* sbase, uint32_t voff, uint32_t dst) {
    uint32_t m0v;
    asm volatile("s_add_u32 m0, %3, %4\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 : "={m0}"(m0v)
                 : "v"(voff), "s"(sbase), "s"(dst), "i"(IMM)
                 : "scc");
}

constexpr int R64_BK = 32;                  // kv rows a tile
constexpr int R64_TILE = R64_BK * ROW_B;    // 16 KiB: K (or V) of a tile
constexpr int R64_STAGE = 2 * R64_TILE;     // K | V
// Tiles copied ahead and K fragments read ahead: 2, 3 and 4 tiles and 2, 3
// and 4 k-steps measured the same within noise at 8k and 32k.
constexpr int R64_DIST = 3;
constexpr int R64_KPF = 3;
constexpr int R64_NST = R64_DIST + 1;
constexpr int R64_LDS = R64_NST * R64_STAGE;   // 128 KiB at R64_DIST 3
static_assert(R64_LDS <= 160 * 1024, "R64_DIST: LDS <= 160 KiB");
constexpr int R64_COPIES = 8;               // copy instructions a wave a tile (4 K + 4 V)
// The 8 V^T fragments (ds_read_b64_tr_b16) of PV step n: k-step kq = n / 2
// (kv rows 16 kq ..), dim blocks 4 (n % 2) .. + 3; b: this lane's offsets
// (the troff of attn_prefill_kernel).
__device__ __forceinline__ void r64_vfrags(s16x4 (&vb)[8], const char* vt,
                                           const uint32_t (&b)[8], int n) {
    const int imm = 16 * ROW_B * (n >> 1) + 256 * (n & 1);
#pragma unroll
    for (int i = 0; i < 8; ++i)
        vb[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(vt + b[i] + imm));
}

}  // namespace
