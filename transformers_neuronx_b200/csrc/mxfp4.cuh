// Microscaled 4-bit numbers (MXFP4), as every kernel here reads them.
//
// A row of K values is ceil(K / 32) blocks of 32 neighbouring values (the last one filled up with zeros).  A block has a scale byte
// E, the power of two 2^(E - 127), and 32 codes of 4 bits, e2m1: a sign, then one of 0, 0.5, 1, 1.5, 2, 3, 4, 6.  Value = code * 2^(E - 127).
//   codes  [rows][blocks * 16] bytes, value 2j of the row in the low half of byte j;   scales [rows][blocks] bytes.
// E = 255 says that the block held something that is no finite number: all 32 values are NaN.
#pragma once
#include "common.cuh"

namespace {

constexpr int MX_BLOCK = 32;

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
    uint32_t r;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
    return r;
}

// 2^(E - 127) as a 32-bit float, exactly: E = 0 is 2^-127, half of the smallest normal number.
__device__ __forceinline__ float mx_scale(uint32_t E) {
    return E == 255u ? __uint_as_float(0x7FC00000u) : __uint_as_float(E ? E << 23 : 0x00400000u);
}
// One code as a 32-bit float: its three bits of magnitude as the last bit of the exponent field's two and the first of the fraction are
// the value times 2^-126 (a subnormal number for 0.5), so one exact multiplication is left.
__device__ __forceinline__ float mx_code(uint32_t c) {
    return __uint_as_float(((c & 8u) << 28) | ((c & 7u) << 22)) * 8.507059173023462e37f;
}

// The eight magnitudes of a block times its scale in the 16-bit type, their high and low bytes apart: a byte permutation then looks
// four codes up at once.  What 16 bits cannot hold exactly is rounded here (bfloat16: only beyond 2^127 and below 2^-133, where no
// matrix's block lies that this library made from finite numbers but the largest; float16: see `shift`).
struct MxTable { uint32_t h0, h1, l0, l1; };

#ifdef TNX_F16
// The scale relative to the largest of its row, `ref`: 2^(E - ref + 13), so that 6 * 2^13 is the largest magnitude and blocks down to
// 2^-36 of the row's largest scale keep every bit in float16's normal and subnormal numbers; the rest of the scale is the row's (mx_row_factor).
constexpr int MX_F16_TOP = 13;
__device__ __forceinline__ uint32_t mx_scale_h16(uint32_t E, int ref) {
    const int d = (int)E - ref + MX_F16_TOP;
    uint32_t b = d >= -14 ? (uint32_t)(d + 15) << 10 : d >= -24 ? 1u << (d + 24) : 0u;
    if (E == 255u) b = 0x7E00u;
    return b | (b << 16);
}
#define MX_PAIR_0_1 0x38000000u          /* 0.5 : 0   */
#define MX_PAIR_2_3 0x3E003C00u          /* 1.5 : 1   */
#define MX_PAIR_4_5 0x42004000u          /* 3   : 2   */
#define MX_PAIR_6_7 0x46004400u          /* 6   : 4   */
#else
__device__ __forceinline__ uint32_t mx_scale_h16(uint32_t E, int) {
    uint32_t b = E ? E << 7 : 0x0040u;
    if (E == 255u) b = 0x7FC0u;
    return b | (b << 16);
}
#define MX_PAIR_0_1 0x3F000000u
#define MX_PAIR_2_3 0x3FC03F80u
#define MX_PAIR_4_5 0x40404000u
#define MX_PAIR_6_7 0x40C04080u
#endif
__device__ __forceinline__ uint32_t mul_h16x2(uint32_t a, uint32_t b) {
    h16x2 r = __hmul2(*(h16x2*)&a, *(h16x2*)&b);
    return *(uint32_t*)&r;
}
__device__ __forceinline__ MxTable mx_table(uint32_t E, int ref) {
    const uint32_t s = mx_scale_h16(E, ref);
    const uint32_t p0 = mul_h16x2(MX_PAIR_0_1, s), p1 = mul_h16x2(MX_PAIR_2_3, s), p2 = mul_h16x2(MX_PAIR_4_5, s), p3 = mul_h16x2(MX_PAIR_6_7, s);
    MxTable t;
    t.l0 = prmt(p0, p1, 0x6420); t.h0 = prmt(p0, p1, 0x7531);
    t.l1 = prmt(p2, p3, 0x6420); t.h1 = prmt(p2, p3, 0x7531);
    return t;
}
// Eight codes -> eight 16-bit values in their order: 17 instructions with the table's share (two lookups of four magnitudes' high bytes and
// low bytes each, the signs spread by the permutation's sign mode, bytes put together).
__device__ __forceinline__ void mx_decode8(uint32_t w, const MxTable& t, uint32_t& o0, uint32_t& o1, uint32_t& o2, uint32_t& o3) {
    const uint32_t s = w & 0x77777777u, s2 = s >> 16, w4 = w << 4;
    const uint32_t ha = prmt(t.h0, t.h1, s) | (prmt(w, w4, 0x9D8C) & 0x80808080u), la = prmt(t.l0, t.l1, s);
    const uint32_t hb = prmt(t.h0, t.h1, s2) | (prmt(w, w4, 0xBFAE) & 0x80808080u), lb = prmt(t.l0, t.l1, s2);
    o0 = prmt(la, ha, 0x5140); o1 = prmt(la, ha, 0x7362);
    o2 = prmt(lb, hb, 0x5140); o3 = prmt(lb, hb, 0x7362);
}

}  // namespace
