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

// The products' activations (common.cuh), but for a sum that is NaN, as the values of a block of scale byte 255 make it: it stays NaN behind relu and its
// square too.
__device__ __forceinline__ float mx_activation(float v, int act) {
    if (act != TNX_ACT_RELU && act != TNX_ACT_RELU2) return apply_activation(v, act);
    float r;
    asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r) : "f"(v));
    return act == TNX_ACT_RELU ? r : r * r;
}

// Eight codes as eight float16 numbers, without a scale.
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t (&o)[4]) {
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3]) : "r"(w));
}

__device__ __forceinline__ uint32_t mul_h16x2(uint32_t a, uint32_t b) {
    h16x2 r = __hmul2(*(h16x2*)&a, *(h16x2*)&b);
    return *(uint32_t*)&r;
}

// A block's codes -> 16-bit values, code times scale, eight at a time in their order.
#ifdef TNX_F16
// float16: the conversion e2m1x2 -> f16x2 and a multiplication, by the scale relative to the largest of its row, `ref`: 2^(E - ref + 13), so that
// 6 * 2^13 is the largest value and blocks down to 2^-36 of the row's largest scale keep every bit in float16's normal and
// subnormal numbers; the rest of the scale is a factor of the row's sums.
constexpr int MX_F16_TOP = 13;
struct MxValues {
    uint32_t s;
    __device__ __forceinline__ MxValues(uint32_t E, int ref) {
        const int d = (int)E - ref + MX_F16_TOP;
        uint32_t b = d >= -14 ? (uint32_t)(d + 15) << 10 : d >= -24 ? 1u << (d + 24) : 0u;
        if (E == 255u) b = 0x7E00u;
        s = b | (b << 16);
    }
    __device__ __forceinline__ void decode8(uint32_t w, uint32_t* o) const {
        uint32_t c[4];
        codes_to_f16(w, c);
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = mul_h16x2(c[j], s);
    }
};
#else
// bfloat16: the eight magnitudes times the scale are a table, high and low bytes apart; a byte permutation looks four codes up at once, signs
// are spread by the permutation's sign mode, bytes put together: 17 instructions for eight values with the table's share.  Every value is
// exact but those beyond 2^127 and below 2^-133.
struct MxValues {
    uint32_t h0, h1, l0, l1;
    __device__ __forceinline__ MxValues(uint32_t E, int) {
        uint32_t s = E ? E << 7 : 0x0040u;
        if (E == 255u) s = 0x7FC0u;
        s |= s << 16;
        const uint32_t p0 = mul_h16x2(0x3F000000u, s), p1 = mul_h16x2(0x3FC03F80u, s), p2 = mul_h16x2(0x40404000u, s), p3 = mul_h16x2(0x40C04080u, s);
        l0 = prmt(p0, p1, 0x6420); h0 = prmt(p0, p1, 0x7531);
        l1 = prmt(p2, p3, 0x6420); h1 = prmt(p2, p3, 0x7531);
    }
    __device__ __forceinline__ void decode8(uint32_t w, uint32_t* o) const {
        const uint32_t s = w & 0x77777777u, s2 = s >> 16, w4 = w << 4;
        const uint32_t ha = prmt(h0, h1, s) | (prmt(w, w4, 0x9D8C) & 0x80808080u), la = prmt(l0, l1, s);
        const uint32_t hb = prmt(h0, h1, s2) | (prmt(w, w4, 0xBFAE) & 0x80808080u), lb = prmt(l0, l1, s2);
        o[0] = prmt(la, ha, 0x5140); o[1] = prmt(la, ha, 0x7362);
        o[2] = prmt(lb, hb, 0x5140); o[3] = prmt(lb, hb, 0x7362);
    }
};
#endif

}  // namespace
