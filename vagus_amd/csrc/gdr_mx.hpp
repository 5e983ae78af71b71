// Block-scaled numbers: the formats, and the rounding to them that every kernel shares.
//
// A block is 32 consecutive elements of a row and one scale 2^(b - 127), held as the byte b in 1 .. 254.
// b = 255 marks a block that had a NaN or an infinity: all its values are NaN.  8 bits are e4m3
// (largest 448), 4 bits e2m1 (0, 1/2, 1, 3/2, 2, 3, 4, 6 and their negatives).  The scale is the smallest 2^s,
// s >= -126, with amax <= 464 2^s (8 bits) or 7 2^s (4 bits): half a step above the format's
// largest value, so that the block's largest element is off by half a step at most, as every other; a scale
// twice as large would cost all others a bit.  Elements are rounded to nearest, ties to even, the ends saturate.
// s >= -126 keeps every scale and its inverse a normal fp32 number; a block of zeros has b = 1.  4 bits: s <= 125, so that
// every weight is a finite bf16 number (6 2^125 = 1.5 2^127, where what is larger ends): as 4 2^126 the largest
// fp32 numbers would be infinities, and NaN to a row of zeros.
//
// Rows in 8 bits: values [rows, 128 ceil(K / 128)] and bytes [rows, 4 ceil(K / 128)]; the padding is zeros with b = 1.
//
// 4-bit weights [n, K]: tiles of 16 rows x 128 columns, a KB each in the order in which a wave's
// lanes read it: values [T][C][g 0..3][r 0..15][16 bytes], lane 16 g + r holding row 16 t + r, columns 128 c + 32 g
// .. + 31, the even column in a byte's low half; C = ceil(K / 128).  Scale bytes [T][ceil(C / 4)][g][r][c mod 4].
// T = ceil(n / 16), or for a gated pair of n / 2 rows each (the FFN's two input projections) 2 ceil(n / 2 / 16): tile
// 2 i holds rows 16 i .. of the first half, tile 2 i + 1 the same rows of the second, so that a wave that
// owns both has a row's two products in the same lane.  The padding is zeros with b = 1.
#pragma once

#include "gdr_common.hpp"

namespace vgdr {

typedef int i32x8 __attribute__((ext_vector_type(8)));

// The biased scale of a block from its largest |x|, as fp32 bits: half a step above the largest value is
// 1.8125 2^8 (8 bits) or 1.75 2^2 (4 bits), so the exponent moves up where the mantissa passes that.
template <int BITS>
__device__ __forceinline__ int mx_scale(uint32_t amax) {
    constexpr uint32_t HALF = BITS == 8 ? 0x680000u : 0x600000u;
    constexpr int TOP = BITS == 8 ? 8 : 2;
    if (amax >= 0x7f800000u) return 255;
    const int b = (int)(amax >> 23) - TOP + ((amax & 0x7fffffu) > HALF ? 1 : 0);
    return b < 1 ? 1 : BITS == 4 && b > 252 ? 252 : b;
}
// 2^-(b - 127), for b in 1 .. 253
__device__ __forceinline__ float mx_inverse(int b) { return __builtin_bit_cast(float, (uint32_t)(254 - b) << 23); }
// 2^(b - 127), NaN for 255
__device__ __forceinline__ float mx_value(int b) {
    return __builtin_bit_cast(float, b == 255 ? 0x7fc00000u : (uint32_t)b << 23);
}

__device__ __forceinline__ uint32_t abs_bits(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7fffffffu; }

// four values of a block with scale byte b as e4m3; NaN's code where the block is none
__device__ __forceinline__ uint32_t mx_pack8(const float *x, int b) {
    if (b == 255) return 0x7f7f7f7fu;
    const float inv = mx_inverse(b);
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = fminf(fmaxf(x[e] * inv, -448.f), 448.f);
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], w, true);
}

// x to fp32 so that rounding it again, to fewer bits, gives what rounding x itself would: towards zero,
// with the last bit set where that was not exact.  Comparisons with numbers of fewer bits stay x's too.
__device__ __forceinline__ float round_to_odd(double x) {
    const float f = (float)x;
    uint32_t u = __builtin_bit_cast(uint32_t, f);
    if ((double)f != x && x == x) {
        u -= fabs((double)f) > fabs(x) ? 1u : 0u;
        u |= 1u;
    }
    return __builtin_bit_cast(float, u);
}

// v as the sum of P bf16 numbers: cut off, not rounded, so that the largest fp32 numbers stay finite; an infinity or a
// NaN is the first part's.  bf16 has 8 bits: fp16's 11 take two parts, fp32's 24 three.  What lies below bf16's least, 2^-133, is cut.
template <int P>
__device__ __forceinline__ void split(__bf16 (&out)[P], float v) {
    uint32_t u = __builtin_bit_cast(uint32_t, v);
    const bool finite = (u & 0x7f800000u) != 0x7f800000u;
    out[0] = finite ? __builtin_bit_cast(__bf16, (uint16_t)(u >> 16)) : (__bf16)v;
    float left = finite ? v - __builtin_bit_cast(float, u & 0xffff0000u) : 0.f;
#pragma unroll
    for (int q = 1; q < P; ++q) {
        u = __builtin_bit_cast(uint32_t, left);
        out[q] = __builtin_bit_cast(__bf16, (uint16_t)(u >> 16));
        left -= __builtin_bit_cast(float, u & 0xffff0000u);
    }
}

}  // namespace vgdr
