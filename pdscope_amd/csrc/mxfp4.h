// Layout of a 4-bit expert block and its device-side decoding.
//
// A block holds the expert's weights in microscaled 4-bit floating point: e2m1
// values (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) with one e8m0 scale
// 2^(byte - 127) per 32 consecutive inputs of a row, 4.25 bits a weight.  It is
// laid out for the matrix cores: weights are the first operand of
// v_mfma_f32_16x16x32_bf16, of which lane l holds row l % 16 and the inputs
// 8 (l / 16) .. + 7, so a lane's 16-byte load brings it one such piece (4
// bytes of codes) of four 16-row tiles, already in its place.
//
// Group: 64 rows x 128 inputs, kGroupBytes = 4352 bytes:
//   piece jj = 0..3 (32 inputs, 1024 bytes): lane l's 16 bytes at 16 l; word i
//     holds the codes of row 16 i + l % 16, inputs 32 jj + 8 (l / 16) + 0..7,
//     input n in bits 4n .. 4n + 3;
//   scales (256 bytes at 4096): byte (r * 4 + jj) * 4 + i is that of row
//     16 i + r, inputs 32 jj .. + 31.
// Gate/up matrix: I / 32 row groups x H / 128 input groups (inputs fastest);
// row group c has rows 0..31 = gate rows 32c .. 32c + 31, rows 32..63 = the same
// up rows, so one wave's accumulators pair for the SwiGLU.
// Down matrix, behind it: H / 64 row groups x I / 128 input groups.
#pragma once

#include "common.h"

namespace pd {

constexpr int kGroupRows = 64, kGroupIn = 128;
constexpr int kGroupScales = 4096;
constexpr int kGroupBytes = kGroupScales + 256;

__host__ __device__ inline size_t mx_gateup_groups(int H, int I) { return (size_t)(I / 32) * (H / kGroupIn); }
__host__ __device__ inline size_t mx_down_groups(int H, int I) { return (size_t)(H / kGroupRows) * (I / kGroupIn); }
__host__ __device__ inline size_t mx_block_bytes(int H, int I) {
    return (mx_gateup_groups(H, I) + mx_down_groups(H, I)) * kGroupBytes;
}
inline bool mx_shape_ok(int H, int I) { return H >= 128 && H % 128 == 0 && I >= 128 && I % 128 == 0; }

// A float whose exponent field is byte B of w (the conversions below read
// nothing else of their scale: 0 is 2^-127, 255 makes every value NaN).
template <int B>
__device__ __forceinline__ float mx_scale(uint32_t w) {
    return __uint_as_float(B == 0 ? w << 23 : B == 1 ? w << 15 : B == 2 ? w << 7 : w >> 1);
}

// The eight values of a word of codes, times the scale, as bf16.  Exact below
// 2^128: two significant bits, and bf16 has the exponents of e8m0 and more below.
// From there on (scale bytes 253 and 254, which quantising never gives, with
// codes of 4 and 2 up) they are infinite.
__device__ __forceinline__ bf16x8_t mx_decode(uint32_t codes, float scale) {
    const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0);
    const bf16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1);
    const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2);
    const bf16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3);
    return bf16x8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

}  // namespace pd
