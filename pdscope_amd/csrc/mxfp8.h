// 8-bit rows: activations as e4m3 codes (finite magnitudes up to 448) with one e8m0
// scale 2^(byte - 127) per 32 consecutive channels, 33/32 byte a value, both
// row-major: codes [rows, n], scales [rows, n / 32].
//
// The scale is the smallest power of two, from 2^-127 on, that brings the
// block's largest magnitude to at most 448: no value is clamped, and the largest
// one keeps at least three of its four significant bits' steps below 448 / 2.  A
// block with an infinity or NaN has the byte 255, which makes all of it NaN.
#pragma once

#include "common.h"

namespace pd {

// max of the values of the four lanes of an aligned quad, in each of them
__device__ __forceinline__ uint32_t max_over_quad(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xb1, 0xf, 0xf, true));  // quad_perm [1,0,3,2]
    return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4e, 0xf, 0xf, true));  // quad_perm [2,3,0,1]
}

// max of the values of lanes l, l ^ 16, l ^ 32 and l ^ 48, in each of them
__device__ __forceinline__ uint32_t max_over_quarters(uint32_t v) {
    const auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = max(a[0], a[1]);
    const auto b = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return max(b[0], b[1]);
}

// the largest magnitude of eight values, as its bits (NaN above everything)
__device__ __forceinline__ uint32_t top_magnitude8(const float (&v)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    return m;
}

// The scale byte of a block whose largest magnitude has these bits: 448 is 1.75 *
// 2^8, so 8 below its exponent field, one more where its mantissa is above 1.75.
__device__ __forceinline__ uint32_t mx8_scale_byte(uint32_t top) {
    if (top >= 0x7f800000u) return 255u;
    const uint32_t ex = (top + 0x1fffffu) >> 23;
    return ex > 8u ? ex - 8u : 0u;
}

// Codes of eight values of a block with this scale byte, first value in the
// lowest byte: the nearest code to value / scale (exact in 32 bits, or far below the smallest code), ties
// to the even one.  Zeros where the block is NaN.
__device__ __forceinline__ uint2 mx8_encode8(const float (&v)[8], uint32_t byte) {
    if (byte == 255u) return make_uint2(0u, 0u);
    const float inv = __uint_as_float((254u - byte) << 23);
    int lo = 0, hi = 0;
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, lo, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, lo, true);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4] * inv, v[5] * inv, hi, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6] * inv, v[7] * inv, hi, true);
    return make_uint2((uint32_t)lo, (uint32_t)hi);
}

// Eight 64-bit values cut to 32 bits, with the last bit set where anything was cut
// off: rounding them further to a type of fewer bits gives what rounding the
// values themselves would.  Below fp32's normal numbers the last bit is a step of
// 2^-149; one branch for all eight (4096 rows of 2048 with the merge and the way back
// 45.6 us, 47.9 with a choice for each value).
__device__ __forceinline__ void round_to_odd8(const double (&v)[8], float (&o)[8]) {
    uint64_t u[8];
    uint32_t least = ~0u;  // the upper halves without their signs, whose order is that of the magnitudes
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        u[i] = (uint64_t)__double_as_longlong(v[i]);
        least = min(least, (uint32_t)(u[i] >> 32) & 0x7fffffffu);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint64_t cut = u[i] & 0x1fffffffull;
        o[i] = (float)__longlong_as_double((long long)((u[i] - cut) | (cut ? 0x20000000ull : 0ull)));
    }
    if (least < 0x38100000u) {  // of 2^-126
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const double steps = fabs(v[i]) * 0x1p149;
            const uint32_t whole = (uint32_t)steps;
            const uint32_t odd = whole | (uint32_t)((double)whole != steps) | (uint32_t)(u[i] >> 32 & 0x80000000u);
            if (fabs(v[i]) < 0x1p-126) o[i] = __uint_as_float(odd);
        }
    }
}

}  // namespace pd
