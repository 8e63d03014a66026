// Layout of a 4-bit matrix with group scales, and its device-side decoding.
//
// W[n, k] = s[n, k / G] * (q[n, k] - z[n, k / G]): q and z whole numbers from 0 to 15
// (z is 8 everywhere in a matrix without zero points), s bf16 or fp16, G = 32,
// 64 or 128 inputs.  It is laid out for the matrix cores: weights are the first operand of
// v_mfma_f32_16x16x32_bf16, of which lane l = r + 16 g holds row r and the inputs
// 8 g .. + 7 of 32.
//
// Unit: 16 rows x 128 inputs, units of a 16-row tile behind one another (inputs
// fastest), rows and inputs past the matrix' end with q, z and s of 0:
//   codes (1024 bytes): lane l's 16 bytes at 16 l; word j holds row r, inputs
//     32 j + 8 g + 0..7, input b (b < 4) in the low and input 4 + b in the high half of byte b;
//   scales (16 bits): rows 4 g .. + 3 of each group in turn, for each g in turn, as
//     an accumulator's lane reads them;
//   zero points (bytes), where there are any: likewise.
#pragma once

#include "common.h"

namespace pd {

constexpr int kI4Rows = 16, kI4In = 128, kI4Codes = 1024;

__host__ __device__ constexpr int i4_unit_bytes(int G, bool zeros) {
    return kI4Codes + (kI4In / G) * (zeros ? 48 : 32);
}
__host__ __device__ inline int64_t i4_units(int N, int K) {
    return (int64_t)((N + kI4Rows - 1) / kI4Rows) * ((K + kI4In - 1) / kI4In);
}
inline bool i4_shape_ok(int N, int K, int G) {
    return N >= 1 && K >= G && (G == 32 || G == 64 || G == 128) && K % G == 0 && K <= (1 << 20) && N <= (1 << 24);
}

// Where a row's scale of the unit's group gi lies, and its zero point
template <typename T = int>
__host__ __device__ inline T i4_scale_at(T r, T gi, T groups) { return kI4Codes + ((r / 4) * groups + gi) * 8 + r % 4 * 2; }
template <typename T = int>
__host__ __device__ inline T i4_zero_at(T r, T gi, T groups) {
    return kI4Codes + groups * 32 + ((r / 4) * groups + gi) * 4 + r % 4;
}

// The eight whole numbers of a word of codes as bf16, exactly: the bytes 0 to 15
// are the e4m3 codes of 0 to 15 times 2^-9 (eight subnormal numbers, then the first
// binade with the same step), so the 8-bit converters with a scale of 2^9 read
// them as they are, two a piece.
__device__ __forceinline__ bf16x8_t i4_decode(uint32_t codes) {
    const uint32_t lo = codes & 0x0f0f0f0fu, hi = (codes >> 4) & 0x0f0f0f0fu;
    const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.0f, false);
    const bf16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.0f, true);
    const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.0f, false);
    const bf16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.0f, true);
    return bf16x8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Eight codes, input i in bits 4 i .. + 3, in the order of a unit's word.
__device__ __forceinline__ uint32_t i4_order(uint32_t w) {
    uint32_t o = 0;
#pragma unroll
    for (int b = 0; b < 4; ++b) o |= (w >> (4 * b) & 15u) << (8 * b) | (w >> (4 * b + 16) & 15u) << (8 * b + 4);
    return o;
}

// A 16-bit scale, widened
__device__ __forceinline__ float i4_scale(uint32_t h16, bool fp16) {
    return fp16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)h16) : bf2f(h16);
}

// The scales and zero points of rows 4 g .. + 3 of a unit.
template <int G, bool ZEROS, bool FP16>
struct I4Side {
    static constexpr int GP = kI4In / G;
    uint32_t s[2 * GP], z[GP];
    __device__ __forceinline__ void load(const uint8_t *unit, int g) {
        const uint8_t *at = unit + kI4Codes + g * (GP * 8), *zt = unit + kI4Codes + GP * 32 + g * (GP * 4);
        if constexpr (GP == 1) {
            const uint2 a = *reinterpret_cast<const uint2 *>(at);
            s[0] = a.x, s[1] = a.y;
            if (ZEROS) z[0] = *reinterpret_cast<const uint32_t *>(zt);
        } else {
#pragma unroll
            for (int i = 0; i < GP / 2; ++i) {
                const uint4 a = ld_g(at + 16 * i);
                s[4 * i] = a.x, s[4 * i + 1] = a.y, s[4 * i + 2] = a.z, s[4 * i + 3] = a.w;
            }
            if constexpr (ZEROS && GP == 2) {
                const uint2 a = *reinterpret_cast<const uint2 *>(zt);
                z[0] = a.x, z[1] = a.y;
            } else if constexpr (ZEROS) {
                const uint4 a = ld_g(zt);
                z[0] = a.x, z[1] = a.y, z[2] = a.z, z[3] = a.w;
            }
        }
    }
    __device__ __forceinline__ float scale(int gi, int q) const {
        const uint32_t w = s[2 * gi + (q >> 1)];
        if (FP16) return (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> (16 * (q & 1))));
        return q & 1 ? hi_bf(w) : lo_bf(w);
    }
    __device__ __forceinline__ float zero(int gi, int q) const { return ZEROS ? (float)(z[gi] >> (8 * q) & 255u) : 8.0f; }
};

}  // namespace pd
