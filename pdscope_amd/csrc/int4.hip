// 4-bit matrices with group scales (int4.h): from a checkpoint's tensors, from
// bf16 matrices, and back.  No counterpart in the reference, which has no
// quantised weights.
//
// One wave per unit, lane l = r + 16 g on the words that it owns: row r, inputs 32 j
// + 8 g .. + 7.  Bound by memory: 2 bytes a value on the bf16 side, a little over half
// a byte on the other.  4096 x 4096, G = 128: pack 7.9 us (2.2 TB/s), quantize 14.9 (2.8), dequantize
// 11.2 (3.8); done once a model.
#include "int4.h"

namespace pd {

struct I4Shape {
    int N, K, KU;   // KU: units of a row tile
    int64_t units;
    int64_t row;    // of the lane
    int u;          // of the wave
    __device__ __forceinline__ bool find(int64_t *unit) {
        *unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
        if (*unit >= units) return false;
        const int64_t nt = *unit / KU;
        u = (int)(*unit - nt * KU);
        row = nt * kI4Rows + (threadIdx.x & 15);
        return true;
    }
};

// Checkpoint: codes [N, K/2] (input 2i of a row in the low half of byte i), scales
// [N, K/G], zero points [N, K/G] or null.  Moves bits only.
__global__ __launch_bounds__(256) void i4_pack_kernel(const uint8_t *__restrict__ codes,
                                                      const uint16_t *__restrict__ scales,
                                                      const uint8_t *__restrict__ zeros, int G, I4Shape s,
                                                      uint8_t *__restrict__ out) {
    int64_t unit;
    if (!s.find(&unit)) return;
    const int lane = lane_id(), g = lane >> 4;
    uint8_t *dst = out + unit * i4_unit_bytes(G, zeros != nullptr);
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int k = s.u * kI4In + 32 * j + 8 * g;
        w[j] = s.row < s.N && k < s.K ? i4_order(*reinterpret_cast<const uint32_t *>(codes + s.row * (s.K / 2) + k / 2)) : 0;
    }
    *reinterpret_cast<uint4 *>(dst + 16 * lane) = make_uint4(w[0], w[1], w[2], w[3]);
    const int groups = kI4In / G, per_row = s.K / G;
    if (g < groups) {
        const int at = s.u * groups + g;
        const bool in = s.row < s.N && at < per_row;
        *reinterpret_cast<uint16_t *>(dst + i4_scale_at(lane & 15, g, groups)) = in ? scales[s.row * per_row + at] : (uint16_t)0;
        if (zeros) dst[i4_zero_at(lane & 15, g, groups)] = in ? zeros[s.row * per_row + at] & 15 : 0;
    }
}

__device__ __forceinline__ float max_quarters(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}

// bf16 [N, K] -> units.  A group with the values lo .. hi: without zero points s =
// bf16(max|w| / 7) and z = 8, with them s = bf16((max(hi, 0) - min(lo, 0)) / 15) and z
// = round(-min(lo, 0) / s); q = round(w / s) + z, cut to 0 .. 15 (a group of zeros has q = z).
template <int G, bool ZEROS>
__global__ __launch_bounds__(256) void i4_quantize_kernel(const uint16_t *__restrict__ weight, I4Shape s,
                                                          uint8_t *__restrict__ out) {
    int64_t unit;
    if (!s.find(&unit)) return;
    constexpr int GP = kI4In / G, JG = 4 / GP;  // groups of a unit, words of a group
    const int lane = lane_id(), g = lane >> 4;
    uint8_t *dst = out + unit * i4_unit_bytes(G, ZEROS);
    float v[4][8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int k = s.u * kI4In + 32 * j + 8 * g;
        uint4 q = make_uint4(0, 0, 0, 0);
        if (s.row < s.N && k < s.K) q = ld_g(weight + s.row * s.K + k);
        const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[j][2 * i] = lo_bf(u[i]);
            v[j][2 * i + 1] = hi_bf(u[i]);
        }
    }
    uint32_t w[4];
#pragma unroll
    for (int gi = 0; gi < GP; ++gi) {
        float top = 0.0f, bottom = 0.0f;  // the largest w, or |w|, and the largest -w, from 0 on
#pragma unroll
        for (int j = gi * JG; j < (gi + 1) * JG; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                top = fmaxf(top, ZEROS ? v[j][i] : fabsf(v[j][i]));
                bottom = fmaxf(bottom, -v[j][i]);
            }
        top = max_quarters(top);
        bottom = max_quarters(bottom);
        // halves, which bf16 values have exactly: the span itself may be past fp32's largest number
        const uint32_t s16 = f2bf(ZEROS ? (0.5f * top + 0.5f * bottom) / 7.5f : top / 7.0f);
        const float sc = bf2f(s16);
        const float z = !ZEROS ? 8.0f : sc > 0.0f ? fminf(rintf(bottom / sc), 15.0f) : 0.0f;
#pragma unroll
        for (int j = gi * JG; j < (gi + 1) * JG; ++j) {
            uint32_t c = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float q = sc > 0.0f ? rintf(v[j][i] / sc) + z : z;
                c |= (uint32_t)fminf(fmaxf(q, 0.0f), 15.0f) << (4 * i);
            }
            const bool in = s.row < s.N && s.u * kI4In + 32 * j < s.K;
            w[j] = in ? i4_order(c) : 0u;
        }
        if (g == 0) {
            const bool in = s.row < s.N && s.u * kI4In + gi * G < s.K;
            *reinterpret_cast<uint16_t *>(dst + i4_scale_at(lane, gi, GP)) = in ? (uint16_t)s16 : (uint16_t)0;
            if (ZEROS) dst[i4_zero_at(lane, gi, GP)] = in ? (uint8_t)z : 0;
        }
    }
    *reinterpret_cast<uint4 *>(dst + 16 * lane) = make_uint4(w[0], w[1], w[2], w[3]);
}

// The values as bf16 [N, K], each rounded once.
__global__ __launch_bounds__(256) void i4_dequantize_kernel(const uint8_t *__restrict__ units, int G, int has_zeros,
                                                            int fp16, I4Shape s, uint16_t *__restrict__ weight) {
    int64_t unit;
    if (!s.find(&unit)) return;
    const int lane = lane_id(), r = lane & 15, g = lane >> 4;
    const uint8_t *src = units + unit * i4_unit_bytes(G, has_zeros);
    const uint4 c = ld_g(src + 16 * lane);
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
    if (s.row >= s.N) return;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int k = s.u * kI4In + 32 * j + 8 * g;
        if (k >= s.K) break;
        const int gi = 32 * j / G;
        const float sc = i4_scale(*reinterpret_cast<const uint16_t *>(src + i4_scale_at(r, gi, kI4In / G)), fp16);
        const float z = has_zeros ? (float)src[i4_zero_at(r, gi, kI4In / G)] : 8.0f;
        const bf16x8_t q = i4_decode(w[j]);
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            o[i] = f2bf(((float)q[2 * i] - z) * sc) | f2bf(((float)q[2 * i + 1] - z) * sc) << 16;
        *reinterpret_cast<uint4 *>(weight + s.row * s.K + k) = make_uint4(o[0], o[1], o[2], o[3]);
    }
}

static int i4_check(const char *what, const void *a, const void *b, const void *c, int N, int K, int G) {
    if (!a || !b || !c) return fail(kEInval, std::string(what) + ": null pointer");
    if (!i4_shape_ok(N, K, G))
        return fail(kEInval, std::string(what) + ": need 1 <= N <= 2^24, G of 32, 64 or 128 and K % G == 0, K <= 2^20");
    for (const void *p : {a, b})
        if (reinterpret_cast<uintptr_t>(p) % 16)
            return fail(kEInval, std::string(what) + ": addresses need 16-byte alignment");
    // a wave per unit, in one grid dimension of fewer than 2^32 threads
    if (i4_units(N, K) > ((int64_t)1 << 26) - 4) return fail(kEInval, std::string(what) + ": too many weights for one call");
    return kOk;
}

static I4Shape i4_at(int N, int K) { return I4Shape{N, K, (K + kI4In - 1) / kI4In, i4_units(N, K), 0, 0}; }

}  // namespace pd

using namespace pd;

PD_API size_t pdscope_int4_bytes(int N, int K, int G, int zeros) {
    return i4_shape_ok(N, K, G) ? (size_t)i4_units(N, K) * i4_unit_bytes(G, zeros != 0) : 0;
}

PD_API int pdscope_int4_pack(const void *codes, const void *scales, const void *zeros, int N, int K, int G, void *out,
                             void *stream) {
    const int rc = i4_check("int4_pack", codes, out, scales, N, K, G);
    if (rc) return rc;
    const I4Shape s = i4_at(N, K);
    i4_pack_kernel<<<(unsigned)((s.units + 3) / 4), 256, 0, reinterpret_cast<hipStream_t>(stream)>>>(
        (const uint8_t *)codes, (const uint16_t *)scales, (const uint8_t *)zeros, G, s, (uint8_t *)out);
    return check_launch("i4_pack_kernel");
}

PD_API int pdscope_int4_quantize(const void *weight, int N, int K, int G, int zeros, void *out, void *stream) {
    const int rc = i4_check("int4_quantize", weight, out, out, N, K, G);
    if (rc) return rc;
    const I4Shape s = i4_at(N, K);
    auto launch = [&](auto kernel) {
        kernel<<<(unsigned)((s.units + 3) / 4), 256, 0, reinterpret_cast<hipStream_t>(stream)>>>(
            (const uint16_t *)weight, s, (uint8_t *)out);
    };
    if (G == 32) zeros ? launch(i4_quantize_kernel<32, true>) : launch(i4_quantize_kernel<32, false>);
    else if (G == 64) zeros ? launch(i4_quantize_kernel<64, true>) : launch(i4_quantize_kernel<64, false>);
    else zeros ? launch(i4_quantize_kernel<128, true>) : launch(i4_quantize_kernel<128, false>);
    return check_launch("i4_quantize_kernel");
}

PD_API int pdscope_int4_dequantize(const void *units, int N, int K, int G, int zeros, int fp16_scales, void *weight,
                                   void *stream) {
    const int rc = i4_check("int4_dequantize", units, weight, weight, N, K, G);
    if (rc) return rc;
    const I4Shape s = i4_at(N, K);
    i4_dequantize_kernel<<<(unsigned)((s.units + 3) / 4), 256, 0, reinterpret_cast<hipStream_t>(stream)>>>(
        (const uint8_t *)units, G, zeros != 0, fp16_scales != 0, s, (uint16_t *)weight);
    return check_launch("i4_dequantize_kernel");
}
