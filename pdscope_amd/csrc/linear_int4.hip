// y = x W^T + bias over a 4-bit matrix with group scales (int4.h): the attention's
// projections and the vocabulary head of a model whose experts run here, which
// the reference leaves to the model's torch modules
// (benchmarks/pdscope_compare.py:198-212).
//
//   y[t, n] = bf16(sum_groups s[n] * (sum_k q[n, k] x[t, k] - z[n] * sum_k x[t, k]) + bias[n])
//
// The whole numbers q are bf16 exactly, so the products with x are exact and a
// group's two sums are held in fp32; the scale enters once a group, in fp32.
#include "int4.h"

namespace pd {

struct I4Linear {
    const uint8_t *w;
    const uint16_t *x, *bias;
    uint16_t *y;
    int T, N, K, fp16;
};

// A workgroup: NT tiles of 16 rows of W x MT tiles of 16 tokens, the K axis split
// over WV waves.
template <int G, bool ZEROS, int NT, int MT, int WV>
__global__ __launch_bounds__(64 * WV) void i4_linear_kernel(I4Linear p) {
    constexpr int GP = kI4In / G, JG = 4 / GP, UB = i4_unit_bytes(G, ZEROS);
    __shared__ f32x4_t s_part[WV][NT * MT][64];
    const int lane = lane_id(), wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
    const int tiles = (p.N + kI4Rows - 1) / kI4Rows, KU = (p.K + kI4In - 1) / kI4In;
    const int across = (tiles + NT - 1) / NT;
    const int tb = blockIdx.x / across, n0 = (blockIdx.x - tb * across) * NT;
    const bf16x8_t ones = {(__bf16)1.0f, (__bf16)1.0f, (__bf16)1.0f, (__bf16)1.0f,
                           (__bf16)1.0f, (__bf16)1.0f, (__bf16)1.0f, (__bf16)1.0f};
    const uint8_t *wt[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) wt[n] = p.w + (size_t)min(n0 + n, tiles - 1) * KU * UB;
    const uint16_t *xr[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) xr[m] = p.x + (size_t)min((tb * MT + m) * 16 + r, p.T - 1) * p.K;

    f32x4_t tot[NT][MT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int m = 0; m < MT; ++m) tot[n][m] = f32x4_t{};
    for (int u = wave; u < KU; u += WV) {
        uint4 c[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) c[n] = ld_nt(wt[n] + (size_t)u * UB + 16 * lane);
        bf16x8_t x[MT][4];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int k = u * kI4In + 32 * j + 8 * g;
                uint4 v = make_uint4(0, 0, 0, 0);
                if (k < p.K) v = ld_g(xr[m] + k);
                x[m][j] = __builtin_bit_cast(bf16x8_t, v);
            }
#pragma unroll
        for (int gi = 0; gi < GP; ++gi) {
            f32x4_t sx[MT];
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                sx[m] = f32x4_t{};
#pragma unroll
                for (int j = gi * JG; j < (gi + 1) * JG; ++j)
                    sx[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, x[m][j], sx[m], 0, 0, 0);
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const uint32_t words[4] = {c[n].x, c[n].y, c[n].z, c[n].w};
                f32x4_t acc[MT];
#pragma unroll
                for (int m = 0; m < MT; ++m) acc[m] = f32x4_t{};
#pragma unroll
                for (int j = gi * JG; j < (gi + 1) * JG; ++j) {
                    const bf16x8_t w = i4_decode(words[j]);
#pragma unroll
                    for (int m = 0; m < MT; ++m)
                        acc[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, x[m][j], acc[m], 0, 0, 0);
                }
                const uint8_t *side = wt[n] + (size_t)u * UB + kI4Codes;
                const uint2 s4 = *reinterpret_cast<const uint2 *>(side + gi * 32 + 8 * g);
                const uint32_t z4 = ZEROS ? *reinterpret_cast<const uint32_t *>(side + GP * 32 + gi * 16 + 4 * g) : 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float s = i4_scale((i < 2 ? s4.x : s4.y) >> (16 * (i & 1)) & 0xffffu, p.fp16);
                    const float z = ZEROS ? (float)(z4 >> (8 * i) & 255u) : 8.0f;
#pragma unroll
                    for (int m = 0; m < MT; ++m) tot[n][m][i] = fmaf(s, fmaf(-z, sx[m][i], acc[m][i]), tot[n][m][i]);
                }
            }
        }
    }
    // ---- the waves' parts, in order; lane l has token r and rows 4 g .. + 3 of a tile
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int m = 0; m < MT; ++m) s_part[wave][n * MT + m][lane] = tot[n][m];
    __syncthreads();
    for (int q = threadIdx.x; q < NT * MT * 64; q += 64 * WV) {
        const int tile = q >> 6, l = q & 63, n = tile / MT, m = tile - n * MT;
        f32x4_t v = s_part[0][tile][l];
#pragma unroll
        for (int w = 1; w < WV; ++w) v += s_part[w][tile][l];
        const int t = (tb * MT + m) * 16 + (l & 15), row = (n0 + n) * 16 + 4 * (l >> 4);
        if (t >= p.T) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (row + i < p.N)
                p.y[(size_t)t * p.N + row + i] = (uint16_t)f2bf(v[i] + (p.bias ? bf2f(p.bias[row + i]) : 0.0f));
    }
}

template <int G, bool ZEROS>
static void i4_linear_launch(const I4Linear &a, hipStream_t s) {
    constexpr int NT = 1, MT = 1, WV = 8;
    const int64_t across = ((a.N + 15) / 16 + NT - 1) / NT, down = (a.T + 16 * MT - 1) / (16 * MT);
    i4_linear_kernel<G, ZEROS, NT, MT, WV><<<(unsigned)(across * down), 64 * WV, 0, s>>>(a);
}

}  // namespace pd

using namespace pd;

PD_API int pdscope_linear_int4(const void *x, const void *w, const void *bias, int T, int N, int K, int G, int zeros,
                               int fp16_scales, void *y, void *stream) {
    if (!x || !w || !y) return fail(kEInval, "linear_int4: null pointer");
    if (!i4_shape_ok(N, K, G) || i4_units(N, K) > ((int64_t)1 << 26) - 4)
        return fail(kEInval, "linear_int4: need 1 <= N <= 2^24, G of 32, 64 or 128 and K % G == 0, K <= 2^20");
    if (T < 1) return fail(kEInval, "linear_int4: need T >= 1");
    for (const void *p : {x, w})
        if (reinterpret_cast<uintptr_t>(p) % 16) return fail(kEInval, "linear_int4: x and w need 16-byte alignment");
    // a launch has fewer than 2^32 threads: at most 512 for 16 rows of W and 16 of x
    if ((((int64_t)N + 15) / 16) * (((int64_t)T + 15) / 16) > ((int64_t)1 << 23) - 1)
        return fail(kEInval, "linear_int4: too many outputs for one launch");
    const I4Linear a{(const uint8_t *)w, (const uint16_t *)x, (const uint16_t *)bias, (uint16_t *)y, T, N, K, fp16_scales != 0};
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (G == 32) zeros ? i4_linear_launch<32, true>(a, s) : i4_linear_launch<32, false>(a, s);
    else if (G == 64) zeros ? i4_linear_launch<64, true>(a, s) : i4_linear_launch<64, false>(a, s);
    else zeros ? i4_linear_launch<128, true>(a, s) : i4_linear_launch<128, false>(a, s);
    return check_launch("i4_linear_kernel");
}
