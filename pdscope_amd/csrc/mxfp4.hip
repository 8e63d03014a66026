// bf16 expert blocks to 4-bit ones and back, and 4-bit checkpoints into blocks.
// No counterpart in the reference, whose experts are bf16 only (ExpertKey's
// representation, expertbench/cache.py).
//
// One wave per 64 x 128 group of the layout in mxfp4.h, or per piece of one (the
// four of a group in one workgroup, which together read whole lines).  Lane l = r + 16 g works
// on the pieces that it owns in the block: of row 16 i + r, inputs 32 jj + 8 g
// .. + 7, 16 bytes of bf16 each, so a scale block's 32 values lie in four
// lanes and its largest magnitude takes two lane swaps.  Bound by HBM: 2 bytes a
// value on the bf16 side, 17/32 on the other (64 experts of the Qwen shape:
// quantised in 145 us, 5.3 TB/s, and back in 142; 165 by whole groups).
#include "mxfp4.h"

namespace pd {

// Where group g of an expert lies in the bf16 block (gate | up | down): the
// element offset of row 0 of its 16-row tile i, the row stride, and the first
// input.
struct GroupAt {
    size_t row[4];
    int ld, k0;
};

__device__ __forceinline__ GroupAt group_at(int g, int H, int I) {
    GroupAt a;
    const int n_gu = (I / 32) * (H / kGroupIn);
    if (g < n_gu) {
        const int rg = g / (H / kGroupIn);
        a.ld = H;
        a.k0 = (g - rg * (H / kGroupIn)) * kGroupIn;
#pragma unroll
        for (int i = 0; i < 4; ++i) a.row[i] = (size_t)((i >> 1) * I + rg * 32 + (i & 1) * 16) * H;
    } else {
        g -= n_gu;
        const int rg = g / (I / kGroupIn);
        a.ld = I;
        a.k0 = (g - rg * (I / kGroupIn)) * kGroupIn;
#pragma unroll
        for (int i = 0; i < 4; ++i) a.row[i] = (size_t)2 * I * H + (size_t)(rg * 64 + i * 16) * I;
    }
    return a;
}

// max of the values of lanes l, l ^ 16, l ^ 32 and l ^ 48, in each of them
__device__ __forceinline__ uint32_t max_over_quarters(uint32_t v) {
    const auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = max(a[0], a[1]);
    const auto b = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return max(b[0], b[1]);
}

// Eight bf16 values to a word of codes: times 2^(127 - byte) (exact), then the
// nearest code, ties to the even one, magnitudes above 6 to 6.
__device__ __forceinline__ uint32_t encode8(const uint4 v, float inv) {
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, lo_bf(v.x) * inv, hi_bf(v.x) * inv, 1.0f, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, lo_bf(v.y) * inv, hi_bf(v.y) * inv, 1.0f, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, lo_bf(v.z) * inv, hi_bf(v.z) * inv, 1.0f, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, lo_bf(v.w) * inv, hi_bf(v.w) * inv, 1.0f, 3);
}

// the largest magnitude of eight bf16 values, as its bits
__device__ __forceinline__ uint32_t top_magnitude(const uint4 v) {
    typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
    auto mag = [](uint32_t w) { return __builtin_bit_cast(u16x2_t, w & 0x7fff7fffu); };
    const u16x2_t m = __builtin_elementwise_max(__builtin_elementwise_max(mag(v.x), mag(v.y)),
                                                __builtin_elementwise_max(mag(v.z), mag(v.w)));
    return max((uint32_t)m[0], (uint32_t)m[1]);
}

// What a wave works on: NJ consecutive 32-input pieces of a group.
template <int NJ>
struct Pieces {
    int64_t expert;
    size_t group;  // in the call
    GroupAt at;
    int j0;
    __device__ __forceinline__ bool find(int64_t groups, int per_expert, int H, int I) {
        const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
        const int64_t q = w / (4 / NJ);
        if (q >= groups) return false;
        group = (size_t)q;
        expert = q / per_expert;
        at = group_at((int)(q - expert * per_expert), H, I);
        j0 = NJ == 4 ? 0 : (int)(w % (4 / NJ)) * NJ;
        return true;
    }
};

// The scale words of NJ pieces (row 16 i + r in byte i of each).
template <int NJ>
__device__ __forceinline__ void store_scales(uint8_t *group, int r, int j0, const uint32_t (&w)[NJ]) {
    uint8_t *p = group + kGroupScales + r * 16 + j0 * 4;
    if constexpr (NJ == 4) *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else *reinterpret_cast<uint32_t *>(p) = w[0];
}

template <int NJ>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const uint16_t *__restrict__ experts, int64_t groups, int H,
                                                          int I, int per_expert, uint8_t *__restrict__ blocks) {
    Pieces<NJ> p;
    if (!p.find(groups, per_expert, H, I)) return;
    const int lane = lane_id(), r = lane & 15, g = lane >> 4;
    const uint16_t *src =
        experts + p.expert * ((int64_t)3 * I * H) + (size_t)r * p.at.ld + p.at.k0 + 32 * p.j0 + 8 * g;
    uint4 v[NJ][4];  // [jj][i]
#pragma unroll
    for (int jj = 0; jj < NJ; ++jj)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[jj][i] = ld_g(src + p.at.row[i] + 32 * jj);
    uint8_t *dst = blocks + p.group * kGroupBytes;
    uint32_t scales[NJ];
#pragma unroll
    for (int jj = 0; jj < NJ; ++jj) {
        uint32_t word[4];
        scales[jj] = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint4 q = v[jj][i];
            const uint32_t top = max_over_quarters(top_magnitude(q));
            // floor(log2 of the largest) - 2 as an e8m0 byte: the bf16 exponent
            // field less 2, not below 2^-127; an infinity or NaN makes the
            // whole block NaN (byte 255)
            const uint32_t ex = top >> 7;
            const uint32_t byte = ex == 255u ? 255u : ex > 2u ? ex - 2u : 0u;
            word[i] = ex == 255u ? 0u : encode8(q, __uint_as_float((254u - byte) << 23));
            scales[jj] |= byte << (8 * i);
        }
        *reinterpret_cast<uint4 *>(dst + (p.j0 + jj) * 1024 + lane * 16) = make_uint4(word[0], word[1], word[2], word[3]);
    }
    if (g == 0) store_scales<NJ>(dst, r, p.j0, scales);
}

__global__ __launch_bounds__(256) void mx_dequantize_kernel(const uint8_t *__restrict__ blocks, int64_t groups, int H,
                                                            int I, int per_expert, uint16_t *__restrict__ experts) {
    Pieces<1> p;
    if (!p.find(groups, per_expert, H, I)) return;
    const int lane = lane_id(), r = lane & 15, g = lane >> 4;
    const uint8_t *src = blocks + p.group * kGroupBytes;
    const uint4 c = ld_g(src + p.j0 * 1024 + lane * 16);
    const uint32_t sw = *reinterpret_cast<const uint32_t *>(src + kGroupScales + r * 16 + p.j0 * 4);
    uint16_t *dst = experts + p.expert * ((int64_t)3 * I * H) + (size_t)r * p.at.ld + p.at.k0 + 32 * p.j0 + 8 * g;
    *reinterpret_cast<bf16x8_t *>(dst + p.at.row[0]) = mx_decode(c.x, mx_scale<0>(sw));
    *reinterpret_cast<bf16x8_t *>(dst + p.at.row[1]) = mx_decode(c.y, mx_scale<1>(sw));
    *reinterpret_cast<bf16x8_t *>(dst + p.at.row[2]) = mx_decode(c.z, mx_scale<2>(sw));
    *reinterpret_cast<bf16x8_t *>(dst + p.at.row[3]) = mx_decode(c.w, mx_scale<3>(sw));
}

// Row-major codes [.., K/2] and scales [.., K/32] of gate | up | down (a
// checkpoint's tensors) into blocks: moves bytes only.
__global__ __launch_bounds__(256) void mx_pack_kernel(const uint8_t *__restrict__ codes,
                                                      const uint8_t *__restrict__ scales, int64_t groups, int H, int I,
                                                      int per_expert, uint8_t *__restrict__ blocks) {
    const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (w >= groups) return;
    const int64_t e = w / per_expert;
    const GroupAt at = group_at((int)(w - e * per_expert), H, I);
    const int lane = lane_id(), r = lane & 15, g = lane >> 4;
    const int64_t n = (int64_t)3 * I * H;
    const uint8_t *cs = codes + e * (n / 2) + ((size_t)r * at.ld + at.k0 + 8 * g) / 2;
    const uint8_t *ss = scales + e * (n / 32) + ((size_t)r * at.ld + at.k0) / 32;
    uint8_t *dst = blocks + (size_t)w * kGroupBytes;
    uint32_t sc[4] = {0, 0, 0, 0};
#pragma unroll
    for (int jj = 0; jj < 4; ++jj) {
        uint32_t word[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            word[i] = *reinterpret_cast<const uint32_t *>(cs + at.row[i] / 2 + 16 * jj);
            sc[jj] |= (uint32_t)ss[at.row[i] / 32 + jj] << (8 * i);
        }
        *reinterpret_cast<uint4 *>(dst + jj * 1024 + lane * 16) = make_uint4(word[0], word[1], word[2], word[3]);
    }
    if (g == 0) *reinterpret_cast<uint4 *>(dst + kGroupScales + r * 16) = make_uint4(sc[0], sc[1], sc[2], sc[3]);
}

static int mx_check(const char *what, const void *a, const void *b, const void *c, int n, int H, int I) {
    if (!a || !b || !c) return fail(kEInval, std::string(what) + ": null pointer");
    if (n < 1 || n > 65536) return fail(kEInval, std::string(what) + ": need 1 to 65536 experts");
    if (!mx_shape_ok(H, I) || H > 65536 || I > 65536)
        return fail(kEInval, std::string(what) + ": need H % 128 == 0 and I % 128 == 0 (at most 65536)");
    for (const void *p : {a, b, c})
        if (reinterpret_cast<uintptr_t>(p) % 16) return fail(kEInval, std::string(what) + ": addresses need 16-byte alignment");
    // up to a workgroup of 256 per group, in one grid dimension of fewer than 2^32 threads
    if ((int64_t)n * (int64_t)(mx_block_bytes(H, I) / kGroupBytes) > ((int64_t)1 << 24) - 1)
        return fail(kEInval, std::string(what) + ": too many weights for one call");
    return kOk;
}

static int64_t mx_groups(int n, int H, int I) { return (int64_t)n * (int64_t)(mx_block_bytes(H, I) / kGroupBytes); }

}  // namespace pd

using namespace pd;

PD_API size_t pdscope_mxfp4_block_bytes(int H, int I) { return mx_shape_ok(H, I) ? mx_block_bytes(H, I) : 0; }

PD_API int pdscope_mxfp4_quantize(const void *experts, int n, int H, int I, void *blocks, void *stream) {
    const int rc = mx_check("mxfp4_quantize", experts, blocks, blocks, n, H, I);
    if (rc) return rc;
    const int64_t groups = mx_groups(n, H, I);
    auto launch = [&](auto kernel, int nj) {
        kernel<<<(unsigned)((groups * (4 / nj) + 3) / 4), 256, 0, reinterpret_cast<hipStream_t>(stream)>>>(
            (const uint16_t *)experts, groups, H, I, (int)(groups / n), (uint8_t *)blocks);
    };
    // a wave per piece where whole groups are too few to fill the card: experts of
    // the Qwen shape (576 groups each) 1: 4.9 us, by group 6.3; 4: 11.9 and 13.2;
    // 16: 38.5 and 39.1; 32: 75.8 and 74.1; 64: 150 and 145
    if (groups < 16384) launch(mx_quantize_kernel<1>, 1);
    else launch(mx_quantize_kernel<4>, 4);
    return check_launch("mx_quantize_kernel");
}

PD_API int pdscope_mxfp4_dequantize(const void *blocks, int n, int H, int I, void *experts, void *stream) {
    const int rc = mx_check("mxfp4_dequantize", blocks, experts, experts, n, H, I);
    if (rc) return rc;
    const int64_t groups = mx_groups(n, H, I);
    mx_dequantize_kernel<<<(unsigned)groups, 256, 0, reinterpret_cast<hipStream_t>(stream)>>>(
        (const uint8_t *)blocks, groups, H, I, (int)(groups / n), (uint16_t *)experts);
    return check_launch("mx_dequantize_kernel");
}

PD_API int pdscope_mxfp4_pack(const void *codes, const void *scales, int n, int H, int I, void *blocks, void *stream) {
    const int rc = mx_check("mxfp4_pack", codes, scales, blocks, n, H, I);
    if (rc) return rc;
    const int64_t groups = mx_groups(n, H, I);
    mx_pack_kernel<<<(unsigned)((groups + 3) / 4), 256, 0, reinterpret_cast<hipStream_t>(stream)>>>(
        (const uint8_t *)codes, (const uint8_t *)scales, groups, H, I, (int)(groups / n), (uint8_t *)blocks);
    return check_launch("mx_pack_kernel");
}
