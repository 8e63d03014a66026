// What stands between two blocks, in one launch: the norm after a block, its
// gate and residual scale, the residual sum and the norm before the next block,
// over the block's output or over the experts' rows that the weighted merge
// would sum first.  The reference leaves all of it to the model's eager torch
// modules around its layer hook (benchmarks/pdscope_compare.py:285-304).
//
//   a[c] = block[t,c],  or  add_in[t,c] + sum_s w[t,s] y[row_of[t k + s], c]
//   a    = a * rsqrt(mean(a^2) + eps) * post_w       (post_w given)
//   r[c] = resid[t,c] + scale * gate * a[c]          -> out_resid
//   n[c] = r[c] * rsqrt(mean(r^2) + eps) * pre_w[c]  -> out_norm
// Everything between loads and stores is fp32; each result is rounded once.
//
// One workgroup per row, its values in registers from the first load to the last
// store, so every byte moves once: bound by HBM for many rows, by the latency
// of a load, two reductions and a store for one.
//
// With 8-bit rows (MX) n also goes out as e4m3 codes with a scale per 32
// channels (mxfp8.h), for the experts' products; out_norm is then optional.  A
// thread's eight channels and its three neighbours' make a scale block.  Everything is
// held in 64 bits then, and the codes are rounded from that: they do not depend
// on the order of the sums, where 32 bits move one code in some hundred
// thousand to its neighbour.  The vector units run 64-bit products at the 32-bit rate.
// 4096 rows of 2048 with the merge of eight rows each: 41.6 us, 4.6 TB/s; 777 rows of 1504 with post
// norm, gate and fp32 parameters 8.0 us, 3.1 by their bytes (all rows run at once, each a chain of block
// and residual, a sum, post weight and gate, a sum, pre weight and the store); one 3.4 to 3.7.
#include <type_traits>

#include "mxfp8.h"

namespace pd {

struct NormArgs {
    const uint16_t *block;  // [T, H], or (k > 0) the experts' rows [y_rows, H], which may be fp32
    const int32_t *row_of;
    const uint16_t *w, *add_in;
    int64_t y_rows;
    int k, y_f32;
    const void *resid;
    const void *post_w, *gate, *pre_w;
    int gate_rows, gate_cols;  // gate has a value per token / per channel
    float scale, eps;
    int H;
    void *out_resid;
    uint16_t *out_norm;
    uint8_t *out_codes, *out_scales;  // 8-bit rows [T, H] and [T, H / 32], or null
};

// Eight values of a row.  VEC: consecutive ones from 8 c on (16-byte aligned);
// else values c, c + n, c + 2n, ... (8-bit rows: consecutive ones, one at a time)
template <bool VEC>
struct Eight {
    int at, step;
    __device__ __forceinline__ int idx(int i) const { return VEC ? at + i : at + i * step; }
};

// NT: rows that nothing reads again are not kept in the caches (k = 8, H = 2048;
// rows from memory, T = 4096: 44.3 us, 4.9 TB/s, against 50.5 with plain loads; right behind
// the kernel that wrote them, T = 256 8.5 against 9.8, T = 4096 40 against 38, T =
// 8192 72 against 75).
template <bool VEC, bool F32, bool NT = false>
__device__ __forceinline__ void load8(const void *base, const Eight<VEC> &e, int H, float (&v)[8]) {
    if (VEC) {
        if (F32) {
            const float *p = (const float *)base + e.at;
            const uint4 a = NT ? ld_nt(p) : ld_g(p), b = NT ? ld_nt(p + 4) : ld_g(p + 4);
            const uint32_t u[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(u[i]);
        } else {
            const uint4 a = NT ? ld_nt((const uint16_t *)base + e.at) : ld_g((const uint16_t *)base + e.at);
            const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] = lo_bf(u[i]);
                v[2 * i + 1] = hi_bf(u[i]);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int c = min(e.idx(i), H - 1);
            v[i] = F32 ? ((const float *)base)[c] : bf2f(((const uint16_t *)base)[c]);
        }
    }
}

template <bool VEC, bool F32>
__device__ __forceinline__ void store8(void *base, const Eight<VEC> &e, int H, const float (&v)[8]) {
    if (VEC) {
        if (F32) {
            float4 *p = reinterpret_cast<float4 *>((float *)base + e.at);
            p[0] = make_float4(v[0], v[1], v[2], v[3]);
            p[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            *reinterpret_cast<uint4 *>((uint16_t *)base + e.at) =
                make_uint4(f2bf(v[0]) | f2bf(v[1]) << 16, f2bf(v[2]) | f2bf(v[3]) << 16,
                           f2bf(v[4]) | f2bf(v[5]) << 16, f2bf(v[6]) | f2bf(v[7]) << 16);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int c = e.idx(i);
            if (c < H) {
                if (F32) ((float *)base)[c] = v[i];
                else ((uint16_t *)base)[c] = (uint16_t)f2bf(v[i]);
            }
        }
    }
}

__device__ __forceinline__ float row_sum(float v) { return wave_sum_dpp(v); }
__device__ __forceinline__ double row_sum(double v) { return wave_sum(v); }

// Sum over the workgroup, the same in every thread: waves in order.
template <typename F>
__device__ __forceinline__ F block_sum(F v, F *s_sum) {
    v = row_sum(v);
    const int nw = blockDim.x >> 6;
    if (nw == 1) return v;
    __syncthreads();  // s_sum may still be read from the sum before
    if (lane_id() == 0) s_sum[threadIdx.x >> 6] = v;
    __syncthreads();
    F t = 0;
    for (int w = 0; w < nw; ++w) t += s_sum[w];
    return t;
}

// 1 / sqrt(mean + eps), correctly rounded root and quotient
__device__ __forceinline__ float inv_rms(float sum, int H, float eps) { return 1.0f / sqrtf(sum / (float)H + eps); }
__device__ __forceinline__ double inv_rms(double sum, int H, float eps) { return 1.0 / sqrt(sum / (double)H + (double)eps); }

// What is stored of eight values: themselves, or the 32-bit values that keep for any
// shorter type on which side of its borders 64-bit ones lie.
__device__ __forceinline__ void narrow8(const float (&v)[8], float (&o)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = v[i];
}
__device__ __forceinline__ void narrow8(const double (&v)[8], float (&o)[8]) { round_to_odd8(v, o); }

// NV: eights of a row per thread; MX: 8-bit rows as well; Y32: the experts' rows in fp32.
template <bool VEC, bool R32, bool P32, int NV, bool MX, bool Y32>
__global__ __launch_bounds__(1024) void norm_kernel(NormArgs a) {
    using F = std::conditional_t<MX, double, float>;
    __shared__ F s_sum[16];
    const int t = blockIdx.x, H = a.H, n = blockDim.x;
    Eight<VEC> at[NV];
    bool on[NV];  // has values of the row (every thread keeps its place in the sums)
    F v[NV][8];
    float res[NV][8];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int q = threadIdx.x + j * n;
        at[j] = VEC || MX ? Eight<VEC>{8 * q, 1} : Eight<VEC>{(int)threadIdx.x + j * 8 * n, n};
        on[j] = at[j].at < H;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[j][i] = res[j][i] = 0.0f;
        if (!on[j]) continue;
        load8<VEC, R32>((const char *)a.resid + (size_t)t * H * (R32 ? 4 : 2), at[j], H, res[j]);
        if (a.k == 0 || a.add_in) {
            float b[8];
            load8<VEC, false>((a.k == 0 ? a.block : a.add_in) + (size_t)t * H, at[j], H, b);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[j][i] = b[i];
        }
    }
    if (a.k) {
        // slot order; a row outside y (an expert computed elsewhere) adds nothing
        const int32_t *rows = a.row_of + (size_t)t * a.k;
        const uint16_t *ws = a.w + (size_t)t * a.k;
#pragma unroll (Y32 ? 4 : 8)
        for (int s = 0; s < a.k; ++s) {
            const int32_t row = rows[s];
            const F w = bf2f(ws[s]);
            if (row < 0 || row >= a.y_rows) continue;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                if (!on[j]) continue;
                float y[8];
                load8<VEC, Y32, true>((const char *)a.block + (size_t)row * H * (Y32 ? 4 : 2), at[j], H, y);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[j][i] = fma(w, (F)y[i], v[j][i]);
            }
        }
    }
    F f = a.scale;
    if (a.gate && !a.gate_cols)
        f *= P32 ? ((const float *)a.gate)[a.gate_rows ? t : 0] : bf2f(((const uint16_t *)a.gate)[a.gate_rows ? t : 0]);
    if (a.post_w) {
        F q = 0;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (on[j] && at[j].idx(i) < H) q = fma(v[j][i], v[j][i], q);
        f *= inv_rms(block_sum(q, s_sum), H, a.eps);
    }
    F q = 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        if (!on[j]) continue;
        float m[8];
        if (a.post_w) {
            load8<VEC, P32>(a.post_w, at[j], H, m);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[j][i] *= m[i];
        }
        if (a.gate && a.gate_cols) {
            load8<VEC, P32>((const char *)a.gate + (a.gate_rows ? (size_t)t * H * (P32 ? 4 : 2) : 0), at[j], H, m);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[j][i] *= m[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[j][i] = fma(f, v[j][i], (F)res[j][i]);
            if (at[j].idx(i) < H) q = fma(v[j][i], v[j][i], q);
        }
        if (a.out_resid) {
            float r[8];
            if constexpr (R32) {
#pragma unroll
                for (int i = 0; i < 8; ++i) r[i] = (float)v[j][i];
            } else {
                narrow8(v[j], r);
            }
            store8<VEC, R32>((char *)a.out_resid + (size_t)t * H * (R32 ? 4 : 2), at[j], H, r);
        }
    }
    if (!MX && !a.out_norm) return;
    const F rs = inv_rms(block_sum(q, s_sum), H, a.eps);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        if (!on[j]) continue;
        float m[8];
        if (a.pre_w) {
            load8<VEC, P32>(a.pre_w, at[j], H, m);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[j][i] *= rs * m[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[j][i] *= rs;
        }
        float o[8];
        narrow8(v[j], o);
        if (!MX || a.out_norm) store8<VEC, false>(a.out_norm + (size_t)t * H, at[j], H, o);
        if constexpr (MX) {
            const uint32_t byte = mx8_scale_byte(max_over_quad(top_magnitude8(o)));
            const uint2 c = mx8_encode8(o, byte);
            uint8_t *codes = a.out_codes + (size_t)t * H + at[j].at;
            if (VEC) {
                *reinterpret_cast<uint2 *>(codes) = c;
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) codes[i] = (uint8_t)((i < 4 ? c.x : c.y) >> (8 * (i & 3)));
            }
            if ((threadIdx.x & 3) == 0) a.out_scales[((size_t)t * H + at[j].at) / 32] = (uint8_t)byte;
        }
    }
}

constexpr int kNormMaxH = 16384;

template <bool VEC, bool R32, bool P32, bool MX, bool Y32>
static void norm_launch(const NormArgs &a, int T, hipStream_t s) {
    const int n = (a.H + 511) / 512 * 64;  // eight values a thread
    if (n <= 1024) norm_kernel<VEC, R32, P32, 1, MX, Y32><<<T, n, 0, s>>>(a);
    else norm_kernel<VEC, R32, P32, 2, MX, Y32><<<T, (n / 2 + 63) / 64 * 64, 0, s>>>(a);
}

template <bool VEC, bool R32, bool P32>
static void norm_launch(const NormArgs &a, int T, hipStream_t s) {
    if (a.out_codes) a.y_f32 ? norm_launch<VEC, R32, P32, true, true>(a, T, s) : norm_launch<VEC, R32, P32, true, false>(a, T, s);
    else a.y_f32 ? norm_launch<VEC, R32, P32, false, true>(a, T, s) : norm_launch<VEC, R32, P32, false, false>(a, T, s);
}

static int norm_call(const char *what, const NormArgs &a, int resid_f32, int params_f32, int T, void *stream) {
    // a row of up to 1024 threads: fewer than 2^32 in a launch
    if (T < 1 || T >= (1 << 22) || a.H < 1 || a.H > kNormMaxH)
        return fail(kEInval, std::string(what) + ": need T >= 1 and below 2^22, and 1 <= H <= 16384");
    if (!a.block || !a.resid || (!a.out_resid && !a.out_norm && !a.out_codes))
        return fail(kEInval, std::string(what) + ": null pointer");
    if (a.out_codes && a.H % 32) return fail(kEInval, std::string(what) + ": 8-bit rows need H % 32 == 0");
    if (!(a.eps >= 0.0f)) return fail(kEInval, std::string(what) + ": eps must not be negative");
    bool vec = a.H % 8 == 0;
    for (const void *p : {(const void *)a.block, (const void *)a.add_in, a.resid, a.post_w, a.gate_cols ? a.gate : nullptr,
                          a.pre_w, (const void *)a.out_resid, (const void *)a.out_norm, (const void *)a.out_codes})
        vec = vec && reinterpret_cast<uintptr_t>(p) % 16 == 0;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const int variant = (vec ? 4 : 0) | (resid_f32 ? 2 : 0) | (params_f32 ? 1 : 0);
    switch (variant) {
    case 0: norm_launch<false, false, false>(a, T, s); break;
    case 1: norm_launch<false, false, true>(a, T, s); break;
    case 2: norm_launch<false, true, false>(a, T, s); break;
    case 3: norm_launch<false, true, true>(a, T, s); break;
    case 4: norm_launch<true, false, false>(a, T, s); break;
    case 5: norm_launch<true, false, true>(a, T, s); break;
    case 6: norm_launch<true, true, false>(a, T, s); break;
    default: norm_launch<true, true, true>(a, T, s); break;
    }
    return check_launch("norm_kernel");
}

}  // namespace pd

using namespace pd;

PD_API int pdscope_norm_residual(const void *block, const void *resid, int resid_f32, const void *post_w,
                                 const void *gate, int gate_rows, int gate_cols, float scale, const void *pre_w,
                                 int params_f32, float eps, int T, int H, void *out_resid, void *out_norm,
                                 void *stream) {
    const NormArgs a{(const uint16_t *)block, nullptr, nullptr, nullptr, 0, 0, 0, resid, post_w, gate, pre_w,
                     gate_rows, gate_cols, scale, eps, H, out_resid, (uint16_t *)out_norm, nullptr, nullptr};
    return norm_call("norm_residual", a, resid_f32, params_f32, T, stream);
}

PD_API int pdscope_merge_norm_residual(const void *y, int64_t y_rows, const int32_t *row_of, const void *w, int k,
                                       const void *add_in, const void *resid, int resid_f32, const void *post_w,
                                       const void *gate, int gate_rows, int gate_cols, float scale, const void *pre_w,
                                       int params_f32, float eps, int T, int H, void *out_resid, void *out_norm,
                                       void *stream) {
    if (!row_of || !w) return fail(kEInval, "merge_norm_residual: null pointer");
    if (k < 1 || y_rows < 1) return fail(kEInval, "merge_norm_residual: need k >= 1 and y_rows >= 1");
    const NormArgs a{(const uint16_t *)y, row_of, (const uint16_t *)w, (const uint16_t *)add_in, y_rows, k, 0, resid, post_w,
                     gate, pre_w, gate_rows, gate_cols, scale, eps, H, out_resid, (uint16_t *)out_norm, nullptr, nullptr};
    return norm_call("merge_norm_residual", a, resid_f32, params_f32, T, stream);
}

PD_API int pdscope_norm_residual_mxfp8(const void *block, const void *resid, int resid_f32, const void *post_w,
                                       const void *gate, int gate_rows, int gate_cols, float scale, const void *pre_w,
                                       int params_f32, float eps, int T, int H, void *out_resid, void *out_norm,
                                       void *out_codes, void *out_scales, void *stream) {
    if (!out_codes || !out_scales) return fail(kEInval, "norm_residual_mxfp8: null pointer");
    const NormArgs a{(const uint16_t *)block, nullptr, nullptr, nullptr, 0, 0, 0, resid, post_w, gate, pre_w,
                     gate_rows, gate_cols, scale, eps, H, out_resid, (uint16_t *)out_norm, (uint8_t *)out_codes,
                     (uint8_t *)out_scales};
    return norm_call("norm_residual_mxfp8", a, resid_f32, params_f32, T, stream);
}

PD_API int pdscope_merge_norm_residual_mxfp8(const void *y, int64_t y_rows, const int32_t *row_of, const void *w, int k,
                                             const void *add_in, const void *resid, int resid_f32, const void *post_w,
                                             const void *gate, int gate_rows, int gate_cols, float scale,
                                             const void *pre_w, int params_f32, float eps, int T, int H,
                                             void *out_resid, void *out_norm, void *out_codes, void *out_scales,
                                             void *stream) {
    if (!row_of || !w || !out_codes || !out_scales) return fail(kEInval, "merge_norm_residual_mxfp8: null pointer");
    if (k < 1 || y_rows < 1) return fail(kEInval, "merge_norm_residual_mxfp8: need k >= 1 and y_rows >= 1");
    const NormArgs a{(const uint16_t *)y, row_of, (const uint16_t *)w, (const uint16_t *)add_in, y_rows, k, 0, resid, post_w,
                     gate, pre_w, gate_rows, gate_cols, scale, eps, H, out_resid, (uint16_t *)out_norm,
                     (uint8_t *)out_codes, (uint8_t *)out_scales};
    return norm_call("merge_norm_residual_mxfp8", a, resid_f32, params_f32, T, stream);
}

PD_API int pdscope_merge_norm_residual_y32(const void *y, int64_t y_rows, const int32_t *row_of, const void *w, int k,
                                           const void *add_in, const void *resid, int resid_f32, const void *post_w,
                                           const void *gate, int gate_rows, int gate_cols, float scale,
                                           const void *pre_w, int params_f32, float eps, int T, int H, void *out_resid,
                                           void *out_norm, void *out_codes, void *out_scales, void *stream) {
    if (!row_of || !w || !out_codes != !out_scales) return fail(kEInval, "merge_norm_residual_y32: null pointer");
    if (k < 1 || y_rows < 1) return fail(kEInval, "merge_norm_residual_y32: need k >= 1 and y_rows >= 1");
    const NormArgs a{(const uint16_t *)y, row_of, (const uint16_t *)w, (const uint16_t *)add_in, y_rows, k, 1, resid, post_w,
                     gate, pre_w, gate_rows, gate_cols, scale, eps, H, out_resid, (uint16_t *)out_norm,
                     (uint8_t *)out_codes, (uint8_t *)out_scales};
    return norm_call("merge_norm_residual_y32", a, resid_f32, params_f32, T, stream);
}
