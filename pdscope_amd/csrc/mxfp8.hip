// bf16 activations to 8-bit rows (mxfp8.h) and back, for callers whose rows do not
// come out of the norms' launch.  No counterpart in the reference, whose
// activations are bf16 only.
//
// A thread has eight channels, four neighbours a scale block.  Bound by memory: 2 bytes
// a value on one side, 33/32 on the other.  4096 rows of 2048: 6.1 to 6.7 us to rows and 5.2 to
// 5.9 back, 3.8 to 4.2 and 4.3 to 4.9 TB/s.
#include "mxfp8.h"

namespace pd {

__global__ __launch_bounds__(256) void mx8_quantize_kernel(const uint16_t *__restrict__ x, int64_t eights,
                                                           uint8_t *__restrict__ codes, uint8_t *__restrict__ scales) {
    const int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (q >= eights) return;  // whole quads: eights % 4 == 0
    const uint4 a = ld_g(x + 8 * q);
    const float v[8] = {lo_bf(a.x), hi_bf(a.x), lo_bf(a.y), hi_bf(a.y), lo_bf(a.z), hi_bf(a.z), lo_bf(a.w), hi_bf(a.w)};
    const uint32_t byte = mx8_scale_byte(max_over_quad(top_magnitude8(v)));
    *reinterpret_cast<uint2 *>(codes + 8 * q) = mx8_encode8(v, byte);
    if ((q & 3) == 0) scales[q / 4] = (uint8_t)byte;
}

__global__ __launch_bounds__(256) void mx8_dequantize_kernel(const uint8_t *__restrict__ codes,
                                                             const uint8_t *__restrict__ scales, int64_t eights,
                                                             uint16_t *__restrict__ x) {
    const int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (q >= eights) return;
    const uint2 c = *reinterpret_cast<const uint2 *>(codes + 8 * q);
    // the conversion reads the exponent field alone: 0 is 2^-127, 255 makes every value NaN
    const float s = __uint_as_float((uint32_t)scales[q / 4] << 23);
    const bf16x2_t v0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.x, s, false);
    const bf16x2_t v1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.x, s, true);
    const bf16x2_t v2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.y, s, false);
    const bf16x2_t v3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.y, s, true);
    *reinterpret_cast<bf16x8_t *>(x + 8 * q) = bf16x8_t{v0[0], v0[1], v1[0], v1[1], v2[0], v2[1], v3[0], v3[1]};
}

static int mx8_check(const char *what, const void *x, const void *codes, const void *scales, int64_t rows, int n) {
    if (!x || !codes || !scales) return fail(kEInval, std::string(what) + ": null pointer");
    if (rows < 1 || n < 32 || n % 32) return fail(kEInval, std::string(what) + ": need rows >= 1 and n % 32 == 0");
    // eight values a thread, fewer than 2^32 threads a launch
    if (rows > (((int64_t)1 << 35) - 4096) / n) return fail(kEInval, std::string(what) + ": too many values for one call");
    for (const void *p : {x, codes})
        if (reinterpret_cast<uintptr_t>(p) % 16) return fail(kEInval, std::string(what) + ": x and codes need 16-byte alignment");
    return kOk;
}

}  // namespace pd

using namespace pd;

PD_API int pdscope_mxfp8_quantize(const void *x, int64_t rows, int n, void *codes, void *scales, void *stream) {
    const int rc = mx8_check("mxfp8_quantize", x, codes, scales, rows, n);
    if (rc) return rc;
    const int64_t eights = rows * n / 8;
    mx8_quantize_kernel<<<(unsigned)((eights + 255) / 256), 256, 0, reinterpret_cast<hipStream_t>(stream)>>>(
        (const uint16_t *)x, eights, (uint8_t *)codes, (uint8_t *)scales);
    return check_launch("mx8_quantize_kernel");
}

PD_API int pdscope_mxfp8_dequantize(const void *codes, const void *scales, int64_t rows, int n, void *x, void *stream) {
    const int rc = mx8_check("mxfp8_dequantize", x, codes, scales, rows, n);
    if (rc) return rc;
    const int64_t eights = rows * n / 8;
    mx8_dequantize_kernel<<<(unsigned)((eights + 255) / 256), 256, 0, reinterpret_cast<hipStream_t>(stream)>>>(
        (const uint8_t *)codes, (const uint8_t *)scales, eights, (uint16_t *)x);
    return check_launch("mx8_dequantize_kernel");
}
