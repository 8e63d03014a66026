// The grouped SwiGLU expert FFN over 8-bit rows (mxfp8.h) and 4-bit expert blocks
// (mxfp4.h): products grouped by expert, every expert with as many rows as were
// routed to it.
//
//   gate/up : h[r,:] = rows8(silu(x_r . gate) * (x_r . up))
//   down    : y[r,n] = h_r . down_n, in fp32 or rounded to bf16
//
// Both operands go to the scaled matrix instruction as they are, codes and
// scales: v_mfma_scale_f32_16x16x128_f8f6f4, whose products are exact and whose
// sums are fp32.  Of its first operand (e2m1) lane l = r + 16 g holds row r and the
// 32 inputs of scale block g; of the second (e4m3) row r and the inputs 16 g
// .. + 15 and 64 + 16 g .. + 15, beside the scale of block g.
//
// The instruction adds groups of eight products, each cut to 2^-13 of the largest
// one's binade, and the groups in fp32: about 4e-6 of an output's size, far below the codes'.
// Rounded to fewer bits is h (8-bit rows, from the unrounded product: what its down
// product takes), and where the caller's y is bf16 each expert's row (as the other grouped kernels
// leave it to the merge, which sums in fp32 and rounds once more: together 2.4e-3 of an output
// against 1.7e-3 for the last rounding alone, more where rows cancel).  Rows in fp32 leave that one only.
//
// Wave tile: 64 rows of weights x BM rows of x.  Weights go from memory to registers,
// where a wave is the only one that needs them, a step of 128 inputs ahead; x through two
// LDS stages, which all waves read.  Few rows (BM = 32) are bound by the weights' bytes: 33
// tokens of the Qwen shape (H 2048, I 768, 128 experts, 8 a token), gate/up 32 us and down 18,
// 5.9 and 5.2 TB/s.  Many are bound by the time that a step's loads take under load, and by
// what a tile does before and after its K loop: 4096 tokens of the DeepSeek-V2-Lite shape (H 2048, I
// 1408, 64 experts, 6 a token) gate/up 156 us and down 89, 1.8 and 1.6 PFLOP/s, the matrix
// units busy 45% of the time; of a gate/up tile's 26 us 3.6 are spent before its loop (where it
// finds its expert and its rows) and 3.0 behind it, three tiles a CU at a time.  Without
// the loop's loads the layer's products take 95 us for 153, with weights from the L2 128.  Tried and
// not kept, all within 5% or slower: 128 rows a tile, two waves on the same weights through
// LDS with two to four stages (154 to 190 and 84 to 101 us), each wave's own weights two steps ahead
// through LDS (155 and 87) or in registers, eight waves a tile, four workgroups a CU (194 and 118 us,
// spilled), a list of experts read beside their tiles before the loop.
#include <algorithm>
#include <type_traits>

#include "mxfp4.h"
#include "mxfp8.h"
#include "ring.h"

typedef int i32x8_t __attribute__((ext_vector_type(8)));

namespace pd {

struct Mx8Grouped {
    const uint8_t *a, *a_scales;  // gate/up: x [T, H]; down: h [rows, I]
    const int32_t *perm_token, *offsets, *sel;
    int nsel;
    const int32_t *tile_start;
    const uint8_t *const *slots;
    int H, I;
    uint8_t *out, *out_scales;  // gate/up: h codes and scales; down: y [rows, H] bf16 or fp32, null
};

// Waves of a workgroup, a row group each.  Eight in the down half of BM = 32, two workgroups a CU: Qwen
// shape T = 33 18.5 us against 19.4, T = 8 14.5 against 12.2; DeepSeek-V2-Lite shape T = 33 22.0 against
// 18.6, T = 128 22.9 against 19.4; of BM = 64 at T = 1303 of the Qwen shape 78 and 49 us against 65 and 39.
constexpr int kMx8Waves = 4;
// bytes of a staged output row: 32 columns of h codes or 64 of bf16 y per wave, off the bank line
template <bool GATEUP>
constexpr int kMx8OutRow = kMx8Waves * (GATEUP ? 32 : 128) + 16;
template <int BM>
constexpr int kMx8Stage = BM * 128 + 256;  // codes and scales of a step's 128 inputs
template <int BM, bool GATEUP, bool Y32>
constexpr int kMx8Lds = std::max(2 * kMx8Stage<BM>, Y32 ? 0 : BM * kMx8OutRow<GATEUP> + (GATEUP ? BM * kMx8Waves : 0));

// BM rows x four groups (128 h columns or 256 y columns), K in steps of 128, two
// stages of activations; at least OCC workgroups per CU.  Y32: rows of y in fp32 (down).
template <int BM, bool GATEUP, int OCC, bool Y32>
__global__ __launch_bounds__(64 * kMx8Waves, OCC) void mx8_grouped_kernel(Mx8Grouped p) {
    __shared__ __attribute__((aligned(1024))) uint8_t smem[kMx8Lds<BM, GATEUP, Y32>];
    constexpr int TM = BM / 16, NW = kMx8Waves;
    const int H = p.H, I = p.I;
    const int K = GATEUP ? H : I, KT = K / kGroupIn;
    const int groups = GATEUP ? I / 32 : H / kGroupRows, NT = (groups + NW - 1) / NW;

    // ---- tile: eight contiguous pieces of the list, one per XCD, columns fastest
    const int total = p.tile_start[p.nsel] * NT;
    const int per_xcd = (total + 7) >> 3, pos = blockIdx.x >> 3;
    if (pos >= per_xcd) return;
    const int t = (blockIdx.x & 7) * per_xcd + pos;
    if (t >= total) return;
    const int mt = t / NT, nt = t - mt * NT;
    // the expert: the last lo with tile_start[lo] <= mt
    int lo = 0;
#pragma unroll 4
    for (int b0 = 1; b0 < p.nsel; b0 += 64) {
        const int j = b0 + (threadIdx.x & 63);
        lo += __popcll(__ballot(j < p.nsel && p.tile_start[j] <= mt));
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    const int e = p.sel[lo];
    const int row_end = p.offsets[e + 1], m0 = p.offsets[e] + (mt - p.tile_start[lo]) * BM;
    const uint8_t *base = p.slots[e];
    if (base == nullptr) return;  // no copy: the rows keep what they hold

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, g = lane >> 4;
    const int rg = nt * NW + wave;            // this wave's row group
    const int rg_in = min(rg, groups - 1);    // past the end: read the last one, store nothing
    const uint8_t *const wbase =
        base + ((GATEUP ? 0 : mx_gateup_groups(H, I)) + (size_t)rg_in * KT) * kGroupBytes;

    // ---- activation loads: load q of wave w fills rows 8 (NW q + w) .. + 7 of 128
    // bytes, whose 16-byte chunk c lies in slot c ^ (row / 2 % 8); lane l takes row + l /
    // 8 and the chunk that belongs in its slot
    constexpr int RQ = 8 * NW, AL = BM / RQ;  // rows per load of all waves, loads of a wave
    static_assert(BM % RQ == 0, "activation loads");
    const uint8_t *arow[AL];
    const int lrow = 8 * wave + (lane >> 3);  // in its load's rows
    const uint32_t achunk = (uint32_t)((lane & 7) ^ ((lrow >> 1) & 7));
#pragma unroll
    for (int q = 0; q < AL; ++q) {
        const int row = min(m0 + RQ * q + lrow, row_end - 1);
        arow[q] = p.a + (size_t)(GATEUP ? p.perm_token[row] : row) * K + achunk * 16;
    }
    // scales: lane l of the first wave takes row l's four of a step
    const uint8_t *srow = nullptr;
    if (wave * 64 < BM) {
        const int row = min(m0 + min(64 * wave + lane, BM - 1), row_end - 1);
        srow = p.a_scales + (size_t)(GATEUP ? p.perm_token[row] : row) * (K / 32);
    }
    // where the lane's pieces lie: of a row tile's codes and scales in a group of
    // weights, and of 16 rows in a stage
    const uint32_t wlane = (uint32_t)(g * 1024 + r * 16), slane = (uint32_t)(kGroupScales + (r * 4 + g) * 4);
    const uint32_t lx0 = (uint32_t)(r * 128 + ((g ^ (r >> 1)) << 4)), lx1 = lx0 ^ 64, lxs = (uint32_t)(r * 4 + g);
    const uint32_t lds0 = lds_offset(smem);

    f32x4_t acc[4][TM];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int m = 0; m < TM; ++m) acc[i][m] = f32x4_t{};

    auto kloop = [&](auto live, auto once) __attribute__((always_inline)) {
        constexpr int L = decltype(live)::value;  // token tiles with rows of the expert
        auto ld = [](const uint8_t *q) -> u32x4_t {
            return decltype(once)::value ? __builtin_nontemporal_load(gptr(q)) : *gptr(q);
        };
        auto issue_a = [&](int kt, uint32_t st) __attribute__((always_inline)) {
#pragma unroll
            for (int q = 0; q < AL; ++q) {
                if (RQ * q + 8 * wave >= 16 * L) continue;  // rows that no product reads
                load_lds_hidden<16>(arow[q] + kt * 128, lds0 + st + (RQ * q + 8 * wave) * 128);
            }
            if (wave == 0) load_lds_hidden<4>(srow + kt * 4, lds0 + st + BM * 128);
        };
        // word i of d[q]: row 16 i + r, inputs 32 g + 8 q .. + 7; word i of the four is
        // what the product of row tile i takes.  s: byte i is the scale of that block
        auto issue_w = [&](int kt, u32x4_t (&d)[4], uint32_t &s) __attribute__((always_inline)) {
            const uint8_t *b = wbase + (size_t)kt * kGroupBytes;
#pragma unroll
            for (int q = 0; q < 4; ++q) d[q] = ld(b + q * 256 + wlane);
            s = *(const __attribute__((address_space(1))) uint32_t *)(uintptr_t)(b + slane);
        };
        // One set of registers for the words that are on their way: a step first puts
        // each row tile's four words side by side, then asks for the next step's.
        u32x4_t d[4];
        uint32_t ds;
        auto step = [&](auto more, int kt) __attribute__((always_inline)) {
            const uint32_t st = (kt & 1) * kMx8Stage<BM>;
            wait_vm<0>();
            ring_barrier();
            u32x4_t w[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) asm volatile("" : "+v"(d[q]));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                w[i] = u32x4_t{d[0][i], d[1][i], d[2][i], d[3][i]};
                asm volatile("" : "+v"(w[i]));
            }
            int s = (int)ds;
            asm volatile("" : "+v"(s));
            if constexpr (decltype(more)::value) {
                issue_a(kt + 1, kMx8Stage<BM> - st);
                issue_w(kt + 1, d, ds);
            }
            __builtin_amdgcn_sched_barrier(0);
            // one address each, the token tiles behind it as offsets of the instruction
            uint32_t at0 = lx0 + st, at1 = lx1 + st, ats = lxs + st;
            opaque(at0);
            opaque(at1);
            opaque(ats);
            auto wide = [](u32x4_t v) { return i32x8_t{(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0}; };
#pragma unroll
            for (int m = 0; m < L; ++m) {
                const uint4 x0 = *reinterpret_cast<const uint4 *>(smem + at0 + m * 2048);
                const uint4 x1 = *reinterpret_cast<const uint4 *>(smem + at1 + m * 2048);
                const int xs = smem[ats + (BM * 128 + m * 64)];
                const i32x8_t x = {(int)x0.x, (int)x0.y, (int)x0.z, (int)x0.w, (int)x1.x, (int)x1.y, (int)x1.z, (int)x1.w};
                acc[0][m] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(w[0]), x, acc[0][m], 4, 0, 0, s, 0, xs);
                acc[1][m] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(w[1]), x, acc[1][m], 4, 0, 1, s, 0, xs);
                acc[2][m] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(w[2]), x, acc[2][m], 4, 0, 2, s, 0, xs);
                acc[3][m] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(w[3]), x, acc[3][m], 4, 0, 3, s, 0, xs);
            }
        };
        issue_w(0, d, ds);
        issue_a(0, 0);
        // no branch round the loads: their registers would be merged, and waited for, behind it
        for (int kt = 0; kt < KT - 1; ++kt) step(std::true_type{}, kt);
        step(std::false_type{}, KT - 1);
    };
    // one straight-line loop for each number of 16-row tiles that hold rows, and for
    // weights that no other tile reads, which are not kept in the caches (Qwen shape, T = 33 gate/up
    // 31.5 us against 35.8 kept, down 18.5 and 19.1; T = 1303, where most are read by two, nothing kept
    // 77 and 44 against 65 and 39)
    const int live = (min(BM, row_end - m0) + 15) / 16;
    auto run = [&](auto once) __attribute__((always_inline)) {
        if (live == 1) kloop(std::integral_constant<int, 1>{}, once);
        else if (live == 2) kloop(std::integral_constant<int, 2>{}, once);
        else if constexpr (TM == 4) {
            if (live == 3) kloop(std::integral_constant<int, 3>{}, once);
            else kloop(std::integral_constant<int, 4>{}, once);
        }
    };
    if (row_end - p.offsets[e] <= BM) run(std::true_type{});
    else run(std::false_type{});

    const int rows = min(BM, row_end - m0);
    if constexpr (Y32) {
        // four neighbouring columns a lane are 16 bytes already: out as they are, 64 bytes of a
        // row side by side and the next 64 by the store behind, and kept for the merge (4096
        // tokens of the DeepSeek-V2-Lite shape: 105 us and 37 in the merge, where bf16 rows take 84 and 21,
        // the bytes' time; not kept 108 and 43; 1303 of the Qwen shape 46 and 16 against 37 and 9)
        if (rg >= groups) return;
#pragma unroll
        for (int m = 0; m < TM; ++m) {
            if (16 * m + r >= rows) continue;
            float *y = reinterpret_cast<float *>(p.out) + (size_t)(m0 + 16 * m + r) * H + rg * kGroupRows + 4 * g;
#pragma unroll
            for (int i = 0; i < 4; ++i) *reinterpret_cast<f32x4_t *>(y + 16 * i) = acc[i][m];
        }
        return;
    }

    // ---- epilogue: a lane holds token row r of each tile and weight rows 4 g ..
    // + 3 of each 16-row tile; through LDS, out in whole-row 16-byte stores.  The 32
    // columns of h that a wave has of a row are one scale block, in four lanes.
    constexpr int OB = kMx8OutRow<GATEUP>;
    uint8_t *const out_s = smem + BM * OB;
    __syncthreads();
#pragma unroll
    for (int m = 0; m < TM; ++m) {
        if (m >= live) continue;
        uint8_t *row = smem + (16 * m + r) * OB;
        if constexpr (GATEUP) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) v[4 * i + q] = silu_fast(acc[i][m][q]) * acc[i + 2][m][q];
            const uint32_t byte = mx8_scale_byte(max_over_quarters(top_magnitude8(v)));
            const uint2 c = mx8_encode8(v, byte);
            *reinterpret_cast<uint32_t *>(row + wave * 32 + 4 * g) = c.x;
            *reinterpret_cast<uint32_t *>(row + wave * 32 + 16 + 4 * g) = c.y;
            if (g == 0) out_s[(16 * m + r) * NW + wave] = (uint8_t)byte;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x4_t v = acc[i][m];
                *reinterpret_cast<uint2 *>(row + wave * 128 + i * 32 + 8 * g) =
                    make_uint2(f2bf2_hw(v[0], v[1]), f2bf2_hw(v[2], v[3]));
            }
        }
    }
    __syncthreads();
    constexpr int CO = NW * (GATEUP ? 32 : 128), CH = CO / 16;  // bytes and 16-byte pieces of a row
    const int ldo = GATEUP ? I : 2 * H, bytes = min(CO, ldo - nt * CO);  // bytes % 128 == 0
    for (int c = tid; c < rows * CH; c += 64 * NW) {
        const int row = c / CH, ch = c % CH;
        if (ch * 16 < bytes)
            st_through(p.out + (size_t)(m0 + row) * ldo + nt * CO + ch * 16,
                       *reinterpret_cast<const uint4 *>(smem + row * OB + ch * 16));
    }
    if constexpr (GATEUP) {
        // scales: four bytes (128 columns) at a time
        for (int c = tid; c < rows * (NW / 4); c += 64 * NW) {
            const int row = c / (NW / 4), ch = c % (NW / 4);
            if (ch * 128 < bytes)
                *reinterpret_cast<uint32_t *>(p.out_scales + (size_t)(m0 + row) * (I / 32) + nt * NW + ch * 4) =
                    *reinterpret_cast<const uint32_t *>(out_s + row * NW + ch * 4);
        }
    }
}

struct Mx8Call {
    const int32_t *offsets, *sel;
    int nsel;
    const int32_t *tile_start;
    int max_tiles;
    const uint8_t *const *slots;
    int H, I;
    hipStream_t s;
};

template <int BM, int OCC, bool Y32>
static int mx8_grouped_launch(const Mx8Call &c, const uint8_t *x, const uint8_t *xs, const int32_t *perm, uint8_t *h,
                              uint8_t *hs, uint8_t *y) {
    constexpr int NW = kMx8Waves;
    auto grid = [&](int nt) { return (unsigned)(((size_t)c.max_tiles * nt + 7) / 8 * 8); };
    mx8_grouped_kernel<BM, true, OCC, false><<<grid((c.I / 32 + NW - 1) / NW), 64 * NW, 0, c.s>>>(
        Mx8Grouped{x, xs, perm, c.offsets, c.sel, c.nsel, c.tile_start, c.slots, c.H, c.I, h, hs});
    const int rc = check_launch("mx8_grouped_kernel<gateup>");
    if (rc) return rc;
    mx8_grouped_kernel<BM, false, OCC, Y32><<<grid((c.H / kGroupRows + NW - 1) / NW), 64 * NW, 0, c.s>>>(
        Mx8Grouped{h, hs, nullptr, c.offsets, c.sel, c.nsel, c.tile_start, c.slots, c.H, c.I, y, nullptr});
    return check_launch("mx8_grouped_kernel<down>");
}

}  // namespace pd

using namespace pd;

// 32-row tiles up to 16 rows an expert on average (Qwen shape, the whole layer: T = 256, 16
// rows, 58.3 us against 63.2 with 64; T = 400, 25 rows, 74.6 against 65.8): weights are read once a tile.
PD_API int pdscope_grouped_mxfp8_block_m(int rows_hint) { return rows_hint <= 16 ? 32 : 64; }

template <bool Y32>
static int swiglu_grouped_mxfp8(const void *x, const void *x_scales, const int32_t *perm_token, const int32_t *offsets,
                                const int32_t *sel, int nsel, const int32_t *tile_start, int max_tiles, int block_m,
                                const void *const *slots, int H, int I, void *h, void *h_scales, void *y, void *stream) {
    if (!x || !x_scales || !perm_token || !offsets || !sel || !tile_start || !slots || !h || !h_scales || !y)
        return fail(kEInval, "grouped_mxfp8: null pointer");
    if (nsel < 1 || max_tiles < 1 || max_tiles > (1 << 22))
        return fail(kEInval, "grouped_mxfp8: need nsel >= 1 and 1 <= max_tiles <= 4194304");
    if (block_m != 32 && block_m != 64) return fail(kEInval, "grouped_mxfp8: block_m must be 32 or 64");
    if (!mx_shape_ok(H, I) || H > 65536 || I > 65536)
        return fail(kEInval, "grouped_mxfp8: need H % 128 == 0 and I % 128 == 0 (at most 65536)");
    for (const void *p : {x, (const void *)h, (const void *)y})
        if (reinterpret_cast<uintptr_t>(p) % 16) return fail(kEInval, "grouped_mxfp8: x, h and y need 16-byte alignment");
    for (const void *p : {x_scales, (const void *)h_scales})
        if (reinterpret_cast<uintptr_t>(p) % 4) return fail(kEInval, "grouped_mxfp8: scales need 4-byte alignment");
    // a launch has fewer than 2^32 threads: 128 columns of h or 256 of y a workgroup of 256
    if ((int64_t)max_tiles * ((std::max(I, H / 2) + 127) / 128) * 256 > ((int64_t)1 << 32) - 8192)
        return fail(kEInval, "grouped_mxfp8: too many tiles for one launch");
    const Mx8Call c{offsets, sel, nsel, tile_start, max_tiles, (const uint8_t *const *)slots, H, I,
                    reinterpret_cast<hipStream_t>(stream)};
    auto *xc = (const uint8_t *)x, *xs = (const uint8_t *)x_scales;
    auto *hc = (uint8_t *)h, *hs = (uint8_t *)h_scales, *out = (uint8_t *)y;
    if (block_m == 32) return mx8_grouped_launch<32, 4, Y32>(c, xc, xs, perm_token, hc, hs, out);
    return mx8_grouped_launch<64, 2, Y32>(c, xc, xs, perm_token, hc, hs, out);
}

PD_API int pdscope_swiglu_grouped_mxfp8(const void *x, const void *x_scales, const int32_t *perm_token,
                                        const int32_t *offsets, const int32_t *sel, int nsel, const int32_t *tile_start,
                                        int max_tiles, int block_m, const void *const *slots, int H, int I, void *h,
                                        void *h_scales, void *y, void *stream) {
    return swiglu_grouped_mxfp8<false>(x, x_scales, perm_token, offsets, sel, nsel, tile_start, max_tiles, block_m, slots, H,
                                       I, h, h_scales, y, stream);
}

PD_API int pdscope_swiglu_grouped_mxfp8_y32(const void *x, const void *x_scales, const int32_t *perm_token,
                                            const int32_t *offsets, const int32_t *sel, int nsel,
                                            const int32_t *tile_start, int max_tiles, int block_m,
                                            const void *const *slots, int H, int I, void *h, void *h_scales, void *y,
                                            void *stream) {
    return swiglu_grouped_mxfp8<true>(x, x_scales, perm_token, offsets, sel, nsel, tile_start, max_tiles, block_m, slots, H, I,
                                      h, h_scales, y, stream);
}
