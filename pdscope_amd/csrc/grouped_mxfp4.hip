// The grouped SwiGLU expert FFN of grouped.hip over 4-bit expert blocks (layout:
// mxfp4.h), for prompts: restates expert_forward (expertbench/adapters/qwen.py:
// 87-90) for every selected expert at once.
//
//   gate/up : h[r,i] = bf16(silu(x_r . gate_i) * (x_r . up_i))
//   down    : y[r,n] = bf16(h_r . down_n)
//
// Weights are the first operand of v_mfma_f32_16x16x32_bf16 and never enter LDS:
// each wave of a tile has a 64-row group of them to itself, whose 4352 bytes for
// 128 inputs go from memory to the registers that hold them until they are
// decoded (16 conversions per lane and 16-row tile, used for every token tile).
// Activation rows are the second operand, shared by the waves: they stream into
// an LDS ring by direct-to-LDS loads, gathered through perm_token, in 256-byte
// rows whose 16-byte chunk c lies in slot c ^ (row % 16), so that the 16 rows of a
// fragment read lie in 16 bank groups.
//
// Thin experts are bound by HBM (Qwen shape T=33, medians of a trace: gate/up 33.4
// us, 5.6 TB/s, down 18.0 and 5.2; the fastest of 30 launches 32.1 and 17.5).  Long
// prompts reach 1.12 PFLOP/s in gate/up and 0.96 in down (Qwen shape T=4096,
// medians 185 and 108 us, the fastest 175 and 102; where a 128-row tile was timed beside
// it, 173 and 101 against 185 and 108): there the matrix cores are busy for 59% and
// 46% of the time, 22% and 34% of the waves' time is waits (barriers and loads: a
// step's loads have one step of three workgroups to land) and 19% and 16% vector
// instructions, the decoding of the weights among them.
// Measured on the 128-row tile and not kept: direct-to-LDS loads through buffer
// descriptors, which need no address arithmetic (1-3%, and 4 GiB of activations
// at most); weights two steps ahead (216 us); eight waves to a tile, which read
// the activations half as often (212); the products' order fixed by scheduling
// barriers (208).  On 64 rows: weight registers reloaded piece by piece (the layer 336
// us against 314); activation fragments read two or three ahead (the same); 32x32x16
// products (361 against 317).
//
// h, and each expert's row of y before the merge, are rounded to bf16 (out is off by
// three bf16 roundings in all, 0.0029 of its norm, against 0.0017 for its own alone).
// h is the matrix cores' input: a second part of it, as few.hip has one, would double the
// products of down, which bound a long prompt, and the workspace that holds h.  y is
// what pdscope_merge and the norms' launch read of either representation; in fp32
// it would be a quarter of the traffic of a long prompt on top.  Neither would cost
// time where experts are thin (T=33: y is 1 MB beside 283 MB of weights); there
// the types of h_ws and y are the reason, which are one for every length.
#include <algorithm>
#include <type_traits>

#include "mxfp4.h"
#include "ring.h"

namespace pd {

struct MxGrouped {
    const uint16_t *a;  // gate/up: x [T, H]; down: h [rows, I]
    const int32_t *perm_token, *offsets, *sel;
    int nsel;
    const int32_t *tile_start;
    const uint8_t *const *slots;
    int H, I;
    uint16_t *out;  // gate/up: h [rows, I]; down: y [rows, H]
};

// bytes of a staged output row: 32 columns of h or 64 of y per wave, off the bank line
template <int NW, bool GATEUP>
constexpr int kMxOutRow = NW * (GATEUP ? 64 : 128) + 16;
template <int BM, int NW, bool GATEUP>
constexpr int kMxLds = 2 * BM * 256 > BM * kMxOutRow<NW, GATEUP> ? 2 * BM * 256 : BM * kMxOutRow<NW, GATEUP>;

// BM rows x four groups (128 h columns or 256 y columns), K in steps of 128, two
// stages of activations; at least OCC workgroups per CU.
template <int BM, int NW, bool GATEUP, int OCC>
__global__ __launch_bounds__(64 * NW, OCC * NW / 4) void mx_grouped_kernel(MxGrouped p) {
    __shared__ __attribute__((aligned(1024))) uint8_t smem[kMxLds<BM, NW, GATEUP>];
    constexpr int TM = BM / 16;
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

    // ---- activation loads: load q of wave w fills rows 4 (NW q + w) .. + 3; lane l
    // takes row + l / 16 and the chunk that belongs in its slot
    constexpr int RQ = 4 * NW, AL = BM / RQ;  // rows per load of all waves, loads of a wave
    static_assert(RQ % 16 == 0 && AL * RQ == BM, "activation loads");
    uint32_t arow[AL];
    const uint32_t achunk = (uint32_t)((lane & 15) ^ ((4 * wave + (lane >> 4)) & 15));
#pragma unroll
    for (int q = 0; q < AL; ++q) {
        const int row = min(m0 + RQ * q + 4 * wave + (lane >> 4), row_end - 1);
        arow[q] = (uint32_t)(GATEUP ? p.perm_token[row] : row) * (uint32_t)(K / 8) + achunk;
    }
    const uint8_t *const abase = reinterpret_cast<const uint8_t *>(p.a);

    f32x4_t acc[4][TM];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int m = 0; m < TM; ++m) acc[i][m] = f32x4_t{};

    auto kloop = [&](auto live, auto once) __attribute__((always_inline)) {
        constexpr int L = decltype(live)::value;  // token tiles with rows of the expert
        auto ld = [](const uint8_t *q) { return decltype(once)::value ? ld_nt(q) : ld_g(q); };
        auto issue_a = [&](int kt) __attribute__((always_inline)) {
            uint8_t *st = smem + (kt & 1) * (BM * 256);
#pragma unroll
            for (int q = 0; q < (16 * L + RQ - 1) / RQ; ++q) {
                uint32_t o = arow[q];
                opaque(o);
                load_lds16(reinterpret_cast<const uint16_t *>(abase + kt * 256 + (size_t)o * 16),
                           st + (RQ * q + 4 * wave) * 256);
            }
        };
        auto issue_w = [&](int kt, uint4 (&d)[5]) __attribute__((always_inline)) {
            const uint8_t *b = wbase + (size_t)kt * kGroupBytes;
#pragma unroll
            for (int jj = 0; jj < 4; ++jj) d[jj] = ld(b + jj * 1024 + lane * 16);
            d[4] = ld(b + kGroupScales + r * 16);
        };
        // Step kt: everything asked for in step kt - 1 has landed (the one wait of
        // the step: loads to registers and to LDS complete in one order that the
        // compiler does not count through, so any wait of its own would be for
        // all of them, and here none is younger than a whole step); then ask for
        // kt + 1 and run the products of kt from d.
        auto step = [&](int kt, uint4 (&d)[5], uint4 (&next)[5]) __attribute__((always_inline)) {
            wait_vm<0>();
            ring_barrier();
            if (kt + 1 < KT) {
                issue_a(kt + 1);
                issue_w(kt + 1, next);
            }
            const uint8_t *st = smem + (kt & 1) * (BM * 256) + r * 256;
            bf16x8_t x[2][L];
            auto read_piece = [&](int jj) __attribute__((always_inline)) {
#pragma unroll
                for (int m = 0; m < L; ++m)
                    x[jj & 1][m] = *reinterpret_cast<const bf16x8_t *>(st + m * 4096 + (((4 * jj + g) ^ r) << 4));
            };
            read_piece(0);
#pragma unroll
            for (int jj = 0; jj < 4; ++jj) {
                if (jj < 3) read_piece(jj + 1);
                const uint32_t sw = jj == 0 ? d[4].x : jj == 1 ? d[4].y : jj == 2 ? d[4].z : d[4].w;
                const bf16x8_t w[4] = {mx_decode(d[jj].x, mx_scale<0>(sw)), mx_decode(d[jj].y, mx_scale<1>(sw)),
                                       mx_decode(d[jj].z, mx_scale<2>(sw)), mx_decode(d[jj].w, mx_scale<3>(sw))};
#pragma unroll
                for (int m = 0; m < L; ++m)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        acc[i][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[i], x[jj & 1][m], acc[i][m], 0, 0, 0);
            }
        };
        uint4 w0[5], w1[5];
        issue_w(0, w0);
        issue_a(0);
        for (int kt = 0; kt < KT; kt += 2) {
            step(kt, w0, w1);
            if (kt + 1 < KT) step(kt + 1, w1, w0);
        }
    };
    // one straight-line loop for each number of 16-row tiles that hold rows, and for
    // weights that no other tile reads, which are not kept in the caches
    // (the layer of the Qwen shape at T=33 66 -> 60 us, T=64 72 -> 64, T=512 95 -> 88;
    // all weights read so, T=4096 takes 335 against 315)
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

    // ---- epilogue: a lane holds token row r of each tile and weight rows 4 g ..
    // + 3 of each 16-row tile; through LDS, out in whole-row 16-byte stores
    constexpr int OB = kMxOutRow<NW, GATEUP>;
    __syncthreads();
#pragma unroll
    for (int m = 0; m < TM; ++m) {
        if (m >= live) continue;
        uint8_t *row = smem + (16 * m + r) * OB + (wave * (GATEUP ? 32 : 64) + 4 * g) * 2;
#pragma unroll
        for (int i = 0; i < (GATEUP ? 2 : 4); ++i) {
            f32x4_t v = acc[i][m];
            if (GATEUP) {
#pragma unroll
                for (int q = 0; q < 4; ++q) v[q] = silu_fast(v[q]) * acc[GATEUP ? i + 2 : i][m][q];
            }
            *reinterpret_cast<uint2 *>(row + i * 32) = make_uint2(f2bf2_hw(v[0], v[1]), f2bf2_hw(v[2], v[3]));
        }
    }
    __syncthreads();
    constexpr int CO = NW * (GATEUP ? 32 : 64), CH = CO / 8;
    const int ldo = GATEUP ? I : H, cols = min(CO, ldo - nt * CO);  // cols % 64 == 0
    const int rows = min(BM, row_end - m0);
    for (int c = tid; c < rows * CH; c += 64 * NW) {
        const int row = c / CH, ch = c % CH;
        if (ch * 8 < cols)
            st_through(p.out + (size_t)(m0 + row) * ldo + nt * CO + ch * 8,
                       *reinterpret_cast<const uint4 *>(smem + row * OB + ch * 16));
    }
}

struct MxCall {
    const int32_t *offsets, *sel;
    int nsel;
    const int32_t *tile_start;
    int max_tiles;
    const uint8_t *const *slots;
    int H, I;
    hipStream_t s;
};

// NWG / NWD waves and OCCG / OCCD workgroups per CU of the gate/up and down halves
template <int BM, int NWG, int OCCG, int NWD, int OCCD>
static int mx_grouped_launch(const MxCall &c, const uint16_t *x, const int32_t *perm, uint16_t *h, uint16_t *y) {
    auto grid = [&](int nt) { return (unsigned)(((size_t)c.max_tiles * nt + 7) / 8 * 8); };
    mx_grouped_kernel<BM, NWG, true, OCCG><<<grid((c.I / 32 + NWG - 1) / NWG), 64 * NWG, 0, c.s>>>(
        MxGrouped{x, perm, c.offsets, c.sel, c.nsel, c.tile_start, c.slots, c.H, c.I, h});
    const int rc = check_launch("mx_grouped_kernel<gateup>");
    if (rc) return rc;
    mx_grouped_kernel<BM, NWD, false, OCCD><<<grid((c.H / kGroupRows + NWD - 1) / NWD), 64 * NWD, 0, c.s>>>(
        MxGrouped{h, nullptr, c.offsets, c.sel, c.nsel, c.tile_start, c.slots, c.H, c.I, y});
    return check_launch("mx_grouped_kernel<down>");
}

}  // namespace pd

using namespace pd;

// Layers of the Qwen shape on 32 and 64 rows: 6 mean rows 68.0 and 71.9 us, 16
// 73.5 and 75.5, 24 89.0 and 82.4, 32 100.7 and 86.8, 44 113 and 103 (DeepSeek-V2-
// Lite shape, 6 mean rows 64.4 and 64.1, 24 75.8 and 71.6). A 128-row tile, whose
// weights are decoded once for twice the rows, is no faster anywhere (256 mean
// rows 322 against 314 then).
PD_API int pdscope_grouped_mxfp4_block_m(int rows_hint) { return rows_hint <= 16 ? 32 : 64; }

PD_API int pdscope_swiglu_grouped_mxfp4(const void *x, const int32_t *perm_token, const int32_t *offsets,
                                        const int32_t *sel, int nsel, const int32_t *tile_start, int max_tiles,
                                        int block_m, const void *const *slots, int H, int I, void *h_ws, void *y,
                                        void *stream) {
    if (!x || !perm_token || !offsets || !sel || !tile_start || !slots || !h_ws || !y)
        return fail(kEInval, "grouped_mxfp4: null pointer");
    if (nsel < 1 || max_tiles < 1 || max_tiles > (1 << 22))
        return fail(kEInval, "grouped_mxfp4: need nsel >= 1 and 1 <= max_tiles <= 4194304");
    if (block_m != 32 && block_m != 64) return fail(kEInval, "grouped_mxfp4: block_m must be 32 or 64");
    if (!mx_shape_ok(H, I) || H > 65536 || I > 65536)
        return fail(kEInval, "grouped_mxfp4: need H % 128 == 0 and I % 128 == 0 (at most 65536)");
    for (const void *p : {x, (const void *)h_ws, (const void *)y})
        if (reinterpret_cast<uintptr_t>(p) % 16) return fail(kEInval, "grouped_mxfp4: x, h_ws and y need 16-byte alignment");
    // a launch has fewer than 2^32 threads: at least 128 columns of h or 256 of y a workgroup
    // of 256, or 512 of y one of 512
    if ((int64_t)max_tiles * ((std::max(I, H / 2) + 127) / 128) * 256 > ((int64_t)1 << 32) - 8192)
        return fail(kEInval, "grouped_mxfp4: too many tiles for one launch");
    const MxCall c{offsets, sel, nsel, tile_start, max_tiles, (const uint8_t *const *)slots, H, I,
                   reinterpret_cast<hipStream_t>(stream)};
    auto *xs = (const uint16_t *)x;
    auto *h = (uint16_t *)h_ws, *out = (uint16_t *)y;
    // 32 rows: bound by the weight stream.  gate/up on four waves, four workgroups
    // per CU; down (a short K loop) on eight, two per CU: fewer, wider workgroups
    // read each expert's h fewer times (Qwen shape T=33, timed beside each other:
    // gate/up 31.0 us, eight waves 32.8; down 17.5, four waves 20.6).  64 rows: four waves;
    // three workgroups fit a CU (166 registers), whose steps interleave.
    if (block_m == 32) return mx_grouped_launch<32, 4, 4, 8, 2>(c, xs, perm_token, h, out);
    return mx_grouped_launch<64, 4, 2, 4, 2>(c, xs, perm_token, h, out);
}
