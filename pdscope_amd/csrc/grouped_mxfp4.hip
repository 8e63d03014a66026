// The grouped SwiGLU expert FFN of grouped.hip over 4-bit expert blocks (layout:
// mxfp4.h), for prompts: restates expert_forward (expertbench/adapters/qwen.py:
// 87-90) for every selected expert at once.
//
//   gate/up : h[r,i] = bf16(silu(x_r . gate_i) * (x_r . up_i))
//   down    : y[r,n] = bf16(h_r . down_n)
//
// Weights are the first operand of v_mfma_f32_16x16x32_bf16 and never enter LDS: a
// wave's four waves' worth of a tile is four 64-row groups, one per wave, and a
// group's 4352 bytes for 128 inputs go from memory to the registers that hold
// them until they are decoded (16 conversions per lane and 16-row tile, used for
// every token tile).  Activation rows are the second operand, shared by the four
// waves: they stream into an LDS ring by direct-to-LDS loads, gathered through
// perm_token, in 256-byte rows whose 16-byte chunk c lies in slot c ^ (row % 16),
// so that the 16 rows of a fragment read lie in 16 bank groups.
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

// bytes of a staged output row: 128 columns of h or 256 of y, off the bank line
template <bool GATEUP>
constexpr int kMxOutRow = (GATEUP ? 256 : 512) + 16;
template <int BM, int S, bool GATEUP>
constexpr int kMxLds = S * BM * 256 > BM * kMxOutRow<GATEUP> ? S * BM * 256 : BM * kMxOutRow<GATEUP>;

// BM rows x four groups (128 h columns or 256 y columns), K in steps of 128, S
// stages of activations.
template <int BM, int S, bool GATEUP, int OCC>
__global__ __launch_bounds__(256, OCC) void mx_grouped_kernel(MxGrouped p) {
    __shared__ __attribute__((aligned(1024))) uint8_t smem[kMxLds<BM, S, GATEUP>];
    constexpr int TM = BM / 16, PF = 2;
    const int H = p.H, I = p.I;
    const int K = GATEUP ? H : I, KT = K / kGroupIn;
    const int groups = GATEUP ? I / 32 : H / kGroupRows, NT = (groups + 3) / 4;

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
    const int rg = nt * 4 + wave;             // this wave's row group
    const int rg_in = min(rg, groups - 1);    // past the end: read the last one, store nothing
    const uint8_t *const wbase =
        base + ((GATEUP ? 0 : mx_gateup_groups(H, I)) + (size_t)rg_in * KT) * kGroupBytes;

    // ---- activation loads: load q of wave w fills rows 16 q + 4 w .. + 3; lane l
    // takes row + l / 16 and the chunk that belongs in its slot
    uint32_t arow[TM];
    const uint32_t achunk = (uint32_t)((lane & 15) ^ (4 * wave + (lane >> 4)));
#pragma unroll
    for (int q = 0; q < TM; ++q) {
        const int row = min(m0 + 16 * q + 4 * wave + (lane >> 4), row_end - 1);
        arow[q] = (uint32_t)(GATEUP ? p.perm_token[row] : row) * (uint32_t)(K / 8) + achunk;
    }
    const uint8_t *const abase = reinterpret_cast<const uint8_t *>(p.a);

    f32x4_t acc[4][TM];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int m = 0; m < TM; ++m) acc[i][m] = f32x4_t{};

    auto kloop = [&](auto live) __attribute__((always_inline)) {
        constexpr int L = decltype(live)::value;  // token tiles with rows of the expert
        // loads that follow those of stage kt by the time it is needed: the weights
        // of its own step (all PF of them for the first stages, whose steps lie in
        // the prologue), and both kinds of the S - 2 steps between
        constexpr int YOUNGER = (S - 2) * L + 5 * (S - 1 < PF ? S - 1 : PF);
        auto issue_a = [&](int kt) __attribute__((always_inline)) {
            uint8_t *st = smem + (kt % S) * (BM * 256);
#pragma unroll
            for (int q = 0; q < L; ++q) {
                uint32_t o = arow[q];
                opaque(o);
                load_lds16(reinterpret_cast<const uint16_t *>(abase + kt * 256 + (size_t)o * 16),
                           st + (16 * q + 4 * wave) * 256);
            }
        };
        uint4 w[PF][5];
        auto issue_w = [&](int kt, uint4 (&d)[5]) __attribute__((always_inline)) {
            const uint8_t *b = wbase + (size_t)kt * kGroupBytes;
#pragma unroll
            for (int jj = 0; jj < 4; ++jj) d[jj] = ld_g(b + jj * 1024 + lane * 16);
            d[4] = ld_g(b + kGroupScales + r * 16);
        };
        auto step = [&](int kt, uint4 (&d)[5], auto steady) __attribute__((always_inline)) {
            constexpr bool STEADY = decltype(steady)::value;
            // this wave's share of stage kt has landed; with the barrier, everyone's
            if (STEADY) wait_vm<YOUNGER>();
            else wait_vm<0>();
            ring_barrier();
            if (STEADY || kt + S - 1 < KT) issue_a(kt + S - 1);
            // the count above needs these loads ahead of the weights' that follow
            asm volatile("" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
            const uint8_t *st = smem + (kt % S) * (BM * 256);
#pragma unroll
            for (int jj = 0; jj < 4; ++jj) {
                const uint32_t sw = jj == 0 ? d[4].x : jj == 1 ? d[4].y : jj == 2 ? d[4].z : d[4].w;
                const bf16x8_t w0 = mx_decode(d[jj].x, mx_scale<0>(sw)), w1 = mx_decode(d[jj].y, mx_scale<1>(sw));
                const bf16x8_t w2 = mx_decode(d[jj].z, mx_scale<2>(sw)), w3 = mx_decode(d[jj].w, mx_scale<3>(sw));
#pragma unroll
                for (int m = 0; m < L; ++m) {
                    const bf16x8_t x =
                        *reinterpret_cast<const bf16x8_t *>(st + (16 * m + r) * 256 + (((4 * jj + g) ^ r) << 4));
                    acc[0][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w0, x, acc[0][m], 0, 0, 0);
                    acc[1][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w1, x, acc[1][m], 0, 0, 0);
                    acc[2][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w2, x, acc[2][m], 0, 0, 0);
                    acc[3][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w3, x, acc[3][m], 0, 0, 0);
                }
            }
            if (STEADY || kt + PF < KT) issue_w(kt + PF, d);
        };
#pragma unroll
        for (int s = 0; s < S - 1; ++s)
            if (s < KT) issue_a(s);
#pragma unroll
        for (int s = 0; s < PF; ++s)
            if (s < KT) issue_w(s, w[s]);
        int kt = 0;
        for (; kt + 1 + (S - 1 > PF ? S - 1 : PF) < KT; kt += 2) {
            step(kt, w[0], std::true_type{});
            step(kt + 1, w[1], std::true_type{});
        }
        for (; kt < KT; kt += 2) {
            step(kt, w[0], std::false_type{});
            if (kt + 1 < KT) step(kt + 1, w[1], std::false_type{});
        }
    };
    // whole quarters of the tile that hold rows
    const int live = (min(BM, row_end - m0) + 15) / 16;
    if constexpr (TM >= 4) {
        if (4 * live <= TM) kloop(std::integral_constant<int, TM / 4>{});
        else if (2 * live <= TM) kloop(std::integral_constant<int, TM / 2>{});
        else if (4 * live <= 3 * TM) kloop(std::integral_constant<int, 3 * TM / 4>{});
        else kloop(std::integral_constant<int, TM>{});
    } else {
        if (live == 1) kloop(std::integral_constant<int, 1>{});
        else kloop(std::integral_constant<int, TM>{});
    }

    // ---- epilogue: a lane holds token row r of each tile and weight rows 4 g ..
    // + 3 of each 16-row tile; through LDS, out in whole-row 16-byte stores
    constexpr int OB = kMxOutRow<GATEUP>;
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
    constexpr int CO = GATEUP ? 128 : 256, CH = CO / 8;
    const int ldo = GATEUP ? I : H, cols = min(CO, ldo - nt * CO);  // cols % 64 == 0
    const int rows = min(BM, row_end - m0);
    for (int c = tid; c < rows * CH; c += 256) {
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

template <int BM, int S, int OCC>
static int mx_grouped_launch(const MxCall &c, const uint16_t *x, const int32_t *perm, uint16_t *h, uint16_t *y) {
    auto grid = [&](int nt) { return (unsigned)(((size_t)c.max_tiles * nt + 7) / 8 * 8); };
    mx_grouped_kernel<BM, S, true, OCC><<<grid(c.I / 128), 256, 0, c.s>>>(
        MxGrouped{x, perm, c.offsets, c.sel, c.nsel, c.tile_start, c.slots, c.H, c.I, h});
    const int rc = check_launch("mx_grouped_kernel<gateup>");
    if (rc) return rc;
    mx_grouped_kernel<BM, S, false, OCC><<<grid((c.H / kGroupRows + 3) / 4), 256, 0, c.s>>>(
        MxGrouped{h, nullptr, c.offsets, c.sel, c.nsel, c.tile_start, c.slots, c.H, c.I, y});
    return check_launch("mx_grouped_kernel<down>");
}

}  // namespace pd

using namespace pd;

PD_API int pdscope_grouped_mxfp4_block_m(int rows_hint) { return rows_hint <= 16 ? 32 : rows_hint <= 44 ? 64 : 128; }

PD_API int pdscope_swiglu_grouped_mxfp4(const void *x, const int32_t *perm_token, const int32_t *offsets,
                                        const int32_t *sel, int nsel, const int32_t *tile_start, int max_tiles,
                                        int block_m, const void *const *slots, int H, int I, void *h_ws, void *y,
                                        void *stream) {
    if (!x || !perm_token || !offsets || !sel || !tile_start || !slots || !h_ws || !y)
        return fail(kEInval, "grouped_mxfp4: null pointer");
    if (nsel < 1 || max_tiles < 1 || max_tiles > (1 << 22))
        return fail(kEInval, "grouped_mxfp4: need nsel >= 1 and 1 <= max_tiles <= 4194304");
    if (block_m != 32 && block_m != 64 && block_m != 128)
        return fail(kEInval, "grouped_mxfp4: block_m must be 32, 64 or 128");
    if (!mx_shape_ok(H, I) || H > 65536 || I > 65536)
        return fail(kEInval, "grouped_mxfp4: need H % 128 == 0 and I % 128 == 0 (at most 65536)");
    for (const void *p : {x, (const void *)h_ws, (const void *)y})
        if (reinterpret_cast<uintptr_t>(p) % 16) return fail(kEInval, "grouped_mxfp4: x, h_ws and y need 16-byte alignment");
    const MxCall c{offsets, sel, nsel, tile_start, max_tiles, (const uint8_t *const *)slots, H, I,
                   reinterpret_cast<hipStream_t>(stream)};
    auto *xs = (const uint16_t *)x;
    auto *h = (uint16_t *)h_ws, *out = (uint16_t *)y;
    if (block_m == 32) return mx_grouped_launch<32, 4, 2>(c, xs, perm_token, h, out);
    if (block_m == 64) return mx_grouped_launch<64, 3, 2>(c, xs, perm_token, h, out);
    return mx_grouped_launch<128, 2, 2>(c, xs, perm_token, h, out);
}
