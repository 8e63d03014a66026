// y = x W^T + bias over a 4-bit matrix with group scales (int4.h): the attention's
// projections and the vocabulary head of a model whose experts run here, which
// the reference leaves to the model's torch modules
// (benchmarks/pdscope_compare.py:198-212).
//
//   y[t, n] = bf16(sum_groups s[n] * (sum_k q[n, k] x[t, k] - z[n] * sum_k x[t, k]) + bias[n])
//
// The whole numbers q are bf16 exactly, so the products with x are exact and a
// group's two sums are held in fp32; the scale enters once a group, in fp32.
//
// Three launches: up to 16 rows of x against many of W with x in registers
// (i4_rows_kernel), few rows with the K axis split over the waves of a workgroup
// (i4_split_kernel), many in tiles through LDS (i4_gemm_kernel).  The first two are
// bound by W's bytes or, for small matrices, by a launch's start, one load and one join: N = 151936, K
// = 2048, G = 64 with zero points, one row 36 us (4.7 TB/s); K = 4096, G = 128 64 us (5.0); N = 2048,
// K = 4096 4.8 us (0.9).  With 16 rows x's bytes cost as much, read again by every workgroup: N = 4096, K
// = 2048 5.1 us, N = 151936, K = 4096 82.
#include <algorithm>
#include <type_traits>

#include "int4.h"
#include "ring.h"

namespace pd {

struct I4Linear {
    const uint8_t *w;
    const uint16_t *x, *bias;
    uint16_t *y;
    int T, N, K;
    int piece;  // outputs that one store takes: 8, 2 or 1, of whose size every row's start is a multiple
};

// What a wave holds of a unit: codes, and its rows' scales and zero points (rows 4 g .. +
// 3, a group each).
template <int G, bool ZEROS, bool FP16>
struct I4Unit {
    static constexpr int GP = kI4In / G, JG = 4 / GP;  // groups of a unit, words of a group
    uint4 c;
    I4Side<G, ZEROS, FP16> side;

    // KEEP: another workgroup reads the weights too.
    template <bool KEEP>
    __device__ __forceinline__ void load(const uint8_t *unit, int lane) {
        c = KEEP ? ld_g(unit + 16 * lane) : ld_nt(unit + 16 * lane);
        side.load(unit, lane >> 4);
    }

    // sx: the groups' sums of x, the same in every register of a column
    template <int MT>
    __device__ __forceinline__ void add(const bf16x8_t (&x)[MT][4], const float (&sx)[MT][GP], f32x4_t (&tot)[MT]) const {
        const uint32_t words[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
        for (int gi = 0; gi < GP; ++gi) {
            f32x4_t acc[MT];
#pragma unroll
            for (int m = 0; m < MT; ++m) acc[m] = f32x4_t{};
#pragma unroll
            for (int j = gi * JG; j < (gi + 1) * JG; ++j) {
                const bf16x8_t w = i4_decode(words[j]);
#pragma unroll
                for (int m = 0; m < MT; ++m) acc[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, x[m][j], acc[m], 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float sc = side.scale(gi, i), zp = side.zero(gi, i);
#pragma unroll
                for (int m = 0; m < MT; ++m) tot[m][i] = fmaf(sc, fmaf(-zp, sx[m][gi], acc[m][i]), tot[m][i]);
            }
        }
    }
};

// Four neighbouring outputs of a token, from row n on.
__device__ __forceinline__ void i4_store(const I4Linear &p, int t, int n, f32x4_t v, const float (&bias)[4]) {
    const uint32_t lo = f2bf2_hw(v[0] + bias[0], v[1] + bias[1]), hi = f2bf2_hw(v[2] + bias[2], v[3] + bias[3]);
    uint16_t *y = p.y + (size_t)t * p.N + n;
    if (n + 3 < p.N && p.piece == 8) {
        *reinterpret_cast<uint2 *>(y) = make_uint2(lo, hi);
    } else {
        if (n < p.N) y[0] = (uint16_t)lo;
        if (n + 1 < p.N) y[1] = (uint16_t)(lo >> 16);
        if (n + 2 < p.N) y[2] = (uint16_t)hi;
        if (n + 3 < p.N) y[3] = (uint16_t)(hi >> 16);
    }
}
__device__ __forceinline__ void i4_bias(const I4Linear &p, int n, float (&bias)[4]) {
#pragma unroll
    for (int q = 0; q < 4; ++q) bias[q] = p.bias ? bf2f(p.bias[min(n + q, p.N - 1)]) : 0.0f;
}

// A workgroup: RT tiles of 16 rows of W x MT tiles of 16 tokens, the units of the K
// axis dealt to WV waves, whose parts meet in LDS.
template <int G, bool ZEROS, bool FP16, int RT, int MT, int WV, bool KEEP>
__global__ __launch_bounds__(64 * WV) void i4_split_kernel(I4Linear p) {
    constexpr int UB = i4_unit_bytes(G, ZEROS), GP = kI4In / G, JG = 4 / GP;
    __shared__ f32x4_t s_part[WV][RT * MT][64];
    const int lane = lane_id(), ks = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int tiles = (p.N + kI4Rows - 1) / kI4Rows, KU = (p.K + kI4In - 1) / kI4In, across = (tiles + RT - 1) / RT;
    const int tb = blockIdx.x / across, n0 = (blockIdx.x - tb * across) * RT;
    const uint8_t *wt[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) wt[i] = p.w + (size_t)min(n0 + i, tiles - 1) * KU * UB;
    const uint16_t *xr[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) xr[m] = p.x + (size_t)min((tb * MT + m) * 16 + r, p.T - 1) * p.K;
    const __bf16 one = (__bf16)1.0f;
    const bf16x8_t ones = {one, one, one, one, one, one, one, one};

    f32x4_t tot[RT][MT];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int m = 0; m < MT; ++m) tot[i][m] = f32x4_t{};
    for (int u = ks; u < KU; u += WV) {
        I4Unit<G, ZEROS, FP16> d[RT];
#pragma unroll
        for (int i = 0; i < RT; ++i) d[i].template load<KEEP>(wt[i] + (size_t)u * UB, lane);
        // inputs past the end of a row are read as its last ones: their scales are 0
        bf16x8_t x[MT][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int k = min(u * kI4In + 32 * j + 8 * g, p.K - 8);
#pragma unroll
            for (int m = 0; m < MT; ++m) x[m][j] = __builtin_bit_cast(bf16x8_t, ld_g(xr[m] + k));
        }
        if (RT > 1) __builtin_amdgcn_sched_barrier(0);  // all loads before the first wait
        float sx[MT][GP];
#pragma unroll
        for (int gi = 0; gi < GP; ++gi)
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                f32x4_t a = {};
#pragma unroll
                for (int j = gi * JG; j < (gi + 1) * JG; ++j) a = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, x[m][j], a, 0, 0, 0);
                sx[m][gi] = a[0];
            }
#pragma unroll
        for (int i = 0; i < RT; ++i) d[i].add(x, sx, tot[i]);
    }
    // ---- the waves' parts, in order; lane l has token r and rows 4 g .. + 3
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int m = 0; m < MT; ++m) s_part[ks][i * MT + m][lane] = tot[i][m];
    __syncthreads();
    for (int q = threadIdx.x; q < RT * MT * 64; q += 64 * WV) {
        const int at = q >> 6, l = q & 63, t = (tb * MT + at % MT) * 16 + (l & 15), n = (n0 + at / MT) * 16 + 4 * (l >> 4);
        if (t >= p.T) continue;
        float bias[4];
        i4_bias(p, n, bias);
        f32x4_t v = s_part[0][at][l];
#pragma unroll
        for (int w = 1; w < WV; ++w) v += s_part[w][at][l];
        i4_store(p, t, n, v, bias);
    }
}

constexpr int kI4RowsWaves = 8, kI4RowsUnits = 2;

// Up to 16 tokens, K up to 2048.  Each wave keeps two units' worth of x (and its groups'
// sums, which do not depend on the row) in registers and takes these units of
// one row tile after the other, the tiles ahead on their way while it works on one; the
// waves' parts meet in LDS.
template <int G, bool ZEROS, bool FP16>
__global__ __launch_bounds__(64 * kI4RowsWaves) void i4_rows_kernel(I4Linear p) {
    constexpr int WV = kI4RowsWaves, U = kI4RowsUnits;
    constexpr int UB = i4_unit_bytes(G, ZEROS), GP = kI4In / G, JG = 4 / GP;
    __shared__ f32x4_t s_part[2][WV][64];
    const int lane = lane_id(), ks = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int tiles = (p.N + kI4Rows - 1) / kI4Rows, KU = (p.K + kI4In - 1) / kI4In, stride = gridDim.x;
    struct Held {
        u32x4_t c;
        I4Side<G, ZEROS, FP16> side;
    };
    // units past the end are read as the last one, with an x of 0; tiles past the end as
    // the first one, whose sums are not used: no branch round a load, whose registers would be
    // waited for behind it
    auto load = [&](int tile, Held (&d)[U]) __attribute__((always_inline)) {
        const uint8_t *at = p.w + (size_t)(tile < tiles ? tile : 0) * KU * UB;
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const uint8_t *unit = at + (size_t)min(ks * U + i, KU - 1) * UB;
            d[i].c = __builtin_nontemporal_load(gptr(unit + 16 * lane));
            d[i].side.load(unit, g);
        }
    };
    Held d0[U], d1[U], d2[U];
    load(blockIdx.x, d0);

    bf16x8_t x[U][4];
    float sx[U][GP];
    const uint16_t *xr = p.x + (size_t)min(r, p.T - 1) * p.K;
    const __bf16 one = (__bf16)1.0f;
    const bf16x8_t ones = {one, one, one, one, one, one, one, one};
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int k = (ks * U + i) * kI4In + 32 * j + 8 * g;
            uint4 v = ld_g(xr + min(k, p.K - 8));
            if (k >= p.K) v = make_uint4(0, 0, 0, 0);
            x[i][j] = __builtin_bit_cast(bf16x8_t, v);
        }
    load(blockIdx.x + stride, d1);
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
        for (int gi = 0; gi < GP; ++gi) {
            f32x4_t a = {};
#pragma unroll
            for (int j = gi * JG; j < (gi + 1) * JG; ++j) a = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, x[i][j], a, 0, 0, 0);
            sx[i][gi] = a[0];
        }

    // tile it of this workgroup from d; the one after the next is asked for, into ahead
    auto step = [&](int tile, int it, const Held (&d)[U], Held (&ahead)[U]) __attribute__((always_inline)) {
        const bool mine = ks == it % WV;
        float bias[4];
        if (mine) i4_bias(p, tile * 16 + 4 * g, bias);
        load(tile + 2 * stride, ahead);
        f32x4_t tot = {};
#pragma unroll
        for (int i = 0; i < U; ++i)
#pragma unroll
            for (int gi = 0; gi < GP; ++gi) {
                f32x4_t acc = {};
#pragma unroll
                for (int j = gi * JG; j < (gi + 1) * JG; ++j)
                    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(i4_decode(d[i].c[j]), x[i][j], acc, 0, 0, 0);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    tot[q] = fmaf(d[i].side.scale(gi, q), fmaf(-d[i].side.zero(gi, q), sx[i][gi], acc[q]), tot[q]);
                }
            }
        // two buffers in turn: who sums tile it is at the barrier of it + 1 before
        // anyone writes the same buffer for it + 2
        f32x4_t(&part)[WV][64] = s_part[it & 1];
        if (r < p.T) part[ks][lane] = tot;
        ring_barrier();
        if (mine && r < p.T) {
            f32x4_t v = part[0][lane];
#pragma unroll
            for (int w = 1; w < WV; ++w) v += part[w][lane];
            i4_store(p, r, tile * 16 + 4 * g, v, bias);
        }
    };
    int tile = blockIdx.x;
    for (int it = 0;; it += 3) {
        step(tile, it, d0, d2);
        if ((tile += stride) >= tiles) break;
        step(tile, it + 1, d1, d0);
        if ((tile += stride) >= tiles) break;
        step(tile, it + 2, d2, d1);
        if ((tile += stride) >= tiles) break;
    }
}

// ---- many tokens

constexpr int kI4GemmM = 64;
constexpr int kI4GemmX = kI4GemmM * 256;           // a stage's x, behind it its scales:
constexpr int kI4GemmStage = kI4GemmX + 4 * 512;  // 128 bytes at most for each of four tiles of four waves

// 64 tokens x 64 RT rows of W, K in steps of 128: a wave has RT row tiles to
// itself, whose codes go from memory to registers a step ahead; x streams through two LDS
// stages in 256-byte rows whose 16-byte chunk c lies in slot c ^ (row % 16).  The
// steps are dealt to KS parts of the workgroup, whose totals meet in LDS.
//
// A step of RT = 4 issues 64 products and 4 for the sums, and some 220 other vector
// instructions (112 decode, 64 scale) through the same port, so two waves take about 3100 cycles
// where the products alone need 2200.  N = 4096, K = 2048, G = 128, T = 2048 37 to
// 38 us in a row of launches (42 traced one by one), 0.90 PFLOP/s (G = 64 43, G = 32 56), of which the loop 26, what is before and behind it
// 4.3; without the loop's loads 33.6, without decoding 35.8, without reading x from LDS 30.4.  T = 4096 and
// K = 4096 1.0 PFLOP/s.  Held back by neither alone; reading x 32 inputs ahead of the products or
// another order of them changed nothing.  RT = 2 without parts has 168 registers, for three workgroups a
// CU (T = 1100 30.5 us against 34.5 with two).
template <int G, bool ZEROS, bool FP16, int RT, int KS>
__global__ __launch_bounds__(256 * KS, KS > 2 ? KS : KS == 1 && RT == 2 ? 3 : 2) void i4_gemm_kernel(I4Linear p, int cut) {
    constexpr int UB = i4_unit_bytes(G, ZEROS), GP = kI4In / G, JG = 4 / GP;
    constexpr int kN = 64 * RT, kOut = kN * 2 + 16;          // rows of W, bytes of a staged output row
    constexpr int kSums = KS > 2 ? 8 : 16;                   // groups whose sums of x are kept at a time
    constexpr int kParts = (KS - 1) * 4 * RT * 4 * 64 * 16;  // fp32 totals of the waves of the other parts of K
    __shared__ __attribute__((aligned(1024))) uint8_t smem_all[std::max({KS * 2 * kI4GemmStage, kParts, kI4GemmM * kOut})];
    __shared__ float s_sums_all[KS][2][kSums][kI4GemmM];
    const int tid = threadIdx.x, lane = tid & 63, wave_all = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int part = wave_all >> 2, wave = wave_all & 3;  // its part of the steps, its row tiles
    uint8_t *const smem = smem_all + part * (2 * kI4GemmStage);
    float(&s_sums)[2][kSums][kI4GemmM] = s_sums_all[part];
    const int r = lane & 15, g = lane >> 4;
    const int tiles = (p.N + kI4Rows - 1) / kI4Rows, KT = (p.K + kI4In - 1) / kI4In;
    // the tiles in `cut` x 8 / `cut` rectangles, one per XCD: tokens and rows of W whose
    // sum in bytes is least, for its L2; tokens fastest
    const int TB = (p.T + kI4GemmM - 1) / kI4GemmM, NB = (p.N + kN - 1) / kN;
    const int xcd = blockIdx.x & 7, pos = blockIdx.x >> 3, per_t = (TB + cut - 1) / cut, per_n = (NB * cut + 7) / 8;
    const int tb = xcd % cut * per_t + pos % per_t, nb = xcd / cut * per_n + pos / per_t;
    if (tb >= TB || nb >= NB) return;
    const int t0 = tb * kI4GemmM, n0 = nb * kN;

    const uint8_t *wt[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) wt[i] = p.w + (size_t)min(n0 / 16 + RT * wave + i, tiles - 1) * KT * UB;
    // x loads: load q of wave w fills rows 16 q + 4 w .. + 3; lane l takes row + l / 16 and
    // the chunk that belongs in its slot
    const uint16_t *xrow[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) xrow[q] = p.x + (size_t)min(t0 + 16 * q + 4 * wave + (lane >> 4), p.T - 1) * p.K;
    const int chunk = (lane & 15) ^ ((4 * wave + (lane >> 4)) & 15);

    // scales: lanes 2 GP i .. + 2 GP - 1 take row tile i's
    const uint8_t *const scales =
        p.w + (size_t)min(n0 / 16 + RT * wave + min(lane / (2 * GP), RT - 1), tiles - 1) * KT * UB + kI4Codes + lane % (2 * GP) * 16;

    // Loads and reads of different stages go through __restrict__ pointers: the compiler
    // lets no LDS read pass a direct-to-LDS load in flight that may write what it reads.
    auto issue_x = [&](int kt, uint8_t *__restrict__ st) __attribute__((always_inline)) {
        // past the end of a row: its last inputs, whose scales are 0
        const uint32_t at = (uint32_t)min(kt * 16 + chunk, p.K / 8 - 1);
#pragma unroll
        for (int q = 0; q < 4; ++q)
            load_lds16(xrow[q] + (size_t)at * 8, st + (16 * q + 4 * wave) * 256);
        if (lane < 2 * RT * GP) load_lds16(reinterpret_cast<const uint16_t *>(scales + (size_t)kt * UB), st + kI4GemmX + 512 * wave);
    };
    const uint32_t lane16 = 16 * (uint32_t)lane;
    auto issue_w = [&](int kt, u32x4_t (&d)[RT]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < RT; ++i) d[i] = *gptr(wt[i] + (size_t)kt * UB + lane16);
    };
    u32x4_t ahead[RT];
    issue_w(min(part, KT - 1), ahead);
    issue_x(min(part, KT - 1), smem);

    f32x4_t tot[RT][4];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int m = 0; m < 4; ++m) tot[i][m] = f32x4_t{};
    const int groups = p.K / G;
    const __bf16 one = (__bf16)1.0f;
    const bf16x8_t ones = {one, one, one, one, one, one, one, one};

    // What the zero points take off: tot -= sum of (s z)[n] sx[t] over up to kSums groups from
    // q0 on, whose sums of x lie in s_sums: fp32 products of four groups at a time
    auto take_off = [&](int q0) __attribute__((always_inline)) {
        const float *const sums = &s_sums[q0 / kSums & 1][0][0];
        uint32_t sz[kSums / 4][RT], zz[kSums / 4][RT];
#pragma unroll
        for (int q = 0; q < kSums / 4; ++q) {
            const uint32_t own = q0 + 4 * q + g, gr = min((own / GP * KS + part) * GP + own % GP, (uint32_t)groups - 1);
            const uint32_t at = gr / GP * UB + i4_scale_at<uint32_t>(r, gr % GP, GP), zt = gr / GP * UB + i4_zero_at<uint32_t>(r, gr % GP, GP);
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                sz[q][i] = *reinterpret_cast<const uint16_t *>(wt[i] + at);
                zz[q][i] = ZEROS ? wt[i][zt] : 8;
            }
        }
#pragma unroll
        for (int q = 0; q < kSums / 4; ++q) {
            const uint32_t own = q0 + 4 * q + g;  // the part's group; the row's:
            const bool on = (own / GP * KS + part) * GP + own % GP < (uint32_t)groups;
            float b[4];
#pragma unroll
            for (int m = 0; m < 4; ++m) b[m] = on ? sums[(4 * q + g) * kI4GemmM + 16 * m + r] : 0.0f;
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                const float a = on ? -i4_scale(sz[q][i], FP16) * (float)zz[q][i] : 0.0f;
#pragma unroll
                for (int m = 0; m < 4; ++m) tot[i][m] = __builtin_amdgcn_mfma_f32_16x16x4f32(a, b[m], tot[i][m], 0, 0, 0);
            }
        }
    };

    auto step = [&](int it, const uint8_t *__restrict__ cur, uint8_t *__restrict__ nxt)
        __attribute__((always_inline)) {
        const int kt = it * KS + part;
        wait_vm<0>();
        ring_barrier();
        if (it && it * GP % kSums == 0) take_off(it * GP - kSums);
        u32x4_t d[RT];
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            d[i] = ahead[i];
            asm volatile("" : "+v"(d[i]));
        }
        issue_x(min(kt + KS, KT - 1), nxt);
        issue_w(min(kt + KS, KT - 1), ahead);
        __builtin_amdgcn_sched_barrier(0);
        if (KS > 1 && kt >= KT) return;
        const uint8_t *st = cur + r * 256, *sc = cur + kI4GemmX + 512 * wave + g * (8 * GP);
#pragma unroll
        for (int gi = 0; gi < GP; ++gi) {
            bf16x8_t x[JG][4];
#pragma unroll
            for (int j = 0; j < JG; ++j)
#pragma unroll
                for (int m = 0; m < 4; ++m)
                    x[j][m] = *reinterpret_cast<const bf16x8_t *>(st + m * 4096 + (((4 * (gi * JG + j) + g) ^ r) << 4));
            // the group's sums of x, of the wave's own token tile
            f32x4_t sx = {};
#pragma unroll
            for (int j = 0; j < JG; ++j)
                sx = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                    ones, *reinterpret_cast<const bf16x8_t *>(st + wave * 4096 + (((4 * (gi * JG + j) + g) ^ r) << 4)), sx, 0, 0, 0);
            const int gr = it * GP + gi;
            // (of every g the same value: a branch round this store has registers spilled)
            s_sums[gr / kSums & 1][gr % kSums][16 * wave + r] = sx[0];
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                f32x4_t acc[4];
#pragma unroll
                for (int j = 0; j < JG; ++j) {
                    const bf16x8_t w = i4_decode(d[i][gi * JG + j]);
#pragma unroll
                    for (int m = 0; m < 4; ++m)
                        acc[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, x[j][m], j == 0 ? f32x4_t{} : acc[m], 0, 0, 0);
                }
                const uint2 s4 = *reinterpret_cast<const uint2 *>(sc + i * (32 * GP) + gi * 8);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float s = i4_scale((q < 2 ? s4.x : s4.y) >> (16 * (q & 1)) & 0xffffu, FP16);
#pragma unroll
                    for (int m = 0; m < 4; ++m) tot[i][m][q] = fmaf(s, acc[m][q], tot[i][m][q]);
                }
            }
            if (GP > 1) __builtin_amdgcn_sched_barrier(0);  // one group's registers at a time
        }
    };
    // one body for every step: the last one asks for its own inputs again
    const int IT = (KT + KS - 1) / KS;
    for (int it = 0; it < IT; ++it) step(it, smem + (it & 1) * kI4GemmStage, smem + (~it & 1) * kI4GemmStage);
    wait_vm<0>();
    __syncthreads();
    take_off((IT - 1) * GP / kSums * kSums);
    if constexpr (KS > 1) {
        // the other parts' totals, to the first, which adds them in order
        f32x4_t *const parts = reinterpret_cast<f32x4_t *>(smem_all) + wave * (4 * RT * 64) + lane;
        if (part) {
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int m = 0; m < 4; ++m) parts[((part - 1) * 16 * RT + 4 * i + m) * 64] = tot[i][m];
        }
        __syncthreads();
        if (!part) {
#pragma unroll
            for (int k = 0; k < KS - 1; ++k)
#pragma unroll
                for (int i = 0; i < RT; ++i)
#pragma unroll
                    for (int m = 0; m < 4; ++m) tot[i][m] += parts[(k * 16 * RT + 4 * i + m) * 64];
        }
    }

    // ---- a lane holds token r of each tile and rows 4 g .. + 3 of each row tile: through
    // LDS, out in whole-row 16-byte stores
    __syncthreads();
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        if (KS > 1 && part) break;
        float bias[4];
        i4_bias(p, n0 + 16 * (RT * wave + i) + 4 * g, bias);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const f32x4_t v = tot[i][m];
            *reinterpret_cast<uint2 *>(smem_all + (16 * m + r) * kOut + (16 * (RT * wave + i) + 4 * g) * 2) =
                make_uint2(f2bf2_hw(v[0] + bias[0], v[1] + bias[1]), f2bf2_hw(v[2] + bias[2], v[3] + bias[3]));
        }
    }
    __syncthreads();
    const int rows = min(kI4GemmM, p.T - t0), cols = min(kN, p.N - n0);
    uint16_t *const y = p.y + (size_t)t0 * p.N + n0;
    // neighbouring lanes beside one another, as wide as every row's start allows
    auto put = [&](auto piece) {
        using Piece = decltype(piece);
        constexpr int PW = sizeof(Piece) / 2, PR = kN / PW;  // values of a piece, pieces of a row
        for (int c = tid; c < rows * PR; c += 256 * KS) {
            const int row = c / PR, col = c % PR * PW;
            if (col >= cols) continue;
            const Piece v = *reinterpret_cast<const Piece *>(smem_all + row * kOut + col * 2);
            if constexpr (PW == 8) st_through(y + (size_t)row * p.N + col, v);
            else *reinterpret_cast<Piece *>(y + (size_t)row * p.N + col) = v;
        }
    };
    if (p.piece == 8) put(uint4{});
    else if (p.piece == 2) put(uint32_t{});
    else put(uint16_t{});
}

template <int G, bool ZEROS, bool FP16, int RT, int KS>
static void i4_gemm_run(const I4Linear &a, hipStream_t s) {
    const int TB = (a.T + kI4GemmM - 1) / kI4GemmM, NB = (a.N + 64 * RT - 1) / (64 * RT);
    // the tokens in `cut` parts and the rows in 8 / cut: by the rounds of the XCD with most
    // tiles (two workgroups a CU at a time, three of RT = 2, one where parts share the K axis), then by the bytes
    // of x and of W that one reads (T = 300, N = 2816, K = 2048 in two parts 12.4 us, by the bytes
    // alone 22.0)
    int cut = 1;
    constexpr int per_xcd = KS > 1 ? 32 : RT == 2 ? 96 : 64;
    auto rounds = [&](int c) { return ((int64_t)((TB + c - 1) / c) * ((NB * c + 7) / 8) + per_xcd - 1) / per_xcd; };
    auto read = [&](int c) { return 2.0 * a.T / c + 0.55 * a.N * c / 8; };
    for (int c : {2, 4, 8})
        if (c <= TB && (rounds(c) < rounds(cut) || (rounds(c) == rounds(cut) && read(c) < read(cut)))) cut = c;
    const int per_t = (TB + cut - 1) / cut, per_n = (NB * cut + 7) / 8;
    i4_gemm_kernel<G, ZEROS, FP16, RT, KS><<<(unsigned)(8 * per_t * per_n), 256 * KS, 0, s>>>(a, cut);
}

template <int G, bool ZEROS, bool FP16, int RT, int MT, int WV, bool KEEP>
static void i4_split_run(const I4Linear &a, hipStream_t s) {
    const int64_t across = ((a.N + 15) / 16 + RT - 1) / RT, down = (a.T + 16 * MT - 1) / (16 * MT);
    i4_split_kernel<G, ZEROS, FP16, RT, MT, WV, KEEP><<<(unsigned)(across * down), 64 * WV, 0, s>>>(a);
}

// The launches, by what pdscope_linear_int4_launch calls them.
enum I4Launch { kI4Rows16 = 1, kI4Split = 2, kI4Tiles64 = 3, kI4Tiles128Halves = 4, kI4Tiles128 = 5, kI4Tiles256 = 6 };

struct I4Plan {
    I4Launch launch;
    int tiles = 0, tokens = 0, waves = 0;  // kI4Split: row tiles of W, tiles of 16 tokens and waves of a workgroup
};

// A launch by token tiles of a workgroup, in the time of one that has a single one, over
// two: workgroups come 256 at a time, and one of MT tiles takes about as long as
// MT + 1.  N = 1024, K = 2048: T = 64 4.6 / 7.1 / 10.6 us for MT = 1 / 2 / 4; N = 4096, K = 2048:
// T = 17 6.1 / 5.7 / 6.7, T = 48 - / 10.0 / 9.8; N = 2048, K = 4096: T = 32 6.9 / 10.3 / 12.5,
// T = 64 - / 11.1 / 17.9, T = 192 - / 26.6 / 32.5.
static int64_t i4_split_cost(int T, int tiles, int MT) {
    return ((int64_t)tiles * ((T + 16 * MT - 1) / (16 * MT)) + 255) / 256 * (MT + 1);
}

static I4Plan i4_plan(int T, int N, int K, int G) {
    const int KU = (K + kI4In - 1) / kI4In, tiles = (N + kI4Rows - 1) / kI4Rows;
    if (T <= 16) {
        // x in registers where a wave has very many tiles to read with it, and either many rows of x,
        // whose bytes count, or two whole units of it a wave.  us there / in the launch below: N =
        // 151936, K = 2048, G = 128 T = 1 28.4 / 29.0, T = 8 30.7 / 31.9, T = 16 33.5 / 39.7; G = 64 with zero
        // points 33.5 / 34.9, 36.0 / 37.9, 39.0 / 44.2; G = 32 48.5 / 48.4, 49.2 / 52.2, 50.1 / 57.5; K = 1664,
        // G = 64 32.8 / 30.8, 35.0 / 32.9, 37.2 / 39.1; N = 98304, K = 2048, G = 128 20.3 / 20.0, 21.8 / 20.9,
        // 24.0 / 26.4; N = 80000, K = 1664, G = 64 T = 14 22.4 / 21.1.  G = 32 has registers for one
        // workgroup per CU.
        const int64_t units = (int64_t)tiles * KU;
        const int full = kI4RowsWaves * kI4RowsUnits;
        if (KU > 12 && KU <= full && (T > 12 ? units > 98304 : KU == full && units > 131072)) return {kI4Rows16};
        // As many row tiles a workgroup, up to four, as leave one per CU: x is read once for all
        // of them, and each has more loads on its way.  G = 128, K = 4096, one / two / four: N = 4096
        // 5.6 / 6.6 / 8.8 us, N = 8192 8.3 / 7.7 / 9.6, N = 16384 12.7 / 11.1 / 10.1, N = 151936 90 / 70 / 64;
        // T = 16 7.2 / 7.8 / 9.6, 12.4 / 8.6 / 10.5, 20.2 / 14.1 / 11.3, 162 / 103 / 82.  G = 32: N =
        // 40000 31.4 / 27.9 / 33.5, T = 16 48.6 / 33.3 / 35.3.
        if (G > 32 && tiles > 512) return {kI4Split, 4, 1, 8};
        if (tiles > 256) return {kI4Split, 2, 1, 8};
        // 16 waves where there are few workgroups and little of x (K = 2816, N = 2048, T = 1 4.5 us
        // against 4.7 with eight, K = 8192, N = 4096 8.3 against 9.2; T = 16 5.9 against 5.7)
        return {kI4Split, 1, 1, T <= 4 && KU > 16 ? 16 : 8};
    }
    const int64_t one = i4_split_cost(T, tiles, 1), two = i4_split_cost(T, tiles, 2), four = i4_split_cost(T, tiles, 4);
    // The tiled launch takes the time of about seven such units (K = 2048: N = 4096, T = 64 10.9
    // us against 10.3 split, T = 128 11.0 and 17.8; N = 16384, T = 24 11.1 and 15.7; K = 4096: N =
    // 2048, T = 128 16.6 and 17.3, T = 192 16.8 and 26.6).  With few tiles a step's time is that
    // of its loads, and small ones that share the K axis have fewer steps: N = 4096,
    // K = 2048, tiles of 64 tokens x 64 rows in four parts / in two / x 128 in two / x 256: T = 256 11.1 / 12.0
    // / 15.6 / 24.7 us, T = 512 - / 22.4 / 15.7 / 24.6, T = 1024 - / 42 / 29 / 25.5, T = 2048 - / 83 / 57 /
    // 37 to 38; K = 4096, N = 2048, T = 512 16.9 / 19.4 / 24.9 / 44.6.  Tiles of 128 rows without
    // parts go by up to three a CU, those of 256 by two; a round of 256 of the former counts as 10, one
    // of 256 of the latter as 24, of 512 as 34 (against 256 rows, G = 128 / 32: T = 640 23.5 / 33.6 us
    // and 24.8 / 38.2, T = 1300 32.3 / 45.0 and 36.0 / 55.0, T = 1600 42.7 / 58.4 and 35.9 / 55.7, N = 4097,
    // T = 2048 57.6 / 74.9 and 64.8 / 91.7).
    if (std::min({one, two, four}) >= 7) {
        const int64_t down = (T + kI4GemmM - 1) / kI4GemmM, narrow = down * ((N + 127) / 128);
        const int64_t n2 = (narrow + 255) / 256, n4 = (down * ((N + 255) / 256) + 255) / 256;
        if (down * ((N + 63) / 64) <= 256) return {kI4Tiles64};
        if (n2 == 1) return {kI4Tiles128Halves};
        if (10 * n2 < 34 * (n4 / 2) + 24 * (n4 % 2)) return {kI4Tiles128};
        return {kI4Tiles256};
    }
    return {kI4Split, 1, one <= two && one <= four ? 1 : two <= four ? 2 : 4, 8};
}

template <int G, bool ZEROS, bool FP16>
static void i4_linear_launch(const I4Linear &a, hipStream_t s) {
    const I4Plan p = i4_plan(a.T, a.N, a.K, G);
    switch (p.launch) {
        case kI4Rows16: {
            const int blocks = std::min((a.N + kI4Rows - 1) / kI4Rows, G == 32 ? 256 : 512);
            i4_rows_kernel<G, ZEROS, FP16><<<(unsigned)blocks, 64 * kI4RowsWaves, 0, s>>>(a);
            return;
        }
        case kI4Tiles64: return i4_gemm_run<G, ZEROS, FP16, 1, 4>(a, s);
        case kI4Tiles128Halves: return i4_gemm_run<G, ZEROS, FP16, 2, 2>(a, s);
        case kI4Tiles128: return i4_gemm_run<G, ZEROS, FP16, 2, 1>(a, s);
        case kI4Tiles256: return i4_gemm_run<G, ZEROS, FP16, 4, 1>(a, s);
        case kI4Split: break;
    }
    if constexpr (G > 32)
        if (p.tiles == 4) return i4_split_run<G, ZEROS, FP16, 4, 1, 8, false>(a, s);
    if (p.tiles == 2) return i4_split_run<G, ZEROS, FP16, 2, 1, 8, false>(a, s);
    if (p.tokens == 4) return i4_split_run<G, ZEROS, FP16, 1, 4, 8, true>(a, s);
    if (p.tokens == 2) return i4_split_run<G, ZEROS, FP16, 1, 2, 8, true>(a, s);
    if (a.T > 16) return i4_split_run<G, ZEROS, FP16, 1, 1, 8, true>(a, s);
    if (p.waves == 16) return i4_split_run<G, ZEROS, FP16, 1, 1, 16, false>(a, s);
    return i4_split_run<G, ZEROS, FP16, 1, 1, 8, false>(a, s);
}

}  // namespace pd

using namespace pd;

PD_API int pdscope_linear_int4(const void *x, const void *w, const void *bias, int T, int N, int K, int G, int zeros,
                               int fp16_scales, void *y, void *stream) {
    if (!x || !w || !y) return fail(kEInval, "linear_int4: null pointer");
    if (!i4_shape_ok(N, K, G) || i4_units(N, K) > ((int64_t)1 << 26) - 4)
        return fail(kEInval, "linear_int4: need 1 <= N <= 2^24, G of 32, 64 or 128 and K % G == 0, K <= 2^20");
    if (T < 1 || T > (1 << 24)) return fail(kEInval, "linear_int4: need 1 <= T <= 2^24");
    for (const void *p : {x, w})
        if (reinterpret_cast<uintptr_t>(p) % 16) return fail(kEInval, "linear_int4: x and w need 16-byte alignment");
    // a launch has fewer than 2^32 threads: 256 a tile of the tiled one, whose rectangles
    // may add 8 tiles a row and a column of them
    if (((int64_t)N + 255) / 256 * (((int64_t)T + kI4GemmM - 1) / kI4GemmM) > (int64_t)1 << 23)
        return fail(kEInval, "linear_int4: too many outputs for one launch");
    const uintptr_t at = reinterpret_cast<uintptr_t>(y);
    const I4Linear a{(const uint8_t *)w, (const uint16_t *)x, (const uint16_t *)bias, (uint16_t *)y, T, N, K,
                     N % 8 == 0 && at % 16 == 0 ? 8 : N % 2 == 0 && at % 4 == 0 ? 2 : 1};
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    auto group = [&](auto g) {
        constexpr int GG = decltype(g)::value;
        if (zeros) fp16_scales ? i4_linear_launch<GG, true, true>(a, s) : i4_linear_launch<GG, true, false>(a, s);
        else fp16_scales ? i4_linear_launch<GG, false, true>(a, s) : i4_linear_launch<GG, false, false>(a, s);
    };
    if (G == 32) group(std::integral_constant<int, 32>{});
    else if (G == 64) group(std::integral_constant<int, 64>{});
    else group(std::integral_constant<int, 128>{});
    return check_launch("linear_int4");
}

PD_API int pdscope_linear_int4_launch(int T, int N, int K, int G) {
    if (!i4_shape_ok(N, K, G) || i4_units(N, K) > ((int64_t)1 << 26) - 4 || T < 1 || T > (1 << 24)) return 0;
    return i4_plan(T, N, K, G).launch;
}
