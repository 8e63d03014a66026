// y = x W^T + bias over a 4-bit matrix with group scales (int4.h): the attention's
// projections and the vocabulary head of a model whose experts run here, which
// the reference leaves to the model's torch modules
// (benchmarks/pdscope_compare.py:198-212).
//
//   y[t, n] = bf16(sum_groups s[n] * (sum_k q[n, k] x[t, k] - z[n] * sum_k x[t, k]) + bias[n])
//
// The whole numbers q are bf16 exactly, so the products with x are exact and a
// group's two sums are held in fp32; the scale enters once a group, in fp32.
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
};

// What a wave holds of a unit: codes, its rows' scales and zero points (rows 4 g .. +
// 3, a group each), and the inputs of MT tiles of 16 tokens (token r, inputs 8 g .. + 7
// of each 32).
template <int G, bool ZEROS, bool FP16, int MT>
struct I4Unit {
    static constexpr int GP = kI4In / G, JG = 4 / GP;  // groups of a unit, words of a group
    uint4 c;
    I4Side<G, ZEROS, FP16> side;
    uint4 x[MT][4];

    // KEEP: another workgroup reads the weights too.  Inputs past the end of a row
    // are read as its last ones: their scales are 0.
    template <bool KEEP>
    __device__ __forceinline__ void load(const uint8_t *unit, const uint16_t *const (&xr)[MT], int u, int K, int lane) {
        const int g = lane >> 4;
        c = KEEP ? ld_g(unit + 16 * lane) : ld_nt(unit + 16 * lane);
        side.load(unit, g);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int k = min(u * kI4In + 32 * j + 8 * g, K - 8);
#pragma unroll
            for (int m = 0; m < MT; ++m) x[m][j] = ld_g(xr[m] + k);
        }
    }

    __device__ __forceinline__ void add(f32x4_t (&tot)[MT]) const {
        const __bf16 one = (__bf16)1.0f;
        const bf16x8_t ones = {one, one, one, one, one, one, one, one};
        const uint32_t words[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
        for (int gi = 0; gi < GP; ++gi) {
            f32x4_t acc[MT], sx[MT];
#pragma unroll
            for (int m = 0; m < MT; ++m) acc[m] = sx[m] = f32x4_t{};
#pragma unroll
            for (int j = gi * JG; j < (gi + 1) * JG; ++j) {
                const bf16x8_t w = i4_decode(words[j]);
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    const bf16x8_t v = __builtin_bit_cast(bf16x8_t, x[m][j]);
                    acc[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, v, acc[m], 0, 0, 0);
                    sx[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, v, sx[m], 0, 0, 0);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float sc = side.scale(gi, i), zp = side.zero(gi, i);
#pragma unroll
                for (int m = 0; m < MT; ++m) tot[m][i] = fmaf(sc, fmaf(-zp, sx[m][i], acc[m][i]), tot[m][i]);
            }
        }
    }
};

// Four neighbouring outputs of a token, from row n on.
__device__ __forceinline__ void i4_store(const I4Linear &p, int t, int n, f32x4_t v, const float (&bias)[4]) {
    const uint32_t lo = f2bf2_hw(v[0] + bias[0], v[1] + bias[1]), hi = f2bf2_hw(v[2] + bias[2], v[3] + bias[3]);
    uint16_t *y = p.y + (size_t)t * p.N + n;
    if (n + 3 < p.N && p.N % 4 == 0) {
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

// A workgroup: one tile of 16 rows of W x MT tiles of 16 tokens, the units of the K
// axis dealt to WV waves, whose parts meet in LDS.
template <int G, bool ZEROS, bool FP16, int MT, int WV, bool KEEP>
__global__ __launch_bounds__(64 * WV) void i4_split_kernel(I4Linear p) {
    constexpr int UB = i4_unit_bytes(G, ZEROS);
    __shared__ f32x4_t s_part[WV][MT][64];
    const int lane = lane_id(), ks = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15;
    const int tiles = (p.N + kI4Rows - 1) / kI4Rows, KU = (p.K + kI4In - 1) / kI4In;
    const int tb = blockIdx.x / tiles, n0 = blockIdx.x - tb * tiles;
    const uint8_t *const wt = p.w + (size_t)n0 * KU * UB;
    const uint16_t *xr[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) xr[m] = p.x + (size_t)min((tb * MT + m) * 16 + r, p.T - 1) * p.K;

    f32x4_t tot[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) tot[m] = f32x4_t{};
    for (int u = ks; u < KU; u += WV) {
        I4Unit<G, ZEROS, FP16, MT> d;
        d.template load<KEEP>(wt + (size_t)u * UB, xr, u, p.K, lane);
        d.add(tot);
    }
    // ---- the waves' parts, in order; lane l has token r and rows 4 g .. + 3
#pragma unroll
    for (int m = 0; m < MT; ++m) s_part[ks][m][lane] = tot[m];
    __syncthreads();
    for (int q = threadIdx.x; q < MT * 64; q += 64 * WV) {
        const int m = q >> 6, l = q & 63, t = (tb * MT + m) * 16 + (l & 15), n = n0 * 16 + 4 * (l >> 4);
        if (t >= p.T) continue;
        float bias[4];
        i4_bias(p, n, bias);
        f32x4_t v = s_part[0][m][l];
#pragma unroll
        for (int w = 1; w < WV; ++w) v += s_part[w][m][l];
        i4_store(p, t, n, v, bias);
    }
}

// Up to 16 tokens.  Each of the WV waves keeps U units' worth of x (and its groups'
// sums, which do not depend on the row) in registers and takes these units of
// one row tile after the other, the tiles ahead on their way while it works on one; the
// waves' parts meet in LDS.  ONE: a workgroup has a single tile.
template <int G, bool ZEROS, bool FP16, int WV, int U, bool ONE>
__global__ __launch_bounds__(64 * WV) void i4_rows_kernel(I4Linear p) {
    constexpr int UB = i4_unit_bytes(G, ZEROS), GP = kI4In / G, JG = 4 / GP;
    __shared__ f32x4_t s_part[ONE ? 1 : 2][WV][64];
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
    if (!ONE) load(blockIdx.x + stride, d1);
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
        if (!ONE) load(tile + 2 * stride, ahead);
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
        f32x4_t(&part)[WV][64] = s_part[ONE ? 0 : it & 1];
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
    if (ONE) {
        step(tile, 0, d0, d2);
        return;
    }
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

constexpr int kI4GemmM = 64, kI4GemmN = 256;
constexpr int kI4GemmX = kI4GemmM * 256;           // a stage's x, behind it its scales:
constexpr int kI4GemmStage = kI4GemmX + 4 * 512;  // 128 bytes at most for each of four tiles of four waves
constexpr int kI4GemmSums = 16;                    // groups whose sums of x are kept at a time
constexpr int kI4GemmOut = kI4GemmN * 2 + 16;

// 64 tokens x 256 rows of W, K in steps of 128: a wave has four row tiles to
// itself, whose codes go from memory to registers a step ahead; x streams through two LDS
// stages in 256-byte rows whose 16-byte chunk c lies in slot c ^ (row % 16).
template <int G, bool ZEROS, bool FP16>
__global__ __launch_bounds__(256, 2) void i4_gemm_kernel(I4Linear p, int cut) {
    constexpr int UB = i4_unit_bytes(G, ZEROS), GP = kI4In / G, JG = 4 / GP;
    __shared__ __attribute__((aligned(1024))) uint8_t smem[std::max(2 * kI4GemmStage, kI4GemmM * kI4GemmOut)];
    __shared__ float s_sums[2][kI4GemmSums][kI4GemmM];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, g = lane >> 4;
    const int tiles = (p.N + kI4Rows - 1) / kI4Rows, KT = (p.K + kI4In - 1) / kI4In;
    // the tiles in `cut` x 8 / `cut` rectangles, one per XCD: tokens and rows of W whose
    // sum in bytes is least, for its L2; tokens fastest
    const int TB = (p.T + kI4GemmM - 1) / kI4GemmM, NB = (p.N + kI4GemmN - 1) / kI4GemmN;
    const int xcd = blockIdx.x & 7, pos = blockIdx.x >> 3, per_t = (TB + cut - 1) / cut, per_n = (NB * cut + 7) / 8;
    const int tb = xcd % cut * per_t + pos % per_t, nb = xcd / cut * per_n + pos / per_t;
    if (tb >= TB || nb >= NB) return;
    const int t0 = tb * kI4GemmM, n0 = nb * kI4GemmN;

    const uint8_t *wt[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) wt[i] = p.w + (size_t)min(n0 / 16 + 4 * wave + i, tiles - 1) * KT * UB;
    // x loads: load q of wave w fills rows 16 q + 4 w .. + 3; lane l takes row + l / 16 and
    // the chunk that belongs in its slot
    const uint16_t *xrow[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) xrow[q] = p.x + (size_t)min(t0 + 16 * q + 4 * wave + (lane >> 4), p.T - 1) * p.K;
    const int chunk = (lane & 15) ^ ((4 * wave + (lane >> 4)) & 15);

    // scales: lanes 2 GP i .. + 2 GP - 1 take row tile i's
    const uint8_t *const scales =
        p.w + (size_t)min(n0 / 16 + 4 * wave + min(lane / (2 * GP), 3), tiles - 1) * KT * UB + kI4Codes + lane % (2 * GP) * 16;

    // Loads and reads of different stages go through __restrict__ pointers: the compiler
    // lets no LDS read pass a direct-to-LDS load in flight that may write what it reads.
    auto issue_x = [&](int kt, uint8_t *__restrict__ st) __attribute__((always_inline)) {
        // past the end of a row: its last inputs, whose scales are 0
        const uint32_t at = (uint32_t)min(kt * 16 + chunk, p.K / 8 - 1);
#pragma unroll
        for (int q = 0; q < 4; ++q)
            load_lds16(xrow[q] + (size_t)at * 8, st + (16 * q + 4 * wave) * 256);
        if (lane < 8 * GP) load_lds16(reinterpret_cast<const uint16_t *>(scales + (size_t)kt * UB), st + kI4GemmX + 512 * wave);
    };
    const uint32_t lane16 = 16 * (uint32_t)lane;
    auto issue_w = [&](int kt, u32x4_t (&d)[4]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) d[i] = *gptr(wt[i] + (size_t)kt * UB + lane16);
    };
    u32x4_t ahead[4];
    issue_w(0, ahead);
    issue_x(0, smem);

    f32x4_t tot[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int m = 0; m < 4; ++m) tot[i][m] = f32x4_t{};
    const int groups = p.K / G;
    const __bf16 one = (__bf16)1.0f;
    const bf16x8_t ones = {one, one, one, one, one, one, one, one};

    // What the zero points take off: tot -= sum of (s z)[n] sx[t] over up to 16 groups from
    // q0 on, whose sums of x lie in s_sums: fp32 products of four groups at a time
    auto take_off = [&](int q0) __attribute__((always_inline)) {
        const float *const sums = &s_sums[q0 / kI4GemmSums & 1][0][0];
        // (not unrolled: with more loads at a time their registers are spilled)
#pragma unroll 1
        for (int q = 0; q < kI4GemmSums; q += 4) {
            const int gr = min(q0 + q + g, groups - 1);
            const bool on = q0 + q + g < groups;
            uint32_t sz[4], zz[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint8_t *unit = wt[i] + (size_t)((uint32_t)gr / GP * UB);
                sz[i] = *reinterpret_cast<const uint16_t *>(unit + i4_scale_at(r, gr % GP, GP));
                zz[i] = ZEROS ? unit[i4_zero_at(r, gr % GP, GP)] : 8;
            }
            float b[4];
#pragma unroll
            for (int m = 0; m < 4; ++m) b[m] = on ? sums[(q + g) * kI4GemmM + 16 * m + r] : 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float a = on ? -i4_scale(sz[i], FP16) * (float)zz[i] : 0.0f;
#pragma unroll
                for (int m = 0; m < 4; ++m) tot[i][m] = __builtin_amdgcn_mfma_f32_16x16x4f32(a, b[m], tot[i][m], 0, 0, 0);
            }
        }
    };

    auto step = [&](int kt, const uint8_t *__restrict__ cur, uint8_t *__restrict__ nxt)
        __attribute__((always_inline)) {
        wait_vm<0>();
        ring_barrier();
        if (kt && kt * GP % kI4GemmSums == 0) take_off(kt * GP - kI4GemmSums);
        u32x4_t d[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            d[i] = ahead[i];
            asm volatile("" : "+v"(d[i]));
        }
        issue_x(min(kt + 1, KT - 1), nxt);
        issue_w(min(kt + 1, KT - 1), ahead);
        __builtin_amdgcn_sched_barrier(0);
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
            const int gr = kt * GP + gi;
            // (of every g the same value: a branch round this store has registers spilled)
            s_sums[gr / kI4GemmSums & 1][gr % kI4GemmSums][16 * wave + r] = sx[0];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
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
    for (int kt = 0; kt < KT; ++kt) step(kt, smem + (kt & 1) * kI4GemmStage, smem + (~kt & 1) * kI4GemmStage);
    wait_vm<0>();
    __syncthreads();
    take_off((KT - 1) * GP / kI4GemmSums * kI4GemmSums);

    // ---- a lane holds token r of each tile and rows 4 g .. + 3 of each row tile: through
    // LDS, out in whole-row 16-byte stores
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float bias[4];
        i4_bias(p, n0 + 64 * wave + 16 * i + 4 * g, bias);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const f32x4_t v = tot[i][m];
            *reinterpret_cast<uint2 *>(smem + (16 * m + r) * kI4GemmOut + (64 * wave + 16 * i + 4 * g) * 2) =
                make_uint2(f2bf2_hw(v[0] + bias[0], v[1] + bias[1]), f2bf2_hw(v[2] + bias[2], v[3] + bias[3]));
        }
    }
    __syncthreads();
    const int rows = min(kI4GemmM, p.T - t0), cols = min(kI4GemmN, p.N - n0);
    for (int c = tid; c < rows * (kI4GemmN / 8); c += 256) {
        const int row = c / (kI4GemmN / 8), col = c % (kI4GemmN / 8) * 8;
        const uint8_t *from = smem + row * kI4GemmOut + col * 2;
        uint16_t *to = p.y + (size_t)(t0 + row) * p.N + n0 + col;
        if (col + 8 <= cols && p.N % 8 == 0) {
            st_through(to, *reinterpret_cast<const uint4 *>(from));
        } else {
            for (int i = 0; i < 8 && col + i < cols; ++i) to[i] = reinterpret_cast<const uint16_t *>(from)[i];
        }
    }
}

template <int G, bool ZEROS, bool FP16>
static void i4_gemm_run(const I4Linear &a, hipStream_t s) {
    const int TB = (a.T + kI4GemmM - 1) / kI4GemmM, NB = (a.N + kI4GemmN - 1) / kI4GemmN;
    // bytes of x and of W that an XCD reads, with the tokens in `cut` parts and the rows in 8 / cut
    int cut = 1;
    auto read = [&](int c) { return 2.0 * a.T / c + 0.55 * a.N * c / 8; };
    for (int c : {2, 4, 8})
        if (c <= TB && read(c) < read(cut)) cut = c;
    const int per_t = (TB + cut - 1) / cut, per_n = (NB * cut + 7) / 8;
    i4_gemm_kernel<G, ZEROS, FP16><<<(unsigned)(8 * per_t * per_n), 256, 0, s>>>(a, cut);
}

template <int G, bool ZEROS, bool FP16, int MT, int WV, bool KEEP>
static void i4_split_run(const I4Linear &a, hipStream_t s) {
    const int64_t tiles = (a.N + 15) / 16, down = (a.T + 16 * MT - 1) / (16 * MT);
    i4_split_kernel<G, ZEROS, FP16, MT, WV, KEEP><<<(unsigned)(tiles * down), 64 * WV, 0, s>>>(a);
}

// Whether T rows take the launch for many tokens: from 48 of its 64 x 256 tiles on (N =
// 4096, K = 2048: T = 128 19.4 us split and 31.0 there, T = 192 28 and 31; a tile's time
// is that of its K axis, however few there are).
static bool i4_many(int T, int N) {
    return T > 16 && (int64_t)((T + kI4GemmM - 1) / kI4GemmM) * ((N + kI4GemmN - 1) / kI4GemmN) >= 48;
}

template <int G, bool ZEROS, bool FP16>
static void i4_linear_launch(const I4Linear &a, hipStream_t s) {
    const int KU = (a.K + kI4In - 1) / kI4In, tiles = (a.N + kI4Rows - 1) / kI4Rows;
    if (i4_many(a.T, a.N)) {
        i4_gemm_run<G, ZEROS, FP16>(a, s);
    } else if (a.T > 32) {
        i4_split_run<G, ZEROS, FP16, 4, 8, true>(a, s);
    } else if (a.T > 16) {
        i4_split_run<G, ZEROS, FP16, 2, 8, true>(a, s);
    } else if (KU > 8 && KU <= 16) {
        if (tiles <= 1024) i4_rows_kernel<G, ZEROS, FP16, 8, 2, true><<<(unsigned)tiles, 512, 0, s>>>(a);
        else i4_rows_kernel<G, ZEROS, FP16, 8, 2, false><<<G == 32 ? 256 : 512, 512, 0, s>>>(a);
    } else if (KU > 24 && KU <= 32 && tiles <= 256) {
        i4_rows_kernel<G, ZEROS, FP16, 8, 4, true><<<(unsigned)tiles, 512, 0, s>>>(a);
    } else if (KU > 32 && tiles <= 512) {
        i4_split_run<G, ZEROS, FP16, 1, 16, false>(a, s);
    } else {
        i4_split_run<G, ZEROS, FP16, 1, 8, false>(a, s);
    }
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
    // a launch has fewer than 2^32 threads: at most 1024 for 16 rows of W and 16 of x
    if ((((int64_t)N + 15) / 16) * (((int64_t)T + 15) / 16) > ((int64_t)1 << 22) - 1)
        return fail(kEInval, "linear_int4: too many outputs for one launch");
    const I4Linear a{(const uint8_t *)w, (const uint16_t *)x, (const uint16_t *)bias, (uint16_t *)y, T, N, K};
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
