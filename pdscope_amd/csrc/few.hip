// The whole MoE layer for 1 to 16 tokens: router, top-k, SwiGLU experts and the
// weighted merge, in three launches that a decode step captures once.  Restates
// what decode.hip does for one token (expertbench/adapters/qwen.py:87-90,
// 140-152; pdscope_runtime.py:450-469) for a small batch and for 4-bit experts.
//
//   few_router_kernel   logits[t,e] = bf16(x_t . gate_e), summed in 64 bits
//   few_experts_kernel  top-k; every expert that a token picked, its gate/up and
//                       down halves in one pass over its weights
//   few_merge_kernel    out[t] = bf16(add_in[t] + sum of the token's partial rows)
//
// A batch this small is bound by the bytes of the touched experts' weights, so
// the experts' kernel is a stream: the touched experts' I columns, in chunks of
// 32, are one list that is cut into equal contiguous pieces, one per CU.  For
// a chunk a workgroup reads the 32 gate, 32 up and 32 down columns' weights, so
// h never leaves the CU, and no workgroup waits for another.  What that costs
// is that a piece holds a partial sum over its columns of every output of its
// tokens, which goes to memory in fp32 (a row per token, expert and piece:
// 1.6 MB against 21 MB of 4-bit weights at T = 1) and is summed in a fixed order
// by the merge.
#include "mxfp4.h"
#include "topk.h"

namespace pd {

constexpr int kFewMaxT = 16;
constexpr int kFewMaxE = 256;
constexpr int kFewMaxK = 16;
constexpr int kFewMaxH = 4096;
constexpr int kFewChunk = 32;  // I columns of a chunk: one 64-row group of gate/up

// 16 bytes at a uniform address plus a lane's offset (one scalar pair and one
// register for the address), not kept in the caches: weights are read once.
typedef __attribute__((address_space(1))) const uint8_t g_u8_t;
__device__ __forceinline__ uint4 ld_stream(const uint8_t *base, uint32_t off) {
    const g_u8_t *p = (const g_u8_t *)base;
    const u32x4_t v = __builtin_nontemporal_load((const g_u32x4_t *)(p + off));
    return make_uint4(v.x, v.y, v.z, v.w);
}
__device__ __forceinline__ uint4 ld_keep(const uint8_t *base, uint32_t off) {
    const u32x4_t v = *(const g_u32x4_t *)((const g_u8_t *)base + off);
    return make_uint4(v.x, v.y, v.z, v.w);
}

struct FewArgs {
    const uint16_t *x, *logits;
    const float *bias;
    int T, H, E, k, normalize, I;
    const uint8_t *const *slots;
    int32_t *ids;
    uint16_t *weights;
    int32_t *row_base;  // [T + 1] first partial row of each token
    float *partial;     // [rows, H]
};

// ---------------------------------------------------------------- router

// One workgroup per expert.  Products of two bf16 values are exact in fp32; the
// sums are kept in fp64, so the logits are the exactly rounded ones (but for a
// double rounding by way of fp32, as a conversion from fp64 to bf16 goes) and the
// selection does not depend on the order of the sum.
__global__ __launch_bounds__(256) void few_router_kernel(const uint16_t *__restrict__ x,
                                                         const uint16_t *__restrict__ gate, int T, int H, int E,
                                                         uint16_t *__restrict__ logits) {
    __shared__ double s_sum[4][kFewMaxT];
    const int e = blockIdx.x, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    double acc[kFewMaxT];
#pragma unroll
    for (int t = 0; t < kFewMaxT; ++t) acc[t] = 0.0;
    for (int c = tid; c < H / 8; c += 256) {
        const uint4 w = ld_g(gate + (size_t)e * H + 8 * c);
#pragma unroll
        for (int t0 = 0; t0 < kFewMaxT; t0 += 4) {
            if (t0 >= T) continue;
            uint4 v[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] = ld_g(x + (size_t)min(t0 + q, T - 1) * H + 8 * c);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                double s = acc[t0 + q];
                s += (double)(lo_bf(v[q].x) * lo_bf(w.x));
                s += (double)(hi_bf(v[q].x) * hi_bf(w.x));
                s += (double)(lo_bf(v[q].y) * lo_bf(w.y));
                s += (double)(hi_bf(v[q].y) * hi_bf(w.y));
                s += (double)(lo_bf(v[q].z) * lo_bf(w.z));
                s += (double)(hi_bf(v[q].z) * hi_bf(w.z));
                s += (double)(lo_bf(v[q].w) * lo_bf(w.w));
                s += (double)(hi_bf(v[q].w) * hi_bf(w.w));
                acc[t0 + q] = s;
            }
        }
    }
#pragma unroll
    for (int t = 0; t < kFewMaxT; ++t) {
        if (t >= T) continue;
#pragma unroll
        for (int d = 32; d; d >>= 1) acc[t] += __shfl_xor(acc[t], d);
        if (lane == 0) s_sum[wave][t] = acc[t];
    }
    __syncthreads();
    if (tid < T)
        logits[(size_t)tid * E + e] =
            (uint16_t)f2bf((float)((s_sum[0][tid] + s_sum[1][tid]) + (s_sum[2][tid] + s_sum[3][tid])));
}

// ---------------------------------------------------------------- experts

// One stage of a wave's weight stream.  4-bit: a 64 x 128 group of gate/up (four
// pieces of codes and their scales) or one 32-input piece of two groups of
// down.  bf16: two of such a group's four 32-input pieces, or the same pieces of
// down.
template <bool MX>
struct FewStage {
    uint4 v[MX ? 5 : 8];
};

// A wave's share of H: KQ groups of 128 inputs (gate/up) and 2 KQ groups of 64
// outputs (down), dealt to the eight waves in turn; groups past the end read the
// last one (an L2 hit) against x = 0, and their outputs are not stored.
template <bool MX, int KQ>
__global__ __launch_bounds__(512) void few_experts_kernel(FewArgs a) {
    __shared__ __attribute__((aligned(16))) float s_part[8 * 4 * 64 * 4];  // 32 KB; the logits before that
    __shared__ __attribute__((aligned(16))) uint16_t s_h[kFewMaxT * 40];   // rows of 32, 80 bytes apart
    __shared__ TopkScratch s_tk[8];
    __shared__ int s_id[256], s_row[256], s_list[256], s_pos[256], s_mask[256];
    __shared__ float s_w[256];
    __shared__ int s_cnt[4], s_seg[4];
    __shared__ const uint8_t *s_base[256];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int T = a.T, H = a.H, E = a.E, k = a.k, I = a.I;
    const int r = lane & 15, g = lane >> 4;

    // ---- the tokens' activations as the second operand of every gate/up product
    const int KG = H / kGroupIn, HG = H / kGroupRows;
    bf16x8_t xf[KQ][4];
#pragma unroll
    for (int q = 0; q < KQ; ++q)
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) {
            const int kg = wave + 8 * q;
            xf[q][jj] = bf16x8_t{};
            if (kg < KG)
                xf[q][jj] = *reinterpret_cast<const bf16x8_t *>(a.x + (size_t)min(r, T - 1) * H + kg * kGroupIn +
                                                                32 * jj + 8 * g);
        }

    // ---- routing, by every workgroup for itself
    for (int i = tid; i < T * E; i += 512) s_part[i] = bf2f(a.logits[i]);
    if (tid < 256) s_mask[tid] = 0;
    __syncthreads();
    for (int t = wave; t < T; t += 8) {
        TopkScratch *sc = s_tk + wave;
        if (E <= 64) topk_token<1>(s_part + t * E, a.bias, E, k, a.normalize, t, nullptr, nullptr, nullptr, sc);
        else if (E <= 128) topk_token<2>(s_part + t * E, a.bias, E, k, a.normalize, t, nullptr, nullptr, nullptr, sc);
        else topk_token<4>(s_part + t * E, a.bias, E, k, a.normalize, t, nullptr, nullptr, nullptr, sc);
        if (lane < k) {
            // a token whose largest logit is not finite has no probabilities
            // (all NaN): it takes experts 0 .. k-1 with NaN weights
            const float p = sc->selp[lane];
            const int id = p == p ? sc->seli[lane] : lane;
            const uint16_t w = sc->selw[lane];
            s_id[t * k + lane] = id;
            s_w[t * k + lane] = bf2f(w);
            if (blockIdx.x == 0) {
                a.ids[t * k + lane] = id;
                a.weights[t * k + lane] = w;
            }
        }
        wave_lds_sync();  // before the next token overwrites the scratch
    }
    __syncthreads();
    // tokens of each expert that has a copy; the list of these experts in order
    if (tid < T * k && a.slots[s_id[tid]]) atomicOr(&s_mask[s_id[tid]], 1 << (tid / k));
    __syncthreads();
    const bool hit = tid < 256 && s_mask[tid] != 0;
    const unsigned long long hits = __ballot(hit);
    if (tid < 256 && lane == 0) s_cnt[wave] = __popcll(hits);
    __syncthreads();
    if (hit) {
        int pos = __popcll(hits & ((1ull << lane) - 1));
        for (int w = 0; w < wave; ++w) pos += s_cnt[w];
        s_list[pos] = tid;
        s_pos[tid] = pos;
        s_base[pos] = a.slots[tid];
    }
    __syncthreads();
    const int ns = I / kFewChunk;
    const int n = __builtin_amdgcn_readfirstlane(s_cnt[0] + s_cnt[1] + s_cnt[2] + s_cnt[3]) * ns;
    const int G = min((int)gridDim.x, n);  // pieces: every one has a chunk
    // piece b takes chunks [b n / G, (b + 1) n / G); the piece of chunk c:
    auto piece_of = [&](int c) { return (int)(((int64_t)(c + 1) * G - 1) / n); };
    // a partial row for every token, expert of it and piece of that expert, in
    // the order of the (token, slot) pairs
    int rows = 0;
    if (tid < T * k && (s_mask[s_id[tid]] != 0)) {
        const int u = s_pos[s_id[tid]];
        rows = piece_of((u + 1) * ns - 1) - piece_of(u * ns) + 1;
    }
    int incl = rows;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int v = __shfl_up(incl, d);
        if (lane >= d) incl += v;
    }
    if (tid < 256 && lane == 63) s_seg[wave] = incl;
    __syncthreads();
    if (tid < 256) {
        int first = incl - rows;
        for (int w = 0; w < wave; ++w) first += s_seg[w];
        s_row[tid] = first;
        if (blockIdx.x == 0) {
            if (tid < T * k && tid % k == 0) a.row_base[tid / k] = first;
            if (tid == T * k - 1) a.row_base[T] = first + rows;
        }
    }
    __syncthreads();
    if ((int)blockIdx.x >= G) return;
    const int c0 = (int)((int64_t)blockIdx.x * n / G), c1 = (int)((int64_t)(blockIdx.x + 1) * n / G);

    // ---- the weight stream: per chunk NS1 stages of gate/up, then KQ of down, in
    // a ring of R; R divides the stages of a chunk, so that every register is
    // named statically
    constexpr int NS1 = MX ? KQ : 2 * KQ, NS = NS1 + KQ;
    constexpr int R = MX ? (KQ == 1 ? 2 : KQ == 2 ? 4 : KQ == 3 ? 3 : 4) : 3;
    static_assert(NS % R == 0, "ring");
    FewStage<MX> st[R];
    // a chunk of the list: its expert's block (a uniform address, so that every
    // load is one lane offset from it) and its place in the expert
    struct Chunk {
        const uint8_t *base;
        int u, j;
    };
    auto block_of = [&](int u) __attribute__((always_inline)) {
        const uint64_t p = reinterpret_cast<uint64_t>(s_base[u]);
        // readfirstlane returns an int: unsigned before it is widened
        const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)p);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(p >> 32));
        return reinterpret_cast<const uint8_t *>((uint64_t)hi << 32 | lo);
    };
    const uint32_t lane16 = lane * 16, row16 = r * 16;
    const uint32_t in_gu = ((uint32_t)r * H + 8 * g) * 2, in_down = ((uint32_t)r * I + 8 * g) * 2;
    auto load = [&](const Chunk &c, int s, FewStage<MX> &d) __attribute__((always_inline)) {
        if (MX) {
            if (s < NS1) {
                const uint8_t *p = c.base + ((size_t)c.j * KG + min(wave + 8 * s, KG - 1)) * kGroupBytes;
#pragma unroll
                for (int jj = 0; jj < 4; ++jj) d.v[jj] = ld_stream(p + jj * 1024, lane16);
                d.v[4] = ld_stream(p + kGroupScales, row16);
            } else {
                const uint8_t *down = c.base + mx_gateup_groups(H, I) * kGroupBytes;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int grp = min(wave + 8 * (2 * (s - NS1) + h), HG - 1);
                    const uint8_t *p = down + ((size_t)grp * (I / kGroupIn) + (c.j >> 2)) * kGroupBytes;
                    d.v[h] = ld_stream(p + (c.j & 3) * 1024, lane16);
                    const uint32_t w = *(const __attribute__((address_space(1))) uint32_t *)((const g_u8_t *)(p + kGroupScales + (c.j & 3) * 4) + row16);
                    if (h == 0) d.v[2].x = w;
                    else d.v[2].y = w;
                }
            }
        } else {
            if (s < NS1) {
                const uint8_t *p = c.base + ((size_t)32 * c.j * H + min(wave + 8 * (s >> 1), KG - 1) * kGroupIn) * 2;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        d.v[4 * h + i] = ld_stream(p + ((size_t)((i >> 1) * I + 16 * (i & 1)) * H + 32 * (2 * (s & 1) + h)) * 2, in_gu);
            } else {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int grp = min(wave + 8 * (2 * (s - NS1) + h), HG - 1);
                    const uint8_t *p = c.base + ((size_t)2 * I * H + (size_t)grp * 64 * I + 32 * c.j) * 2;
#pragma unroll
                    for (int i = 0; i < 4; ++i) d.v[4 * h + i] = ld_keep(p + (size_t)32 * i * I, in_down);
                }
            }
        }
    };

    f32x4_t acc2[2 * KQ][4];
#pragma unroll
    for (int q = 0; q < 2 * KQ; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc2[q][i] = f32x4_t{};

    auto chunk = [&](const Chunk &c, const Chunk &next, bool more) __attribute__((always_inline)) {
        f32x4_t acc1[4] = {};
        bf16x8_t hf = {};
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            if (s == NS1) {
                // sum the eight waves' shares of the inputs, then SwiGLU: thread
                // (i, lane, q) has gate column 16 i + 4 (lane / 16) + q of token
                // lane % 16, and the same up column two tiles further
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<f32x4_t *>(s_part + ((wave * 4 + i) * 64 + lane) * 4) = acc1[i];
                __syncthreads();
                float gs = 0.0f, us = 0.0f;
#pragma unroll
                for (int w = 0; w < 8; ++w) {
                    gs += s_part[w * 1024 + tid];
                    us += s_part[w * 1024 + 512 + tid];
                }
                // h is rounded to bf16, the matrix cores' input
                s_h[((tid >> 2) & 15) * 40 + (tid >> 8) * 16 + ((tid >> 6) & 3) * 4 + (tid & 3)] =
                    (uint16_t)f2bf(silu_fast(gs) * us);
                __syncthreads();
                hf = *reinterpret_cast<const bf16x8_t *>(s_h + r * 40 + 8 * g);
            }
            FewStage<MX> &d = st[s % R];
            if (MX) {
                if (s < NS1) {
#pragma unroll
                    for (int jj = 0; jj < 4; ++jj) {
                        const uint32_t sw = jj == 0 ? d.v[4].x : jj == 1 ? d.v[4].y : jj == 2 ? d.v[4].z : d.v[4].w;
                        acc1[0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(mx_decode(d.v[jj].x, mx_scale<0>(sw)), xf[s < NS1 ? s : 0][jj], acc1[0], 0, 0, 0);
                        acc1[1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(mx_decode(d.v[jj].y, mx_scale<1>(sw)), xf[s < NS1 ? s : 0][jj], acc1[1], 0, 0, 0);
                        acc1[2] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(mx_decode(d.v[jj].z, mx_scale<2>(sw)), xf[s < NS1 ? s : 0][jj], acc1[2], 0, 0, 0);
                        acc1[3] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(mx_decode(d.v[jj].w, mx_scale<3>(sw)), xf[s < NS1 ? s : 0][jj], acc1[3], 0, 0, 0);
                    }
                } else {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        f32x4_t *o = acc2[2 * (s - NS1) + h];
                        const uint32_t sw = h == 0 ? d.v[2].x : d.v[2].y;
                        o[0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(mx_decode(d.v[h].x, mx_scale<0>(sw)), hf, o[0], 0, 0, 0);
                        o[1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(mx_decode(d.v[h].y, mx_scale<1>(sw)), hf, o[1], 0, 0, 0);
                        o[2] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(mx_decode(d.v[h].z, mx_scale<2>(sw)), hf, o[2], 0, 0, 0);
                        o[3] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(mx_decode(d.v[h].w, mx_scale<3>(sw)), hf, o[3], 0, 0, 0);
                    }
                }
            } else {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const bf16x8_t w = __builtin_bit_cast(bf16x8_t, d.v[4 * h + i]);
                        if (s < NS1)
                            acc1[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, xf[s < NS1 ? s >> 1 : 0][2 * (s & 1) + h], acc1[i], 0, 0, 0);
                        else
                            acc2[2 * (s - NS1) + h][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, hf, acc2[2 * (s - NS1) + h][i], 0, 0, 0);
                    }
            }
            // the slot is free: the stage R further on, in this chunk or the next
            if (s + R < NS) load(c, s + R, d);
            else if (more) load(next, s + R - NS, d);
        }
    };
    // the sums of a piece's columns of one expert leave as one row per token
    auto flush = [&](int u) __attribute__((always_inline)) {
        const int e = s_list[u], seg = (int)blockIdx.x - piece_of(u * ns);
        if (s_mask[e] >> r & 1) {
            int p = r * k;
            while (s_id[p] != e) ++p;
            float *row = a.partial + (size_t)(s_row[p] + seg) * H;
            const float w = s_w[p];
#pragma unroll
            for (int q = 0; q < 2 * KQ; ++q) {
                const int grp = wave + 8 * q;
                if (grp < HG)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const f32x4_t v = acc2[q][i];
                        *reinterpret_cast<float4 *>(row + grp * 64 + 16 * i + 4 * g) =
                            make_float4(v[0] * w, v[1] * w, v[2] * w, v[3] * w);
                    }
            }
        }
#pragma unroll
        for (int q = 0; q < 2 * KQ; ++q)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc2[q][i] = f32x4_t{};
    };

    Chunk cur{nullptr, c0 / ns, c0 % ns};
    cur.base = block_of(cur.u);
#pragma unroll
    for (int s = 0; s < R; ++s) load(cur, s, st[s]);
    for (int c = c0; c + 1 < c1; ++c) {
        Chunk next{cur.base, cur.u, cur.j + 1};
        if (next.j == ns) next = Chunk{block_of(cur.u + 1), cur.u + 1, 0};
        chunk(cur, next, true);
        if (next.u != cur.u) flush(cur.u);
        cur = next;
    }
    chunk(cur, cur, false);
    flush(cur.u);
}

// ---------------------------------------------------------------- merge

// One workgroup per token and 256 columns; eight waves take its rows in turn.
__global__ __launch_bounds__(512) void few_merge_kernel(const float *__restrict__ partial,
                                                        const int32_t *__restrict__ row_base,
                                                        const uint16_t *__restrict__ add_in, int H,
                                                        uint16_t *__restrict__ out) {
    __shared__ __attribute__((aligned(16))) float s_sum[8][256];
    const int t = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = blockIdx.x * 256 + 4 * lane;
    const int r0 = row_base[t], r1 = row_base[t + 1];
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (col < H) {
#pragma unroll 4
        for (int r = r0 + wave; r < r1; r += 8) {
            const float4 p = *reinterpret_cast<const float4 *>(partial + (size_t)r * H + col);
            v.x += p.x;
            v.y += p.y;
            v.z += p.z;
            v.w += p.w;
        }
    }
    *reinterpret_cast<float4 *>(&s_sum[wave][4 * lane]) = v;
    __syncthreads();
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (threadIdx.x < 256 && c < H) {
        float s = add_in ? bf2f(add_in[(size_t)t * H + c]) : 0.0f;
#pragma unroll
        for (int w = 0; w < 8; ++w) s += s_sum[w][threadIdx.x];
        out[(size_t)t * H + c] = (uint16_t)f2bf(s);
    }
}

// ---------------------------------------------------------------- launch

static bool few_shape_ok(int T, int H, int I, int E, int k) {
    return T >= 1 && T <= kFewMaxT && H <= kFewMaxH && I <= 65536 && mx_shape_ok(H, I) && E >= 1 && E <= kFewMaxE &&
           k >= 1 && k <= kFewMaxK && k <= E;
}

// the partial rows: of each (token, slot) pair at most one per chunk
static size_t few_rows(int T, int k, int I) { return (size_t)T * k * (I / kFewChunk); }

template <bool MX>
static int few_launch_experts(const FewArgs &a, int cus, hipStream_t s) {
    switch ((a.H / kGroupIn + 7) / 8) {
    case 1: few_experts_kernel<MX, 1><<<cus, 512, 0, s>>>(a); break;
    case 2: few_experts_kernel<MX, 2><<<cus, 512, 0, s>>>(a); break;
    case 3: few_experts_kernel<MX, 3><<<cus, 512, 0, s>>>(a); break;
    default: few_experts_kernel<MX, 4><<<cus, 512, 0, s>>>(a); break;
    }
    return check_launch("few_experts_kernel");
}

}  // namespace pd

using namespace pd;

PD_API int pdscope_moe_few_supported(int T, int H, int I, int E, int k) { return few_shape_ok(T, H, I, E, k); }

PD_API size_t pdscope_moe_few_workspace_size(int T, int H, int I, int E, int k) {
    return few_shape_ok(T, H, I, E, k) ? 256 + few_rows(T, k, I) * H * sizeof(float) : 0;
}

PD_API int pdscope_moe_few(const void *x, const void *gate, const float *bias, int T, int H, int E, int k,
                           int normalize, const void *const *slots, int mxfp4, int I, const void *add_in, void *logits,
                           int32_t *ids, void *weights, void *out, void *workspace, void *stream) {
    if (!x || !gate || !slots || !logits || !ids || !weights || !out || !workspace)
        return fail(kEInval, "moe_few: null pointer");
    if (!few_shape_ok(T, H, I, E, k))
        return fail(kEInval, "moe_few: need 1 <= T <= 16, H % 128 == 0, H <= 4096, I % 128 == 0, 1 <= k <= min(E, 16), "
                             "E <= 256");
    for (const void *p : {x, gate, (const void *)workspace})
        if (reinterpret_cast<uintptr_t>(p) % 16) return fail(kEInval, "moe_few: x, gate and workspace need 16-byte alignment");
    int dev = 0, cus = 0;
    hipError_t err = hipGetDevice(&dev);
    if (err == hipSuccess) err = hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev);
    if (err != hipSuccess) return fail(kEHip, std::string("moe_few: ") + hipGetErrorString(err));
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    few_router_kernel<<<E, 256, 0, s>>>((const uint16_t *)x, (const uint16_t *)gate, T, H, E, (uint16_t *)logits);
    int rc = check_launch("few_router_kernel");
    if (rc) return rc;
    const FewArgs a{(const uint16_t *)x, (const uint16_t *)logits, bias, T, H, E, k, normalize, I,
                    (const uint8_t *const *)slots, ids, (uint16_t *)weights, (int32_t *)workspace,
                    (float *)((char *)workspace + 256)};
    rc = mxfp4 ? few_launch_experts<true>(a, cus, s) : few_launch_experts<false>(a, cus, s);
    if (rc) return rc;
    few_merge_kernel<<<dim3((H + 255) / 256, T), 512, 0, s>>>(a.partial, a.row_base, (const uint16_t *)add_in, H,
                                                             (uint16_t *)out);
    return check_launch("few_merge_kernel");
}
