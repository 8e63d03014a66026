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
#include <algorithm>
#include <type_traits>

#include "mxfp4.h"
#include "topk.h"

namespace pd {

constexpr int kFewMaxT = 16;
constexpr int kFewMaxE = 256;
constexpr int kFewMaxK = 16;
constexpr int kFewMaxH = 4096;
constexpr int kFewChunk = 32;  // I columns of a chunk: one 64-row group of gate/up (I % 128 == 0: an even number of them)

// 16 bytes at a uniform address plus a lane's offset (one scalar pair and one
// register for the address).  4-bit weights, whose loads are whole lines that
// nothing reads again, are not kept in the caches (128 experts of the Qwen
// shape 65.3 us a layer against 73.1); bf16 ones, 64 bytes of a row at a time, are
// (238 us as streamed loads, 224 as these).
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
    const uint16_t *x;
    const int *keys;  // [T, EK] order_key of logit + bias, kNoKey behind E
    int T, H, E, k, normalize, I;
    const uint8_t *const *slots;
    int32_t *ids;
    uint16_t *weights;
    int32_t *row_base;  // [T + 1] first partial row of each token
    float *partial;     // [rows, H]
};

// ---------------------------------------------------------------- router

// An integer in the order of v (-0 is 0).  A NaN comes last, so that a token of NaN
// takes experts 0 .. k-1 (with NaN weights); kNoKey is behind every value.
constexpr int kNoKey = (int)0x80000000, kNanKey = kNoKey + 1;
__device__ __forceinline__ int order_key(float v) {
    const int bits = __float_as_int(v + 0.0f);
    return v == v ? bits ^ ((bits >> 31) & 0x7fffffff) : kNanKey;
}
__device__ __forceinline__ float key_value(int key) {
    return key == kNanKey ? __int_as_float(0x7fc00000) : __int_as_float(key ^ ((key >> 31) & 0x7fffffff));
}

// The same double of lane l ^ 32 / l ^ 16 (in one of the two results; the other
// is the lane's own) and of a lane N further around its row of 16.
__device__ __forceinline__ double sum_swap32(double v) {
    const uint64_t u = __double_as_longlong(v);
    const auto lo = __builtin_amdgcn_permlane32_swap((uint32_t)u, (uint32_t)u, false, false);
    const auto hi = __builtin_amdgcn_permlane32_swap((uint32_t)(u >> 32), (uint32_t)(u >> 32), false, false);
    return __longlong_as_double((uint64_t)hi[0] << 32 | lo[0]) + __longlong_as_double((uint64_t)hi[1] << 32 | lo[1]);
}
__device__ __forceinline__ double sum_swap16(double v) {
    const uint64_t u = __double_as_longlong(v);
    const auto lo = __builtin_amdgcn_permlane16_swap((uint32_t)u, (uint32_t)u, false, false);
    const auto hi = __builtin_amdgcn_permlane16_swap((uint32_t)(u >> 32), (uint32_t)(u >> 32), false, false);
    return __longlong_as_double((uint64_t)hi[0] << 32 | lo[0]) + __longlong_as_double((uint64_t)hi[1] << 32 | lo[1]);
}
template <int CTRL>
__device__ __forceinline__ double sum_ror(double v) {
    const uint64_t u = __double_as_longlong(v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)u, CTRL, 0xf, 0xf, true);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)(u >> 32), CTRL, 0xf, 0xf, true);
    return v + __longlong_as_double((uint64_t)hi << 32 | lo);
}
// Sum over the wave, in every lane (the steps of wave_sum, on doubles).
__device__ __forceinline__ double wave_sum64(double v) {
    v = sum_swap16(sum_swap32(v));
    v = sum_ror<0x124>(sum_ror<0x128>(v));     // row_ror 8, 4
    return sum_ror<0x121>(sum_ror<0x122>(v));  // row_ror 2, 1
}

// Keys of a token lie in rows of EK = E rounded up to four.
__host__ __device__ inline int few_key_row(int E) { return (E + 3) & ~3; }

// One workgroup per expert (and key behind the last) and four tokens.  Products of two bf16 values are
// exact in fp32; the sums are kept in fp64, so the logits are the exactly rounded
// ones (but for a double rounding by way of fp32, as a conversion from fp64 to
// bf16 goes) and the selection does not depend on the order of the sum.  Bound by
// latency: one load of the gate row's piece and of each token's, the sums
// (fp64 runs at the rate of fp32 here), a store.
constexpr int kRouterT = 4;
__global__ __launch_bounds__(256) void few_router_kernel(const uint16_t *__restrict__ x,
                                                         const uint16_t *__restrict__ gate,
                                                         const float *__restrict__ bias, int T, int H, int E,
                                                         uint16_t *__restrict__ logits, int *__restrict__ keys) {
    __shared__ double s_sum[4][kRouterT];
    const int e = blockIdx.x, t0 = blockIdx.y * kRouterT, tid = threadIdx.x, wave = tid >> 6;
    const int nt = min(kRouterT, T - t0), EK = few_key_row(E);  // uniform
    if (e >= E) {
        if (tid < nt) keys[(t0 + tid) * EK + e] = kNoKey;
        return;
    }
    double acc[kRouterT] = {};
    for (int c = tid; c < H / 8; c += 256) {
        const uint4 w = ld_g(gate + (size_t)e * H + 8 * c);
        uint4 v[kRouterT];
#pragma unroll
        for (int q = 0; q < kRouterT; ++q)
            if (q < nt) v[q] = ld_g(x + (size_t)(t0 + q) * H + 8 * c);
#pragma unroll
        for (int q = 0; q < kRouterT; ++q)
            if (q < nt) {
                acc[q] += (double)(lo_bf(v[q].x) * lo_bf(w.x));
                acc[q] += (double)(hi_bf(v[q].x) * hi_bf(w.x));
                acc[q] += (double)(lo_bf(v[q].y) * lo_bf(w.y));
                acc[q] += (double)(hi_bf(v[q].y) * hi_bf(w.y));
                acc[q] += (double)(lo_bf(v[q].z) * lo_bf(w.z));
                acc[q] += (double)(hi_bf(v[q].z) * hi_bf(w.z));
                acc[q] += (double)(lo_bf(v[q].w) * lo_bf(w.w));
                acc[q] += (double)(hi_bf(v[q].w) * hi_bf(w.w));
            }
    }
#pragma unroll
    for (int q = 0; q < kRouterT; ++q)
        if (q < nt) {
            acc[q] = wave_sum64(acc[q]);
            if ((tid & 63) == 0) s_sum[wave][q] = acc[q];
        }
    __syncthreads();
    if (tid < nt) {
        const uint32_t v = f2bf((float)((s_sum[0][tid] + s_sum[1][tid]) + (s_sum[2][tid] + s_sum[3][tid])));
        logits[(t0 + tid) * E + e] = (uint16_t)v;
        keys[(t0 + tid) * EK + e] = order_key(bf2f(v) + (bias ? bias[e] : 0.0f));
    }
}

// ---------------------------------------------------------------- experts

// a / b for 0 <= a < 2^22, 0 < b: the quotient in floats is off by one at most.
__device__ __forceinline__ int small_div(int a, int b) {
    int q = (int)((float)a * __builtin_amdgcn_rcpf((float)b));
    const int rest = a - q * b;
    q += rest >= b;
    return q - (rest < 0);
}

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
// last one (an L2 hit), whose values are not used.  The activations stay in
// registers where they fit beside the sums and the ring, and in LDS above that (XL;
// the shares of the inputs are then summed in two steps, to fit both).  H = 4096, I = 1408, 40 experts touched by 16 tokens: 79 us a layer from
// LDS against 118 from spilled registers over 4-bit experts, 292 against 453 over
// bf16 ones.
template <bool MX, int KQ>
__global__ __launch_bounds__(512) void few_experts_kernel(FewArgs a) {
    constexpr bool XL = KQ >= (MX ? 4 : 3);
    constexpr int kShares = XL ? 4 : 8, kRowX = XL ? KQ * 1024 + 8 : 8;  // row ends 16 bytes further: no bank conflicts
    __shared__ __attribute__((aligned(16))) uint16_t s_x[XL ? kFewMaxT * kRowX : 8];
    __shared__ __attribute__((aligned(16))) float s_part[kShares * 4 * 64 * 4];  // 32 KB; the keys before that
    __shared__ __attribute__((aligned(16))) uint16_t s_h[2 * kFewMaxT * 40];  // h and its rest; rows of 32, 80 bytes apart
    __shared__ int s_id[256], s_first[256], s_mask[256];
    __shared__ float s_w[256];
    __shared__ int s_rows[4];
    __shared__ const uint8_t *s_base[256];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int T = a.T, H = a.H, E = a.E, k = a.k, I = a.I;
    const int r = lane & 15, g = lane >> 4;

    // ---- everything the routing reads, then the tokens' activations as the second
    // operand of every gate/up product (loads complete in order: these are waited
    // for where they are used, behind the routing)
    int *const s_key = reinterpret_cast<int *>(s_part);
    const int EK = few_key_row(E), n_keys = T * EK;
    uint4 key4[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (4 * (tid + 512 * i) < n_keys) key4[i] = ld_g(a.keys + 4 * (tid + 512 * i));
    const uint8_t *slot = tid < E ? a.slots[tid] : nullptr;
    const int KG = H / kGroupIn, HG = H / kGroupRows;
    bf16x8_t xf[XL ? 1 : KQ][4];
    if (XL)
        for (int i = tid; i < T * KQ * 128; i += 512) {
            const int t = i / (KQ * 128), c = i % (KQ * 128);
            *reinterpret_cast<uint4 *>(s_x + t * kRowX + 8 * c) =
                8 * c < H ? ld_g(a.x + (uint32_t)(t * H + 8 * c)) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
    for (int q = 0; q < (XL ? 0 : KQ); ++q)
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) {
            const int kg = wave + 8 * q;
            xf[q][jj] = bf16x8_t{};
            if (kg < KG)
                xf[q][jj] = *reinterpret_cast<const bf16x8_t *>(a.x + (uint32_t)(min(r, T - 1) * H + kg * kGroupIn +
                                                                                 32 * jj + 8 * g));
        }
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (4 * (tid + 512 * i) < n_keys) *reinterpret_cast<uint4 *>(s_key + 4 * (tid + 512 * i)) = key4[i];
    if (tid < 256) {
        s_mask[tid] = 0;
        s_base[tid] = slot;
    }
    __syncthreads();

    // ---- selection, by every workgroup for itself: the k largest keys of a token,
    // equal ones by their expert
    auto picked = [&](int t, int rank, int e) __attribute__((always_inline)) {
        s_id[t * k + rank] = e;
        if (s_base[e]) atomicOr(&s_mask[e], 1 << t);  // the tokens of each expert that has a copy
    };
    if (n_keys <= 512) {
        // A lane (or up to eight neighbouring ones) per token and expert counts the
        // experts ahead of it: no step waits for another.  One token of 128
        // experts: 2.3 thousand cycles from the keys to the picks, against 3.1 by rounds.
        int parts = 1;
        int shift = 0;
        while (parts < 8 && 2 * parts * n_keys <= 512) parts *= 2, ++shift;
        const int pair = min(tid >> shift, n_keys - 1), part = tid & (parts - 1);
        const int t = small_div(pair, EK), e = pair - t * EK;
        const int *row = s_key + t * EK;
        const int mine = row[e];
        // equal keys count where their expert is lower: those of the groups of four
        // before e's own, and of that group the first e % 4
        const int4 own = *reinterpret_cast<const int4 *>(row + (e & ~3));
        int rank = part ? 0 : (own.x == mine && (e & 3) > 0) + (own.y == mine && (e & 3) > 1) +
                                  (own.z == mine && (e & 3) > 2);
#pragma unroll 8
        for (int j = 4 * part; j < EK; j += 4 * parts) {
            const int4 o = *reinterpret_cast<const int4 *>(row + j);
            const int least = mine + (j >= (e & ~3));
            rank += (o.x >= least) + (o.y >= least) + (o.z >= least) + (o.w >= least);
        }
        if (parts > 1) rank += __builtin_amdgcn_mov_dpp(rank, 0xb1, 0xf, 0xf, true);   // lanes ^ 1
        if (parts > 2) rank += __builtin_amdgcn_mov_dpp(rank, 0x4e, 0xf, 0xf, true);   // lanes ^ 2
        if (parts > 4) rank += __builtin_amdgcn_mov_dpp(rank, 0x141, 0xf, 0xf, true);  // lane i with 7 - i
        if (tid < n_keys * parts && part == 0 && rank < k && e < E) picked(t, rank, e);
    } else {
        // a wave per token: the largest of those left, k times
        auto rounds = [&](auto j_c) __attribute__((always_inline)) {
            constexpr int J = decltype(j_c)::value;
            for (int t = wave; t < T; t += 8) {
                int key[J];
#pragma unroll
                for (int j = 0; j < J; ++j) key[j] = 64 * j + lane < E ? s_key[t * EK + 64 * j + lane] : kNoKey;
                int mine = 0;  // lane i: the expert of rank i
                for (int i = 0; i < k; ++i) {
                    int most = key[0];
#pragma unroll
                    for (int j = 1; j < J; ++j) most = max(most, key[j]);
                    most = dpp_max_i32(most);
                    int e = -1;
#pragma unroll
                    for (int j = 0; j < J; ++j) {
                        const uint64_t at = __ballot(key[j] == most);
                        if (e < 0 && at) e = 64 * j + __builtin_ctzll(at);
                    }
#pragma unroll
                    for (int j = 0; j < J; ++j) key[j] = 64 * j + lane == e ? kNoKey : key[j];
                    mine = lane == i ? e : mine;
                }
                if (lane < k) picked(t, lane, mine);
            }
        };
        if (E <= 64) rounds(std::integral_constant<int, 1>{});
        else if (E <= 128) rounds(std::integral_constant<int, 2>{});
        else rounds(std::integral_constant<int, 4>{});
    }
    __syncthreads();
    // The list: these experts in ascending order, as four 64-bit masks that every
    // wave holds.
    uint64_t hits[4];
    int total = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        hits[j] = __ballot(s_mask[64 * j + lane] != 0);
        total += __popcll(hits[j]);
    }
    auto expert_at = [&](int u) __attribute__((always_inline)) {  // the u-th of the list
        int e = 0, before = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int rank = before + __builtin_amdgcn_mbcnt_hi((uint32_t)(hits[j] >> 32),
                                                                __builtin_amdgcn_mbcnt_lo((uint32_t)hits[j], 0));
            const uint64_t at = __ballot((hits[j] >> lane & 1) && rank == u);
            if (at) e = 64 * j + __builtin_ctzll(at);
            before += __popcll(hits[j]);
        }
        return __builtin_amdgcn_readfirstlane(e);
    };
    auto place_of = [&](int e) __attribute__((always_inline)) {  // and the reverse
        int pos = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int below = e - 64 * j;
            pos += __popcll(below >= 64 ? hits[j] : below > 0 ? hits[j] & ((1ull << below) - 1) : 0);
        }
        return pos;
    };
    // n pairs of chunks (ns of them an expert) in G pieces, each for the two
    // workgroups of one XCD that stand next to each other there (block b runs on
    // XCD b % 8): one takes the first chunk of every pair and the other the
    // second, at about the same time, so that the 128-byte lines of the down
    // matrix that hold both (bf16: 64 bytes of a row each) come from HBM once.
    const int ns = I / (2 * kFewChunk), n = __builtin_amdgcn_readfirstlane(total) * ns;
    const int b = blockIdx.x, pairs = gridDim.x / 2, G = min(pairs, n);
    const bool by_xcd = gridDim.x % 16 == 0;
    const int piece = by_xcd ? (b & 7) + 8 * (b >> 4) : b >> 1, second = by_xcd ? b >> 3 & 1 : b & 1;
    // the first `longer` pieces take per + 1 pairs, the others per
    const int per = n >= pairs ? __builtin_amdgcn_readfirstlane(small_div(n, pairs)) : 1, longer = n - per * G;
    auto piece_of = [&](int c) {  // of pair c
        const int in_longer = longer * (per + 1);
        return c < in_longer ? small_div(c, per + 1) : longer + small_div(c - in_longer, per);
    };
    // A partial row for every token, expert of it and workgroup of that expert, in
    // the order of the (token, slot) pairs: s_first counts within 64 pairs, s_rows
    // the 64s.  Read behind the barriers of the first chunk.
    auto count_rows = [&]() __attribute__((always_inline)) {
        if (tid >= 256) return;
        int rows = 0;
        if (tid < T * k && s_mask[s_id[tid]] != 0) {
            const int u = place_of(s_id[tid]);
            rows = 2 * (piece_of((u + 1) * ns - 1) - piece_of(u * ns) + 1);
        }
        int incl = rows;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int v = __shfl_up(incl, d);
            if (lane >= d) incl += v;
        }
        s_first[tid] = incl - rows;
        if (lane == 63) s_rows[wave] = incl;
    };
    auto first_row = [&](int p) __attribute__((always_inline)) {
        int v = s_first[p];
        for (int w = 0; w < p >> 6; ++w) v += s_rows[w];
        return v;
    };
    // One wave per token: the softmax's sum over the chosen experts (or all of
    // them) and the weights of its slots.
    auto weigh = [&]() __attribute__((always_inline)) {
        for (int t = wave; t < T; t += 8) {
            const int *row = s_key + t * EK;
            const float top = key_value(row[s_id[t * k]]);
            const float ex = lane < k ? expf(key_value(row[s_id[t * k + lane]]) - top) : 0.0f;
            float sum = ex;
            if (!a.normalize) {
                sum = 0.0f;
                for (int e = lane; e < E; e += 64) sum += expf(key_value(row[e]) - top);
            }
            const uint16_t w = (uint16_t)f2bf(ex / wave_sum_dpp(sum));
            if (lane < k) {
                s_w[t * k + lane] = bf2f(w);
                if (b == 0) {
                    a.ids[t * k + lane] = s_id[t * k + lane];
                    a.weights[t * k + lane] = w;
                }
            }
        }
    };
    auto write_rows = [&]() __attribute__((always_inline)) {  // for the merge
        if (tid < T) a.row_base[tid] = first_row(tid * k);
        if (tid == T) a.row_base[T] = s_rows[0] + s_rows[1] + s_rows[2] + s_rows[3];
    };
    if (n == 0 && b == 0) {  // no expert has a copy
        weigh();
        count_rows();
        __syncthreads();
        write_rows();
    }
    if (piece >= G) return;
    const int c0 = piece * per + min(piece, longer), c1 = c0 + per + (piece < longer);

    // ---- the weight stream: per chunk NS1 stages of gate/up, then KQ of down, in
    // a ring of R; R divides the stages of a chunk, so that every register is
    // named statically
    constexpr int NS1 = MX ? KQ : 2 * KQ, NS = NS1 + KQ;
    constexpr int R = MX ? (KQ == 1 ? 2 : KQ == 2 ? 4 : KQ == 3 ? 3 : 2) : KQ == 4 ? 2 : 3;
    static_assert(NS % R == 0, "ring");
    FewStage<MX> st[R];
    // a chunk of the list: its expert's block (a uniform address, so that every
    // load is one lane offset from it) and its place in the expert
    struct Chunk {
        const uint8_t *base;
        int e, u, j;  // expert, its place in the list, the chunk's in the expert
    };
    auto block_of = [&](int e) __attribute__((always_inline)) {
        const uint64_t p = reinterpret_cast<uint64_t>(s_base[e]);
        // readfirstlane returns an int: unsigned before it is widened
        const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)p);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(p >> 32));
        return reinterpret_cast<const uint8_t *>((uint64_t)hi << 32 | lo);
    };
    // Offsets in a block (32 bits: the launch refuses larger ones): a lane's part,
    // this wave's groups, and per chunk one product.
    const uint32_t lane16 = lane * 16, row16 = r * 16;
    const uint32_t in_gu = ((uint32_t)r * H + 8 * g) * 2, in_down = ((uint32_t)r * I + 8 * g) * 2;
    const uint32_t gu_chunk = MX ? (uint32_t)KG * kGroupBytes : 64u * H;  // between chunks of gate/up
    const uint32_t down0 = MX ? (uint32_t)mx_gateup_groups(H, I) * kGroupBytes : 4u * I * H;
    const uint32_t down_group = MX ? (uint32_t)(I / kGroupIn) * kGroupBytes : 128u * I;
    auto load = [&](const Chunk &c, int s, FewStage<MX> &d) __attribute__((always_inline)) {
        if (s < NS1) {
            const uint32_t kg = min(wave + 8 * (MX ? s : s >> 1), KG - 1);
            const uint8_t *p = c.base + (c.j * gu_chunk + kg * (MX ? kGroupBytes : 2 * kGroupIn));
            if (MX) {
#pragma unroll
                for (int jj = 0; jj < 4; ++jj) d.v[jj] = ld_stream(p + jj * 1024, lane16);
                d.v[4] = ld_stream(p + kGroupScales, row16);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint8_t *q = p + ((uint32_t)(i >> 1) * I + 16 * (i & 1)) * 2u * H + 128 * (s & 1);
                    d.v[i] = ld_keep(q, in_gu);
                    d.v[4 + i] = ld_keep(q + 64, in_gu);
                }
            }
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t grp = min(wave + 8 * (2 * (s - NS1) + h), HG - 1);
                const uint8_t *p = c.base + (down0 + grp * down_group + (MX ? (c.j >> 2) * kGroupBytes : 64 * c.j));
                if (MX) {
                    d.v[h] = ld_stream(p + (c.j & 3) * 1024, lane16);
                    const uint32_t w = *(const __attribute__((address_space(1))) uint32_t *)((const g_u8_t *)(p + kGroupScales + (c.j & 3) * 4) + row16);
                    if (h == 0) d.v[2].x = w;
                    else d.v[2].y = w;
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) d.v[4 * h + i] = ld_keep(p + (uint32_t)(32 * i) * I, in_down);
                }
            }
        }
    };

    f32x4_t acc2[2 * KQ][4];
#pragma unroll
    for (int q = 0; q < 2 * KQ; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc2[q][i] = f32x4_t{};

    const uint32_t held = wave + 8 * (KQ - 1) < KG ? ~0u : 0u;  // all bits, or none for a last group past the end
    const uint16_t *x_row = s_x + (XL ? min(r, T - 1) * kRowX + wave * kGroupIn + 8 * g : 0);
    auto chunk = [&](const Chunk &c, const Chunk &next, bool more) __attribute__((always_inline)) {
        f32x4_t acc1[4] = {};
        bf16x8_t hf[2] = {};
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            if (s == NS1) {
                // sum the eight waves' shares of the inputs, then SwiGLU: thread
                // (i, lane, q) has gate column 16 i + 4 (lane / 16) + q of token
                // lane % 16, and the same up column two tiles further
                f32x4_t *const share = reinterpret_cast<f32x4_t *>(s_part) + ((wave & (kShares - 1)) * 4 * 64 + lane);
                if (XL) {
                    if (wave >= kShares)
#pragma unroll
                        for (int i = 0; i < 4; ++i) share[64 * i] = acc1[i];
                    __syncthreads();
                    if (wave < kShares)
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc1[i] += share[64 * i];
                }
                if (wave < kShares)
#pragma unroll
                    for (int i = 0; i < 4; ++i) share[64 * i] = acc1[i];
                __syncthreads();
                float gs = 0.0f, us = 0.0f;
#pragma unroll
                for (int w = 0; w < kShares; ++w) {
                    gs += s_part[w * 1024 + tid];
                    us += s_part[w * 1024 + 512 + tid];
                }
                // h as the sum of two bf16 values (off by 2^-16 of it): the matrix cores
                // take bf16, and a second product per weight costs nothing beside
                // the stream, so h adds no rounding that out would show.  The first
                // part is cut off, not rounded, and the second is never 0: both
                // have the sign of h, so an infinite weight's two products are the
                // same infinity (they were opposite ones, or infinity times 0)
                const float h = silu_fast(gs) * us;
                const uint32_t h0 = __float_as_uint(h) >> 16;
                float rest = h - bf2f(h0);
                rest = rest == 0.0f ? bf2f(h0) * 0x1p-24f : rest;
                rest = (h0 & 0x7f80u) == 0x7f80u ? h : rest;  // an infinity or NaN in both
                const int at = ((tid >> 2) & 15) * 40 + (tid >> 8) * 16 + ((tid >> 6) & 3) * 4 + (tid & 3);
                s_h[at] = (uint16_t)h0;
                s_h[kFewMaxT * 40 + at] = (uint16_t)f2bf(rest);
                __syncthreads();
                hf[0] = *reinterpret_cast<const bf16x8_t *>(s_h + r * 40 + 8 * g);
                hf[1] = *reinterpret_cast<const bf16x8_t *>(s_h + kFewMaxT * 40 + r * 40 + 8 * g);
            }
            FewStage<MX> &d = st[s % R];
            auto mfma = [](bf16x8_t w, bf16x8_t v, f32x4_t c) {
                return __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, v, c, 0, 0, 0);
            };
            if (s < NS1) {
                // an input group past the end counts as weights of 0 (4-bit: any code at
                // the smallest scale) against x = 0: an infinite weight of the group that
                // is read in its place would be NaN.  A branch around the products costs
                // the widest bf16 layers 2 to 11% (H = 2560, 16 tokens, 201 us a layer
                // to 223; this 202)
                if ((MX ? s : s >> 1) == KQ - 1) {
#pragma unroll
                    for (int i = MX ? 4 : 0; i < (MX ? 5 : 8); ++i)
                        d.v[i] = make_uint4(d.v[i].x & held, d.v[i].y & held, d.v[i].z & held, d.v[i].w & held);
                }
#pragma unroll
                for (int jj = 0; jj < (MX ? 4 : 2); ++jj) {
                    const int q = MX ? s : s >> 1, piece32 = MX ? jj : 2 * (s & 1) + (jj & 1);
                    const bf16x8_t v = XL ? *reinterpret_cast<const bf16x8_t *>(x_row + q * 8 * kGroupIn + 32 * piece32)
                                          : xf[XL || q >= KQ ? 0 : q][piece32];
                    if (MX) {
                        const uint32_t sw = jj == 0 ? d.v[4].x : jj == 1 ? d.v[4].y : jj == 2 ? d.v[4].z : d.v[4].w;
                        acc1[0] = mfma(mx_decode(d.v[jj].x, mx_scale<0>(sw)), v, acc1[0]);
                        acc1[1] = mfma(mx_decode(d.v[jj].y, mx_scale<1>(sw)), v, acc1[1]);
                        acc1[2] = mfma(mx_decode(d.v[jj].z, mx_scale<2>(sw)), v, acc1[2]);
                        acc1[3] = mfma(mx_decode(d.v[jj].w, mx_scale<3>(sw)), v, acc1[3]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            acc1[i] = mfma(__builtin_bit_cast(bf16x8_t, d.v[4 * jj + i]), v, acc1[i]);
                    }
                }
            } else {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    f32x4_t *o = acc2[2 * (s - NS1) + h];
                    bf16x8_t w[4];
                    if (MX) {
                        const uint32_t sw = h == 0 ? d.v[2].x : d.v[2].y;
                        w[0] = mx_decode(d.v[h].x, mx_scale<0>(sw));
                        w[1] = mx_decode(d.v[h].y, mx_scale<1>(sw));
                        w[2] = mx_decode(d.v[h].z, mx_scale<2>(sw));
                        w[3] = mx_decode(d.v[h].w, mx_scale<3>(sw));
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) w[i] = __builtin_bit_cast(bf16x8_t, d.v[4 * h + i]);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[i] = mfma(w[i], hf[1], mfma(w[i], hf[0], o[i]));
                }
            }
            // the slot is free: the stage R further on, in this chunk or the next
            if (s + R < NS) load(c, s + R, d);
            else if (more) load(next, s + R - NS, d);
        }
    };
    // The sums of a workgroup's columns of one expert leave as one row per token.
    // Where to is looked up (seek) before the last chunk of them is consumed.
    float *row = nullptr;
    float weight = 0.0f;
    auto seek = [&](const Chunk &c) __attribute__((always_inline)) {
        row = nullptr;
        if (s_mask[c.e] >> r & 1) {
            int p = 0;
            for (int i = 0; i < k; ++i) p = s_id[r * k + i] == c.e ? r * k + i : p;
            row = a.partial + (size_t)(first_row(p) + 2 * (piece - piece_of(c.u * ns)) + second) * H + 4 * g;
            weight = s_w[p];
        }
    };
    auto flush = [&]() __attribute__((always_inline)) {
        if (row) {
#pragma unroll
            for (int q = 0; q < 2 * KQ; ++q) {
                const int grp = wave + 8 * q;
                if (grp < HG)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const f32x4_t v = acc2[q][i];
                        *reinterpret_cast<float4 *>(row + grp * 64 + 16 * i) =
                            make_float4(v[0] * weight, v[1] * weight, v[2] * weight, v[3] * weight);
                    }
            }
        }
#pragma unroll
        for (int q = 0; q < 2 * KQ; ++q)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc2[q][i] = f32x4_t{};
    };

    Chunk cur{nullptr, 0, __builtin_amdgcn_readfirstlane(small_div(c0, ns)), 0};
    cur.j = 2 * (c0 - cur.u * ns) + second;
    cur.e = expert_at(cur.u);
    cur.base = block_of(cur.e);
#pragma unroll
    for (int s = 0; s < R; ++s) load(cur, s, st[s]);
    weigh();
    count_rows();
    __syncthreads();
    for (int c = c0; c + 1 < c1; ++c) {
        Chunk next{cur.base, cur.e, cur.u, cur.j + 2};
        if (next.j >= 2 * ns) {
            next = Chunk{nullptr, expert_at(cur.u + 1), cur.u + 1, second};
            next.base = block_of(next.e);
            seek(cur);
        }
        chunk(cur, next, true);
        if (next.u != cur.u) flush();
        cur = next;
    }
    seek(cur);
    chunk(cur, cur, false);
    flush();
    if (b == 0) write_rows();
}

// ---------------------------------------------------------------- merge

// One workgroup per token and 64 columns: 32 quarter-waves take its rows in turn,
// 16 bytes a lane, and are summed in order.  Bound by latency (1.6 MB of rows at
// T = 1, 192 of them).
// out may be add_in (each value is read by the thread that writes it, before it does).
__global__ __launch_bounds__(512) void few_merge_kernel(const float *__restrict__ partial,
                                                        const int32_t *__restrict__ row_base,
                                                        const uint16_t *add_in, int H, uint16_t *out) {
    __shared__ float s_sum[32][65];
    const int t = blockIdx.y, q = threadIdx.x >> 4, l = threadIdx.x & 15;
    const int col = blockIdx.x * 64 + 4 * l;
    const int r0 = row_base[t], r1 = row_base[t + 1];
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    // six rows at a time, the missing ones as zeros: a loop of the compiler's own
    // takes the rows behind a multiple one after the other (T=4 26.7 us a layer
    // against 26.4)
    constexpr int U = 6;
    for (int r = r0 + q; r < r1; r += 32 * U) {
        float4 p[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            p[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (r + 32 * u < r1) p[u] = *reinterpret_cast<const float4 *>(partial + (size_t)(r + 32 * u) * H + col);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            v.x += p[u].x;
            v.y += p[u].y;
            v.z += p[u].z;
            v.w += p[u].w;
        }
    }
    s_sum[q][4 * l] = v.x;
    s_sum[q][4 * l + 1] = v.y;
    s_sum[q][4 * l + 2] = v.z;
    s_sum[q][4 * l + 3] = v.w;
    __syncthreads();
    if (threadIdx.x < 64) {
        const int c = blockIdx.x * 64 + threadIdx.x;
        float s = add_in ? bf2f(add_in[(size_t)t * H + c]) : 0.0f;
#pragma unroll
        for (int w = 0; w < 32; ++w) s += s_sum[w][threadIdx.x];
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

// the workspace: row_base, the keys, the partial rows
constexpr size_t kFewKeysAt = 256, kFewRowsAt = kFewKeysAt + kFewMaxT * kFewMaxE * sizeof(int);

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
    return few_shape_ok(T, H, I, E, k) ? kFewRowsAt + few_rows(T, k, I) * H * sizeof(float) : 0;
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
    cus = std::min(cus, 1024) & ~1;  // an even grid, one workgroup a CU
    if (cus < 2) return fail(kEHip, "moe_few: no compute units");
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    char *ws = (char *)workspace;
    int *keys = (int *)(ws + kFewKeysAt);
    few_router_kernel<<<dim3(few_key_row(E), (T + kRouterT - 1) / kRouterT), 256, 0, s>>>(
        (const uint16_t *)x, (const uint16_t *)gate, bias, T, H, E, (uint16_t *)logits, keys);
    int rc = check_launch("few_router_kernel");
    if (rc) return rc;
    const FewArgs a{(const uint16_t *)x, keys, T, H, E, k, normalize, I, (const uint8_t *const *)slots, ids,
                    (uint16_t *)weights, (int32_t *)ws, (float *)(ws + kFewRowsAt)};
    rc = mxfp4 ? few_launch_experts<true>(a, cus, s) : few_launch_experts<false>(a, cus, s);
    if (rc) return rc;
    few_merge_kernel<<<dim3(H / 64, T), 512, 0, s>>>(a.partial, a.row_base, (const uint16_t *)add_in, H,
                                                             (uint16_t *)out);
    return check_launch("few_merge_kernel");
}
