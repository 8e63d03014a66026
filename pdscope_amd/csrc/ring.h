// Direct-to-LDS loads and the waits of the kernels that stream tiles through LDS
// rings with them.
#pragma once

#include "common.h"

namespace pd {

typedef __attribute__((address_space(3))) void lds_void_t;
typedef __attribute__((address_space(1))) const void g_void_t;

// One wave-wide direct-to-LDS load: lane l's 16 bytes at src land at
// dst + 16 l (dst is wave-uniform), bypassing the registers.  AUX is the
// cache-policy field.  kDeviceScope (sc1) makes the load device-coherent, so
// it is served by the L2 without allocating in the CU's vector L1; kStream
// (nt) marks the lines as not to be kept.  A weight tile is read once per
// m-tile of its expert: where the expert has one m-tile nothing will ask for
// it again, and streaming reads run at 7.0 TB/s against 6.3 and leave the L2
// to the activations; where it has more, the m-tiles read it at about the
// same time and the second should hit the L2.  Chosen per tile, against sc1
// throughout: Qwen shape T=201 gate/up 143 -> 128 us, down 79 -> 71; T=512
// 145 -> 135 and 83 -> 76; T=4096 (about half the experts have two tiles)
// 289 -> 284 and 167 -> 160; DeepSeek-V2-Lite shape T=1304 down 95 -> 82.
// nt throughout: T=512 with Zipf routing 159 against 148, T=4096 301.
// Streamed lines are not kept in the Infinity Cache either, so a pass whose
// weights all fit there (256 MB) and that is repeated at once is the one that
// loses: 16 experts of the Qwen shape, gate/up again and again, 19.8 us under
// sc1 and 28.8 here (32.3 and 29.3 when other experts come in between; weights
// just copied from the host 34.3 and 29.7, 4 experts); one layer of T=2 57.0
// and 59.5, two layers in turn 65.0 and 57.3.
// Activation tiles keep the default policy.
constexpr int kDeviceScope = 16;
constexpr int kStream = 2;
template <int AUX = 0>
__device__ __forceinline__ void load_lds16(const uint16_t *src, uint8_t *dst) {
    __builtin_amdgcn_global_load_lds((g_void_t *)(uintptr_t)src, (lds_void_t *)(uint32_t)(uintptr_t)dst, 16, 0, AUX);
}

// Hides a per-lane load offset from loop-invariant code motion, so each
// 64-bit address (uniform base + offset) is formed next to its load instead
// of being hoisted out of the K loop as a live register pair per load.
__device__ __forceinline__ void opaque(uint32_t &v) { asm volatile("" : "+v"(v)); }

// Wait until at most n vector-memory operations of this wave are in flight
// (n is a compile-time constant in every use).
template <int N>
__device__ __forceinline__ void wait_vm() {
    static_assert(N >= 0 && N < 64, "vmcnt range");
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}

// wait_vm<n> for a wave-uniform n in [0, 24] known only at run time
__device__ __forceinline__ void wait_vm_rt(int n) {
#define PD_W(K) else if (n == K) wait_vm<K>();
    if (n <= 0) wait_vm<0>();
    PD_W(1) PD_W(2) PD_W(3) PD_W(4) PD_W(5) PD_W(6) PD_W(7) PD_W(8) PD_W(9) PD_W(10) PD_W(11) PD_W(12)
    PD_W(13) PD_W(14) PD_W(15) PD_W(16) PD_W(17) PD_W(18) PD_W(19) PD_W(20) PD_W(21) PD_W(22) PD_W(23)
    else wait_vm<24>();
#undef PD_W
}

// Workgroup barrier for the LDS ring.  __syncthreads() would also wait for
// every outstanding direct-to-LDS load (its release fence covers them) and
// drain the pipeline; here the caller waits for exactly the stage it needs
// (wait_stage), this wave's LDS reads are complete (lgkmcnt 0) before the
// slot they read can be refilled, and the memory clobber keeps the
// compiler from moving LDS accesses across the barrier.
__device__ __forceinline__ void ring_barrier() {
    // lgkmcnt(0) through the builtin, so the compiler's own wait analysis
    // knows every earlier LDS read has completed here
    __builtin_amdgcn_s_waitcnt(0xc07f);
    asm volatile("s_barrier" ::: "memory");
}

// Wait until the stage to be consumed has landed, `younger` (0 .. S-2)
// later stages of LPW loads each being allowed to stay in flight.
template <int S, int LPW, int Y = S - 2>
__device__ __forceinline__ void wait_stage(int younger) {
    if constexpr (Y <= 0) {
        wait_vm<0>();
    } else {
        if (younger >= Y) {
            wait_vm<Y * LPW>();
            return;
        }
        wait_stage<S, LPW, Y - 1>(younger);
    }
}

}  // namespace pd
