// What the attention kernels (attention.hip, attn_paged.hip) share: the LDS tile image that serves row reads and transposed reads, the fragments of the
// 32x32x16 bf16 MFMA taken from it, and the softmax's small parts.  Orientation: S^T = K Q^T, so a lane owns ONE query column
// (lane & 31) with its keys in registers, and P^T in bf16 is directly the B operand of O^T = V^T P^T.
#pragma once
#include "common.h"

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float RESCALE_THR = 8.0f;   // log2 domain: O/l are rescaled only when the running max grows by more than this
                                      // (the max is deferred); P then stays <= 2^8, far inside bf16/fp32 range

// raw v_exp_f32 (2^x): inputs here are <= RESCALE_THR or -inf; no denormal range handling needed
__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// One LDS image serves row reads (ds_read_b128: tile row on the lane) AND transposed reads (ds_read_b64_tr_b16: tile
// row = contraction index).  The image is SUB-TILED: blocks of 4 rows x 16 columns (128 B, row pitch 32 B),
// block (rowblk, colblk) stored at block index  rowblk*NCB + (colblk ^ (rowblk&1)),  NCB = HD/16, and inside a block the
// two 16-byte halves of a row are swapped when (rowblk>>1)&1.  Consequences:
//  * a transposed read (4 rows x 16 cols per 16-lane group, two adjacent column blocks per half-wave) touches 256
//    CONTIGUOUS bytes -> conflict-free; a b128 row read of 16 rows distinct mod 16 hits 16 distinct 16-B slots ->
//    conflict-free (the two swaps spread the four row-blocks of a lane group over the bank row);
//  * every address is  lane_base + compile-time constant  (the swaps only involve lane bits), so the unrolled reads
//    share a couple of base VGPRs and use DS immediate offsets instead of one hoisted address register each.
template <int HD> __device__ __forceinline__ int img_off(int row, int col) {      // element offset of (row, col..col+3)
    constexpr int NCB = HD / 16;
    const int rowblk = row >> 2, q = row & 3, b0 = rowblk & 1, b1 = (rowblk >> 1) & 1;
    const int colblk = col >> 4, half = (col >> 3) & 1;
    return (rowblk * NCB + (colblk ^ b0)) * 64 + (q * 2 + (half ^ b1)) * 8 + (col & 7);
}

// "this register has arrived": an empty asm that READS v makes hipcc place the wait for v's pending global load HERE.  Used on
// the per-kernel operand fragments (Q, dO, K, V rows, row statistics) right after their loads: left to itself hipcc waits for
// them lazily inside the tile loop with counted `vmcnt(N)` that cannot see the asm-issued LDS-DMA — and those waits would then
// drain the DMA pipeline every tile (it counts only the loads it knows).
template <class T> __device__ __forceinline__ void arrived(const T& v) { asm volatile("" ::"v"(v)); }

// every LDS-DMA piece this wave issued has landed (the barrier behind it publishes the tile to the other waves)
__device__ __forceinline__ void dma_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// row-read fragment: tile[row][16*s + 8*h .. +7]   (row = 32*sub + (lane&31); s is a compile-time constant at call sites)
template <int HD>
__device__ __forceinline__ bf16x8 row_frag(const bf16_t* tile, int row, int s, int h) {
    constexpr int NCB = HD / 16;
    const int rowblk = row >> 2, q = row & 3, b0 = rowblk & 1, b1 = (rowblk >> 1) & 1;
    // colblk = s, half = h:  (s ^ b0) written as (s & ~1) + ((s & 1) ^ b0) so that only the parity term is per-lane
    const int off = (rowblk * NCB + ((s & 1) ^ b0)) * 64 + (q * 2 + (h ^ b1)) * 8 + (s & ~1) * 64;
    return *reinterpret_cast<const bf16x8*>(tile + off);
}

// A operand (row index = column d of the tile, contraction = tile row) of a 32x32x16 MFMA via ds_read_b64_tr_b16:
// returns tile[row0 + 16*sp + perm(j,h)][32*dt + (lane&31)], j = 0..7, perm = the accumulator-as-operand k order
// (16 sp + 8 (j>>2) + 4 h + (j&3)).  row0 must be a multiple of 32.
template <int HD>
__device__ __forceinline__ bf16x8 tr_frag(const bf16_t* tile, int row0, int sp, int dt, int lane) {
    constexpr int NCB = HD / 16;
    const int h = lane >> 5, g1 = (lane >> 4) & 1, gi = lane & 15, gq = gi >> 2, gp = gi & 3;
    // rows 16sp + 4h + gq (+8): rowblk = row0/4 + 4sp + h (+2) -> b0 = h, b1 = 0 (+8: 1); colblk = 2dt + g1, half = gp>>1
    const int base_a = (h * NCB + (g1 ^ h)) * 64 + (gq * 2 + (gp >> 1)) * 8 + (gp & 1) * 4;
    const int base_b = ((h + 2) * NCB + (g1 ^ h)) * 64 + (gq * 2 + ((gp >> 1) ^ 1)) * 8 + (gp & 1) * 4;
    const int cst = ((row0 >> 2) + 4 * sp) * NCB * 64 + dt * 128;
    const bf16x4 va = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) bf16x4*)(tile + base_a + cst));
    const bf16x4 vb = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) bf16x4*)(tile + base_b + cst));
    return bf16x8{va[0], va[1], va[2], va[3], vb[0], vb[1], vb[2], vb[3]};
}

__device__ __forceinline__ bf16x8 acc_to_frag(const f32x16& a, int base) {
    u32x4 w;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = pack_bf2(a[base + 2 * j], a[base + 2 * j + 1]);
    return __builtin_bit_cast(bf16x8, w);
}

// max over the two half-waves' copies of a row statistic without an LDS round trip: after the swap `a` holds the lower half's
// value in both halves and `b` the upper half's.  (asm with two registers: chained on one value the builtin is folded away by
// hipcc — the note in stage_kv; MOLLY_ATTN_XHALF_LDS=1 at compile time restores the ds_bpermute form for an A/B)
__device__ __forceinline__ float xhalf_max(float v) {
#if defined(MOLLY_ATTN_XHALF_LDS) && MOLLY_ATTN_XHALF_LDS
    return fmaxf(v, __shfl_xor(v, 32, 64));
#else
    float a = v, b = v;
    asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b));
    return fmaxf(a, b);
#endif
}

}  // namespace
