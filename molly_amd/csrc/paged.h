// The paged key / value cache of `generate`: its layout, its e4m3 form, and what its entry points (paged.hip, attn_paged.hip) ask of one.
// The reference's `generate` keeps HF's DynamicCache (reference src/model/omics_one.py:220-232), one dense tensor a layer that is
// concatenated to at every step; here a layer's cache is a pool of pages [n_pages][n_kv_heads][page_size][head_dim], and a sequence is a
// row of page ids.  Head-major: the keys of one (page, head) are contiguous, so what one workgroup of the attention reads are
// whole lines, page_size * head_dim values at a time.
//
// e4m3 pools: a head of a token is held as codes and ONE exponent byte e in 1 .. 247: value = code * 2^(e - 127).  e - 127 is the smallest power of two (from
// -126 on) that brings the head's largest finite magnitude to 448 (the format's largest value) or less.  With a power of two the division and the product
// are exact: the only rounding is the code's own (round to nearest even, half a step: 2^-4 of the value), the value read back is
// a bf16 without another rounding for e in 3 .. 246, and one conversion instruction (v_cvt_scalef32_pk_bf16_fp8) makes two of them.  Beyond that bf16 ends before the format
// does: with e 1 and 2 (a head of magnitudes up to 448 * 2^-125 = 1.1e-35) the smallest codes, multiples of 2^-135 and 2^-134, are rounded to nearest even to bf16's subnormals of 2^-133;
// with e 247 (a magnitude above 1.75 * 2^127 = 3.0e38) the code that stands for 2^128 is read back as infinity.  What a
// free scale would gain is nothing above the format's subnormals: a code keeps its 4 significant bits wherever it sits in the 15 octaves.
#pragma once
#include "common.h"

namespace {

__device__ __forceinline__ float exp2i(int e) { return __builtin_bit_cast(float, (unsigned)(e + 127) << 23); }      // 2^e, -126 <= e <= 127

// eight codes -> eight bf16, times the power of two `scale`
__device__ __forceinline__ u32x4 e4m3_to_bf8(u32x2 c, float scale) {
    u32x4 r;
    r[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[0], scale, false));
    r[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[0], scale, true));
    r[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[1], scale, false));
    r[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[1], scale, true));
    return r;
}

// ---- host side
inline int log2_exact(int x) {
    for (int s = 0; s < 31; ++s)
        if (x == 1 << s) return s;
    return -1;
}
inline bool aligned16(const void* p) { return ((uintptr_t)p % 16) == 0; }

// what the three entry points ask of a cache
inline int check_pool(const char* what, const void* kpool, const void* vpool, const void* kscale, const void* vscale, int n_pages, int page_size,
               int n_kv_heads, int head_dim) {
    MOLLY_CHECK(head_dim == 64 || head_dim == 128, "%s: head_dim=%d (built for 64 and 128)", what, head_dim);
    MOLLY_CHECK(n_pages > 0 && n_kv_heads > 0 && page_size >= 16 && page_size <= 256 && log2_exact(page_size) >= 0,
                "%s: n_pages=%d n_kv_heads=%d page_size=%d (a power of two in 16..256)", what, n_pages, n_kv_heads, page_size);
    MOLLY_CHECK((long)n_pages * page_size <= 0x7fffffffL, "%s: %d pages of %d places: places are 32-bit", what, n_pages, page_size);
    MOLLY_CHECK(kpool && vpool && aligned16(kpool) && aligned16(vpool), "%s: the pools must be 16-byte aligned device memory", what);
    MOLLY_CHECK((kscale == nullptr) == (vscale == nullptr), "%s: e4m3 pools have exponents for K and for V", what);
    return 0;
}

}  // namespace
