// Rows into the paged key / value cache and back (the layout and the e4m3 form: paged.h).
//   molly_paged_kv_append : rows of k and v (and q) -> q/k-norm, rotary -> the pages of the cache, bf16 or e4m3
//   molly_paged_kv_read   : the rows of a list of places, back as bf16
#include "common.h"
#include "molly_hip.h"
#include "paged.h"

namespace {

// the exponent byte of a head whose largest finite magnitude is amax (448 = 1.75 * 2^8)
__device__ __forceinline__ int e4m3_exponent(float amax) {
    const unsigned u = __builtin_bit_cast(unsigned, amax);
    const int e = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return min(max(e, 1), 254);
}
// four codes; a value that is not finite becomes the format's NaN (e4m3 has no infinity)
__device__ __forceinline__ unsigned e4m3_pack4(const float* x, float inv) {
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = fabsf(x[i]) < INFINITY ? x[i] * inv : __builtin_nanf("");
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
    return (unsigned)w;
}

struct AppendArgs {
    const bf16_t* q; const bf16_t* k; const bf16_t* v; bf16_t* q_out;
    void* kpool; void* vpool; uint8_t* kscale; uint8_t* vscale;
    const int* slot; const bf16_t* qw; const bf16_t* kw; const float* cos; const float* sin; const int* pos;
    long n_slots;                                    // pages * page size
    int n, nq, nkv, ldq, ldk, ldv, ldqo, page_shift, n_pos;
    float eps;
};

// One block = a run of tokens x HPB heads: the tokens of a prompt lie next to each other in a page, so what the block stores of a head is one contiguous
// run of the pool (and of its exponent bytes), and it reads HPB * HD * 2 contiguous bytes of every row.  A thread owns 8 + 8 elements of a
// head, rotary partners among them, in each of the block's heads: the token's cos / sin and place are fetched once for all of them.
// HD / 16 lanes hold a head.  Bound by HBM: every byte is touched once.
template <int HD, bool FP8, int HPB>
__global__ __launch_bounds__(256) void paged_append_kernel(AppendArgs p) {
    constexpr int LPH = HD / 16, TPB = 256 / LPH, half = HD / 2;
    const int sub = threadIdx.x % LPH;
    const int heads = p.nq + 2 * p.nkv, groups = (heads + HPB - 1) / HPB;
    const int head0 = blockIdx.x % groups * HPB;     // q heads, k heads, v heads
    const int row = blockIdx.x / groups * TPB + threadIdx.x / LPH;
    const bool live = row < p.n;
    const int r = live ? row : p.n - 1;              // (the lanes behind the last row stay: the head's sums are taken over lanes)
    u32x4 a[HPB], b[HPB];
#pragma unroll
    for (int i = 0; i < HPB; ++i) {
        const int head = min(head0 + i, heads - 1);
        const bf16_t* src = head < p.nq ? p.q + (size_t)r * p.ldq + head * HD : head < p.nq + p.nkv ? p.k + (size_t)r * p.ldk + (head - p.nq) * HD
                                        : p.v + (size_t)r * p.ldv + (head - p.nq - p.nkv) * HD;
        a[i] = ld_stream<u32x4>(src + sub * 8);
        b[i] = ld_stream<u32x4>(src + half + sub * 8);
    }
    const long s = live ? p.slot[row] : -1;
    const bool keep = s >= 0 && s < p.n_slots;       // anything else: a row of padding
    const size_t page = (size_t)(s >> p.page_shift) * p.nkv, offset = s & ((1 << p.page_shift) - 1);
    float c[8], t[8];
    if (p.cos && head0 < p.nq + p.nkv) {
        const int pos = p.pos[r];
        const bool known = pos >= 0 && pos < p.n_pos;                 // a position outside the tables: the head is NaN
        const size_t at = (size_t)(known ? pos : 0) * half + sub * 8;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const f32x4 cv = *reinterpret_cast<const f32x4*>(p.cos + at + 4 * g), sv = *reinterpret_cast<const f32x4*>(p.sin + at + 4 * g);
#pragma unroll
            for (int e = 0; e < 4; ++e) { c[4 * g + e] = known ? cv[e] : __builtin_nanf(""); t[4 * g + e] = sv[e]; }
        }
    }
    auto pack8 = [](const float* f) { return u32x4{pack_bf2(f[0], f[1]), pack_bf2(f[2], f[3]), pack_bf2(f[4], f[5]), pack_bf2(f[6], f[7])}; };
#pragma unroll
    for (int i = 0; i < HPB; ++i) {
        const int head = head0 + i;
        if (head >= heads) return;
        const bool isq = head < p.nq, isk = !isq && head < p.nq + p.nkv;
        const int h = isq ? head : isk ? head - p.nq : head - p.nq - p.nkv;
        float x[8], y[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const unsigned ae = a[i][e], be = b[i][e];
            x[2 * e] = bflo(ae); x[2 * e + 1] = bfhi(ae);
            y[2 * e] = bflo(be); y[2 * e + 1] = bfhi(be);
        }
        const bf16_t* w = isq ? p.qw : isk ? p.kw : nullptr;
        if (w) {                                     // (block-uniform) fp32 throughout: the row is rounded once, where it is stored
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) ss += x[e] * x[e] + y[e] * y[e];
#pragma unroll
            for (int o = 1; o < LPH; o <<= 1) ss += __shfl_xor(ss, o, 64);
            const float rstd = rsqrtf(ss * (1.f / HD) + p.eps);
            const u32x4 wa = *reinterpret_cast<const u32x4*>(w + sub * 8), wb = *reinterpret_cast<const u32x4*>(w + half + sub * 8);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const unsigned u = wa[e], v = wb[e];
                x[2 * e] *= rstd * bflo(u); x[2 * e + 1] *= rstd * bfhi(u);
                y[2 * e] *= rstd * bflo(v); y[2 * e + 1] *= rstd * bfhi(v);
            }
        }
        if (p.cos && (isq || isk)) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float x1 = x[e], x2 = y[e];
                x[e] = x1 * c[e] - x2 * t[e];
                y[e] = x2 * c[e] + x1 * t[e];
            }
        }
        if (isq) {
            if (!live) continue;
            bf16_t* d = p.q_out + (size_t)row * p.ldqo + h * HD + sub * 8;
            *reinterpret_cast<u32x4*>(d) = pack8(x);
            *reinterpret_cast<u32x4*>(d + half) = pack8(y);
            continue;
        }
        const size_t key = ((page + h) << p.page_shift) + offset;
        if constexpr (FP8) {
            float m = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float u = fabsf(x[e]), v = fabsf(y[e]);
                m = fmaxf(m, fmaxf(u < INFINITY ? u : 0.f, v < INFINITY ? v : 0.f));
            }
#pragma unroll
            for (int o = 1; o < LPH; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
            const int e = e4m3_exponent(m);
            const float inv = exp2i(127 - e);                          // (e <= 247: m is finite)
            // 16 contiguous codes a lane: even lanes take their and the next lane's lower half, odd lanes the upper ones
            const u32x2 lo = u32x2{e4m3_pack4(x, inv), e4m3_pack4(x + 4, inv)}, hi = u32x2{e4m3_pack4(y, inv), e4m3_pack4(y + 4, inv)};
            const bool odd = sub & 1;
            const unsigned g0 = __shfl_xor(odd ? lo[0] : hi[0], 1, 64), g1 = __shfl_xor(odd ? lo[1] : hi[1], 1, 64);
            if (!keep) continue;
            uint8_t* d = (uint8_t*)(isk ? p.kpool : p.vpool) + key * HD + (odd ? half - 8 : 0) + sub * 8;
            *reinterpret_cast<u32x4*>(d) = odd ? u32x4{g0, g1, hi[0], hi[1]} : u32x4{lo[0], lo[1], g0, g1};
            if (sub == 0) (isk ? p.kscale : p.vscale)[key] = (uint8_t)e;
        } else {
            if (!keep) continue;
            bf16_t* d = (bf16_t*)(isk ? p.kpool : p.vpool) + key * HD + sub * 8;
            *reinterpret_cast<u32x4*>(d) = pack8(x);
            *reinterpret_cast<u32x4*>(d + half) = pack8(y);
        }
    }
}

template <int HD, bool FP8>
void launch_append(hipStream_t st, const AppendArgs& p) {
    const int blocks = cdiv(p.n, 256 / (HD / 16)), heads = p.nq + 2 * p.nkv;
    // Four heads a block, for longer runs of the rows, where that leaves enough blocks to fill the chip (3 a CU): 16,384 rows of 32 + 16 heads of 128 74.9
    // -> 69.7 us (5.1 TB/s), 2,048 12.0 -> 11.4; below it one, whose loads are spread over more of them: 1,536 rows 9.9 -> 9.5, 32 rows 4.6 -> 2.7.
    if ((long)blocks * cdiv(heads, 4) >= 768) hipLaunchKernelGGL((paged_append_kernel<HD, FP8, 4>), dim3(blocks * cdiv(heads, 4)), dim3(256), 0, st, p);
    else hipLaunchKernelGGL((paged_append_kernel<HD, FP8, 1>), dim3(blocks * heads), dim3(256), 0, st, p);
}

struct ReadArgs {
    const void* kpool; const void* vpool; const uint8_t* kscale; const uint8_t* vscale;
    const int* slot; bf16_t* k_out; bf16_t* v_out;
    long n_slots;
    int n, nkv, ldk, ldv, page_shift;
};

// The append's block shape the other way round: a run of places x one head of K or V, 16 elements a thread.
template <int HD, bool FP8>
__global__ __launch_bounds__(256) void paged_read_kernel(ReadArgs p) {
    constexpr int LPH = HD / 16, TPB = 256 / LPH;
    const int sub = threadIdx.x % LPH;
    const int row = blockIdx.x * TPB + threadIdx.x / LPH;
    if (row >= p.n) return;
    const bool isk = (int)blockIdx.y < p.nkv;
    const int h = isk ? blockIdx.y : blockIdx.y - p.nkv;
    const long s = p.slot[row];
    u32x4 a = {0, 0, 0, 0}, b = {0, 0, 0, 0};        // a place outside the pool holds nothing
    if (s >= 0 && s < p.n_slots) {
        const size_t key = (((size_t)(s >> p.page_shift) * p.nkv + h) << p.page_shift) + (s & ((1 << p.page_shift) - 1));
        if constexpr (FP8) {
            const u32x4 c = *reinterpret_cast<const u32x4*>((const uint8_t*)(isk ? p.kpool : p.vpool) + key * HD + sub * 16);
            const float scale = exp2i((int)(isk ? p.kscale : p.vscale)[key] - 127);
            a = e4m3_to_bf8(u32x2{c[0], c[1]}, scale);
            b = e4m3_to_bf8(u32x2{c[2], c[3]}, scale);
        } else {
            const u32x4* c = reinterpret_cast<const u32x4*>((const bf16_t*)(isk ? p.kpool : p.vpool) + key * HD + sub * 16);
            a = c[0]; b = c[1];
        }
    }
    u32x4* d = reinterpret_cast<u32x4*>((isk ? p.k_out + (size_t)row * p.ldk : p.v_out + (size_t)row * p.ldv) + h * HD + sub * 16);
    d[0] = a; d[1] = b;
}

}  // namespace

extern "C" int molly_paged_kv_append(void* stream, const void* k, const void* v, const void* q_or_null, void* q_out_or_null, void* kpool,
                                     void* vpool, void* kscale_or_null, void* vscale_or_null, const int* slot, int n_rows, int n_pages,
                                     int page_size, int n_heads, int n_kv_heads, int head_dim, int ldq, int ldk, int ldv, int ldqo,
                                     const void* q_norm_w, const void* k_norm_w, const float* cos, const float* sin, const int* positions,
                                     int n_pos, float eps) {
    MOLLY_ENTER();
    if (int rc = check_pool("paged_kv_append", kpool, vpool, kscale_or_null, vscale_or_null, n_pages, page_size, n_kv_heads, head_dim)) return rc;
    const int nq = q_or_null ? n_heads : 0;
    MOLLY_CHECK(n_rows >= 0, "paged_kv_append: n_rows=%d", n_rows);
    if (n_rows == 0) return 0;                       // (no rows have no address: nothing else is asked of them)
    MOLLY_CHECK(nq >= 0 && k && v && slot, "paged_kv_append: n_heads=%d; k, v, slot required", n_heads);
    MOLLY_CHECK((q_or_null == nullptr) == (q_out_or_null == nullptr), "paged_kv_append: q and q_out go together");
    MOLLY_CHECK((cos == nullptr) == (sin == nullptr) && (cos == nullptr) == (positions == nullptr) && (cos == nullptr || n_pos > 0),
                "paged_kv_append: cos, sin and positions go together (n_pos=%d)", n_pos);
    MOLLY_CHECK((nq + 2L * n_kv_heads) * ((long)n_rows / 32 + 1) <= 0x7fffffffL, "paged_kv_append: %d rows of %d + 2 * %d heads: more than one call takes",
                n_rows, nq, n_kv_heads);
    MOLLY_CHECK(aligned16(k) && aligned16(v) && ldk % 8 == 0 && ldv % 8 == 0 && ldk >= n_kv_heads * head_dim && ldv >= n_kv_heads * head_dim,
                "paged_kv_append: k / v rows must be 16-byte aligned and hold n_kv_heads * head_dim values (ldk=%d ldv=%d)", ldk, ldv);
    MOLLY_CHECK(nq == 0 || (aligned16(q_or_null) && aligned16(q_out_or_null) && ldq % 8 == 0 && ldqo % 8 == 0 && ldq >= nq * head_dim &&
                            ldqo >= nq * head_dim), "paged_kv_append: q rows must be 16-byte aligned and hold n_heads * head_dim values (ldq=%d ldqo=%d)",
                ldq, ldqo);
    MOLLY_CHECK(aligned16(q_norm_w) && aligned16(k_norm_w) && aligned16(cos) && aligned16(sin), "paged_kv_append: gains / tables must be 16-byte aligned");
    AppendArgs p{};
    p.q = (const bf16_t*)q_or_null; p.k = (const bf16_t*)k; p.v = (const bf16_t*)v; p.q_out = (bf16_t*)q_out_or_null;
    p.kpool = kpool; p.vpool = vpool; p.kscale = (uint8_t*)kscale_or_null; p.vscale = (uint8_t*)vscale_or_null;
    p.slot = slot; p.qw = (const bf16_t*)q_norm_w; p.kw = (const bf16_t*)k_norm_w; p.cos = cos; p.sin = sin; p.pos = positions;
    p.n_slots = (long)n_pages * page_size;
    p.n = n_rows; p.nq = nq; p.nkv = n_kv_heads; p.ldq = ldq; p.ldk = ldk; p.ldv = ldv; p.ldqo = ldqo;
    p.page_shift = log2_exact(page_size); p.n_pos = n_pos; p.eps = eps;
    hipStream_t st = (hipStream_t)stream;
    if (head_dim == 128) {
        if (kscale_or_null) launch_append<128, true>(st, p);
        else launch_append<128, false>(st, p);
    } else {
        if (kscale_or_null) launch_append<64, true>(st, p);
        else launch_append<64, false>(st, p);
    }
    MOLLY_LAUNCH_CHECK();
    return 0;
}

extern "C" int molly_paged_kv_read(void* stream, const void* kpool, const void* vpool, const void* kscale_or_null, const void* vscale_or_null,
                                   const int* slot, int n_rows, int n_pages, int page_size, int n_kv_heads, int head_dim, void* k_out,
                                   void* v_out, int ldk, int ldv) {
    MOLLY_ENTER();
    if (int rc = check_pool("paged_kv_read", kpool, vpool, kscale_or_null, vscale_or_null, n_pages, page_size, n_kv_heads, head_dim)) return rc;
    MOLLY_CHECK(n_rows >= 0, "paged_kv_read: n_rows=%d", n_rows);
    if (n_rows == 0) return 0;
    MOLLY_CHECK(slot && k_out && v_out && 2L * n_kv_heads <= 65535, "paged_kv_read: slot, k_out, v_out required (n_kv_heads=%d)", n_kv_heads);
    MOLLY_CHECK(aligned16(k_out) && aligned16(v_out) && ldk % 8 == 0 && ldv % 8 == 0 && ldk >= n_kv_heads * head_dim && ldv >= n_kv_heads * head_dim,
                "paged_kv_read: output rows must be 16-byte aligned and hold n_kv_heads * head_dim values (ldk=%d ldv=%d)", ldk, ldv);
    ReadArgs p{};
    p.kpool = kpool; p.vpool = vpool; p.kscale = (const uint8_t*)kscale_or_null; p.vscale = (const uint8_t*)vscale_or_null;
    p.slot = slot; p.k_out = (bf16_t*)k_out; p.v_out = (bf16_t*)v_out;
    p.n_slots = (long)n_pages * page_size; p.n = n_rows; p.nkv = n_kv_heads; p.ldk = ldk; p.ldv = ldv; p.page_shift = log2_exact(page_size);
    const dim3 grid(cdiv(n_rows, 256 / (head_dim / 16)), 2 * n_kv_heads);
    hipStream_t st = (hipStream_t)stream;
    if (head_dim == 128) {
        if (kscale_or_null) hipLaunchKernelGGL((paged_read_kernel<128, true>), grid, dim3(256), 0, st, p);
        else hipLaunchKernelGGL((paged_read_kernel<128, false>), grid, dim3(256), 0, st, p);
    } else {
        if (kscale_or_null) hipLaunchKernelGGL((paged_read_kernel<64, true>), grid, dim3(256), 0, st, p);
        else hipLaunchKernelGGL((paged_read_kernel<64, false>), grid, dim3(256), 0, st, p);
    }
    MOLLY_LAUNCH_CHECK();
    return 0;
}
