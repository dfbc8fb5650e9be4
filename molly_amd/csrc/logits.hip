// Logit processors in front of the draw: penalties for repeated tokens, a bias and a mask of allowed tokens, in one pass over the row.
//   c    = how often the token occurs in the row's generated sequence
//   c > 0:  s = (s < 0 ? s * repetition : s / repetition) - presence       (the first as in HF:generation/logits_process.py; the
//   s   -= frequency * c                                                    reference's generate passes repetition_penalty through,
//   s   += bias[token]                                                      src/model/omics_one.py:220-232)
//   s    = -inf where the token's bit of the mask is 0                     (HF's prefix_allowed_tokens_fn / bad_words_ids)
// One workgroup = one row x one slice of the vocabulary: it counts the row's history into LDS (integer atomics: the order changes
// nothing), then makes the slice's pass.  Bound by HBM: the logits are read once and written once; the history comes from L2 once per slice.
#include "common.h"
#include "molly_hip.h"

namespace {

// every workgroup reads the row's whole history: from this many tokens on, four times fewer, larger workgroups do (V = 151,936, one row | 32 rows, 256 -> 1,024
// threads: 1,024 tokens 4.2 -> 4.4 | 8.2 -> 8.6 us, 2,048 5.0 -> 4.9 | 9.4 -> 9.3, 8,192 9.0 -> 6.3 | 18.3 -> 13.2, 32,768 22.6 -> 10.1 | 49.5 -> 22.7)
constexpr int LONG_HISTORY = 2048;

struct LogitArgs {
    const void* x; float* out;
    const long* gen; const int* n_gen;
    const float* rep_v; const float* pres_v; const float* freq_v;       // per row (nullable: the scalars)
    const float* bias; const unsigned* mask;
    float rep, pres, freq;
    int V, n_hist;
    long ldx, ldo, ldg, ldb, ldm;                     // ldb / ldm 0: one row for all
};

// THREADS * 16 tokens a workgroup, four groups of four a thread: 16-byte loads and stores at whatever token the row's first aligned address falls on
// (`shift` tokens of the first group lie in front of the row).  Logits, bias and mask are asked for in front of the
// history's pass and wait in registers.
template <int THREADS, bool BF16, bool HIST>
__global__ __launch_bounds__(THREADS) void logits_kernel(LogitArgs p) {
    constexpr int SLICE = THREADS * 16;
    __shared__ unsigned cnt[HIST ? SLICE : 1];
    const int row = blockIdx.y, t = threadIdx.x;
    const size_t x0 = (size_t)row * p.ldx, o0 = (size_t)row * p.ldo;
    // tokens of the first aligned group that lie in front of the row; where the two rows are aligned differently: one token at a time
    const int sx = (int)((((uintptr_t)p.x >> (BF16 ? 1 : 2)) + x0) & 3), so = (int)((((uintptr_t)p.out >> 2) + o0) & 3);
    const int shift = sx == so ? sx : 0;
    const bool vec = sx == so;
    const int v0 = blockIdx.x * SLICE - shift;       // token of the slice's first place
    if (v0 >= p.V) return;
    const unsigned* m = p.mask ? p.mask + (size_t)row * p.ldm : nullptr;
    const float* bias = p.bias ? p.bias + (size_t)row * p.ldb : nullptr;
    const bool bias_vec = bias && ((uintptr_t)(bias + v0) & 15) == 0;
    float x[4][4];
    f32x4 add[4];
    unsigned wa[4], wb[4];                           // mask words of the group's first and last token
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int v = v0 + (j * THREADS + t) * 4;
        const bool whole = v >= 0 && v + 4 <= p.V;
        if (vec && whole) {
            if constexpr (BF16) {
                const u32x2 w = *reinterpret_cast<const u32x2*>((const bf16_t*)p.x + x0 + v);
                x[j][0] = bflo(w[0]); x[j][1] = bfhi(w[0]); x[j][2] = bflo(w[1]); x[j][3] = bfhi(w[1]);
            } else {
                const f32x4 w = *reinterpret_cast<const f32x4*>((const float*)p.x + x0 + v);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[j][e] = w[e];
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                x[j][e] = v + e < 0 || v + e >= p.V ? 0.f : BF16 ? bf2f(((const bf16_t*)p.x)[x0 + v + e]) : ((const float*)p.x)[x0 + v + e];
        }
        if (bias) {
            if (whole && bias_vec) {
                add[j] = *reinterpret_cast<const f32x4*>(bias + v);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) add[j][e] = v + e >= 0 && v + e < p.V ? bias[v + e] : 0.f;
            }
        }
        if (m && v + 4 > 0 && v < p.V) {
            wa[j] = m[max(v, 0) >> 5];
            wb[j] = m[min(v + 3, p.V - 1) >> 5];
        }
    }
    if constexpr (HIST) {
#pragma unroll
        for (int j = 0; j < 4; ++j) *reinterpret_cast<u32x4*>(cnt + (j * THREADS + t) * 4) = u32x4{0, 0, 0, 0};
        const int n = min(max(p.n_gen ? p.n_gen[row] : p.n_hist, 0), p.n_hist);
        __syncthreads();
        const long* g = p.gen + (size_t)row * p.ldg;
#pragma unroll 4
        for (int i = t; i < n; i += THREADS) {
            const long at = g[i] - v0;
            if (at >= 0 && at < SLICE && g[i] < p.V && g[i] >= 0) atomicAdd(&cnt[(int)at], 1u);
        }
        __syncthreads();
    }
    const float rep = p.rep_v ? p.rep_v[row] : p.rep, pres = p.pres_v ? p.pres_v[row] : p.pres, freq = p.freq_v ? p.freq_v[row] : p.freq;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int v = v0 + (j * THREADS + t) * 4;
        if (v + 4 <= 0 || v >= p.V) continue;
        const bool whole = v >= 0 && v + 4 <= p.V;
        if constexpr (HIST) {
            const u32x4 c = *reinterpret_cast<const u32x4*>(cnt + (j * THREADS + t) * 4);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (c[e]) x[j][e] = (x[j][e] < 0.f ? x[j][e] * rep : x[j][e] / rep) - pres - freq * (float)c[e];
        }
        if (bias)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[j][e] += add[j][e];
        if (m)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const unsigned w = ((v + e) >> 5) == (max(v, 0) >> 5) ? wa[j] : wb[j];
                if (!((w >> ((v + e) & 31)) & 1u)) x[j][e] = -INFINITY;
            }
        float* o = p.out + o0 + v;
        if (vec && whole) {
            *reinterpret_cast<f32x4*>(o) = f32x4{x[j][0], x[j][1], x[j][2], x[j][3]};
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (v + e >= 0 && v + e < p.V) o[e] = x[j][e];
        }
    }
}

template <int THREADS, bool HIST>
void launch(hipStream_t st, const LogitArgs& p, int rows, bool bf16) {
    const dim3 grid(cdiv(p.V + 3L, THREADS * 16), rows);              // (+ 3: a row may start in the middle of its first group)
    if (bf16) hipLaunchKernelGGL((logits_kernel<THREADS, true, HIST>), grid, dim3(THREADS), 0, st, p);
    else hipLaunchKernelGGL((logits_kernel<THREADS, false, HIST>), grid, dim3(THREADS), 0, st, p);
}

}  // namespace

extern "C" int molly_process_logits(void* stream, const void* logits, int logits_bf16, float* out, int rows, int V, long ld_logits, long ld_out,
                                    const int64_t* generated, const int* n_generated_or_null, int n_history, long ld_generated,
                                    float repetition, float presence, float frequency, const float* repetition_rows,
                                    const float* presence_rows, const float* frequency_rows, const float* bias, long ld_bias,
                                    const void* allowed, long ld_allowed) {
    MOLLY_ENTER();
    MOLLY_CHECK(rows >= 0 && rows <= 65535 && V > 0 && V <= 0x40000000 && ld_logits >= V && ld_out >= V, "process_logits: rows=%d (at most 65535) V=%d (at most 2^30) ld=%ld/%ld", rows, V,
                ld_logits, ld_out);
    MOLLY_CHECK(n_history >= 0 && (n_history == 0 || (generated && ld_generated >= n_history)), "process_logits: %d generated tokens, ld=%ld", n_history,
                ld_generated);
    MOLLY_CHECK(repetition > 0.f, "process_logits: repetition penalty %g must be > 0", (double)repetition);
    MOLLY_CHECK(!bias || ld_bias == 0 || ld_bias >= V, "process_logits: ld_bias=%ld", ld_bias);
    MOLLY_CHECK(!allowed || ld_allowed == 0 || ld_allowed >= (V + 31) / 32, "process_logits: ld_allowed=%ld words for %d tokens", ld_allowed, V);
    if (rows == 0) return 0;
    MOLLY_CHECK(logits && out, "process_logits: logits and out required");
    LogitArgs p{};
    p.x = logits; p.out = out; p.gen = n_history ? (const long*)generated : nullptr; p.n_gen = n_generated_or_null;
    p.rep_v = repetition_rows; p.pres_v = presence_rows; p.freq_v = frequency_rows; p.bias = bias; p.mask = (const unsigned*)allowed;
    p.rep = repetition; p.pres = presence; p.freq = frequency; p.V = V; p.n_hist = n_history;
    p.ldx = ld_logits; p.ldo = ld_out; p.ldg = ld_generated; p.ldb = ld_bias; p.ldm = ld_allowed;
    hipStream_t st = (hipStream_t)stream;
    if (n_history == 0) launch<256, false>(st, p, rows, logits_bf16 != 0);
    else if (n_history < LONG_HISTORY) launch<256, true>(st, p, rows, logits_bf16 != 0);
    else launch<1024, true>(st, p, rows, logits_bf16 != 0);
    MOLLY_LAUNCH_CHECK();
    return 0;
}
