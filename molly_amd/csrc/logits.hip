// Logit processors in front of the draw: penalties for repeated tokens, a bias and a mask of allowed tokens, in one pass over the row.
//   c    = how often the token occurs in the row's generated sequence
//   c > 0:  s = (s < 0 ? s * repetition : s / repetition) - presence       (the first is HF's RepetitionPenaltyLogitsProcessor,
//   s   -= frequency * c                                                    HF:generation/logits_process.py; the reference's generate passes
//   s   += bias[token]                                                      repetition_penalty through, src/model/omics_one.py:220-232)
//   s    = -inf where the token's bit of the mask is 0                     (HF's prefix_allowed_tokens_fn / bad_words_ids)
// One workgroup = one row x one slice of the vocabulary: it counts the row's history into LDS (integer atomics: the order changes
// nothing), then makes the slice's pass.  Bound by HBM: the logits are read once and written once; the history comes from L2 once per slice.
#include "common.h"
#include "molly_hip.h"

namespace {

struct LogitArgs {
    const void* x; float* out;
    const long* gen; const int* n_gen;
    const float* rep_v; const float* pres_v; const float* freq_v;       // per row (nullable: the scalars)
    const float* bias; const unsigned* mask;
    float rep, pres, freq;
    int V, n_hist;
    long ldx, ldo, ldg, ldb, ldm;                     // ldb / ldm 0: one row for all
};

template <int SLICE, bool BF16>
__global__ __launch_bounds__(256) void logits_kernel(LogitArgs p) {
    __shared__ unsigned cnt[SLICE];
    const int row = blockIdx.y, v0 = blockIdx.x * SLICE, v1 = min(v0 + SLICE, p.V), t = threadIdx.x;
    const int n = p.gen ? min(max(p.n_gen ? p.n_gen[row] : p.n_hist, 0), p.n_hist) : 0;
    if (n > 0) {                                      // (block-uniform)
        for (int i = t; i < SLICE; i += 256) cnt[i] = 0u;
        __syncthreads();
        const long* g = p.gen + (size_t)row * p.ldg;
        for (int i = t; i < n; i += 256) {
            const long id = g[i];
            if (id >= v0 && id < v1) atomicAdd(&cnt[(int)(id - v0)], 1u);
        }
        __syncthreads();
    }
    const float rep = p.rep_v ? p.rep_v[row] : p.rep, pres = p.pres_v ? p.pres_v[row] : p.pres, freq = p.freq_v ? p.freq_v[row] : p.freq;
    for (int v = v0 + t; v < v1; v += 256) {
        float s = BF16 ? bf2f(((const bf16_t*)p.x)[(size_t)row * p.ldx + v]) : ((const float*)p.x)[(size_t)row * p.ldx + v];
        const unsigned c = n > 0 ? cnt[v - v0] : 0u;
        if (c) s = (s < 0.f ? s * rep : s / rep) - pres - freq * (float)c;
        if (p.bias) s += p.bias[(size_t)row * p.ldb + v];
        if (p.mask && !((p.mask[(size_t)row * p.ldm + (v >> 5)] >> (v & 31)) & 1u)) s = -INFINITY;
        p.out[(size_t)row * p.ldo + v] = s;
    }
}

}  // namespace

extern "C" int molly_process_logits(void* stream, const void* logits, int logits_bf16, float* out, int rows, int V, long ld_logits, long ld_out,
                                    const int64_t* generated, const int* n_generated_or_null, int n_history, long ld_generated,
                                    float repetition, float presence, float frequency, const float* repetition_rows,
                                    const float* presence_rows, const float* frequency_rows, const float* bias, long ld_bias,
                                    const void* allowed, long ld_allowed) {
    MOLLY_ENTER();
    MOLLY_CHECK(rows >= 0 && rows <= 65535 && V > 0 && ld_logits >= V && ld_out >= V, "process_logits: rows=%d (at most 65535) V=%d ld=%ld/%ld", rows, V,
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
    constexpr int SLICE = 4096;
    const dim3 grid(cdiv(V, SLICE), rows);
    if (logits_bf16) hipLaunchKernelGGL((logits_kernel<SLICE, true>), grid, dim3(256), 0, (hipStream_t)stream, p);
    else hipLaunchKernelGGL((logits_kernel<SLICE, false>), grid, dim3(256), 0, (hipStream_t)stream, p);
    MOLLY_LAUNCH_CHECK();
    return 0;
}
