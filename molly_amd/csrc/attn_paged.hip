// Attention of ragged chunks of new tokens over the paged cache (layout: paged.h).
//   out[t, h] = sum_j softmax_j(scale q . k_j) v_j   over the keys j <= kv_len - n + i  of the sequence that row t, its i-th of n new ones, is in
// replaces the attention of HF's generate over a DynamicCache (reference src/model/omics_one.py:220-232; HF:models/qwen3/
// modeling_qwen3.py:185-208) for prompts taken in pieces, continued sequences and batches that mix both with decode steps.
//
// The query heads of a kv head are packed into the rows of one tile (row = token * G + head of the group), so K and V are read once for all of
// them whatever G is; the arithmetic is that of attention.hip: S^T = K Q^T and O^T = V^T P^T by 32x32x16 MFMA, online softmax in the exp2
// domain in fp32, P in bf16 for the second product (one bf16 in the tiles, the sum of two in the rows: attend32).  Two kernels:
//   attn_paged_rows_kernel : up to 32 rows a tile (decode, short chunks).  The 4 | 8 waves of a block take turns at steps of 32 keys, each with
//                            K / V images of its own in LDS: no workgroup barrier in the loop, the waves meet at the end.  Bound by HBM.
//   attn_paged_tile_kernel : 128 rows a tile (prompt chunks, mixed batches), 64 where there are few tiles (KS 2: two waves a row, half of the keys each).  The waves
//                            own 32 rows each and share K / V tiles of 64 keys, double-buffered.  Bound by the matrix pipes where the chunk is long.
// Either cuts the key axis over blocks where there are too few tiles to fill the chip; attn_paged_join_kernel joins the parts.
// A bf16 step's rows go straight to LDS by DMA (16 keys lie within one page, so one page id serves a wave's piece); e4m3 codes pass through registers,
// are turned into bf16 there (exactly, but for paged.h's two ends) and stored into the same image: one set of fragment reads serves both.
#include "attn_frag.h"
#include "common.h"
#include "molly_hip.h"
#include "paged.h"

namespace {

constexpr int RROWS = 32;                            // rows of a tile in the rows kernel; the tile kernel has 32 a wave
constexpr int MAX_PARTS = 64;
// Most keys a sequence's row of the table may hold.  Key numbers are ints, and some are taken beyond the last key: the lookup of the page ids asks 31 steps of 256
// keys and 16 ahead (7,952), and the parts of a cut axis, each rounded up to 256 keys, end up to 64 * 256 = 16,384 behind it.
constexpr long MAX_KEYS = 0x7fffffffL - 32768;

// The parts that a tile's key axis is cut into, at most `parts`, and a part's keys (whole ones of `align`).  A part has 2^shift keys or so at least (`round`: what
// counts as the last one); an axis of which a cut would take fewer than min_cut keys out of a block's way stays whole.
//   single steps: a round of the block's waves or more, min_cut 700: 828 keys and more are cut where a round is 128 keys, 956 where it is 256.  On the GPU the join costs 4 us
//     and a key 9 ns, and a cut pays from 400 keys saved on (in a graph, bf16: 1 x 700 11.1 -> 9.5 us, 1 x 300 7.9 -> 9.8, 1 x 828 11.8 -> 9.2, 1 x 2,000 20.9 -> 10.0, 4 x 2,000
//     23.7 -> 12.0).  Called one by one the second launch and its scratch are host time, and it pays from some 1,100 keys on (1 x 700 11.5 -> 15.2, 1 x 828 11.9 -> 14.2,
//     1 x 1,000 13.0 -> 14.1, 1 x 1,200 15.2 -> 14.1; with a scratch of the caller's 12.2 each): 700 lies between.  16 x 700 e4m3, cut in two in a graph, 12.7 -> 14.7
//   tiles: 512 keys or more, for their parts carry more rows (2 x 100 new tokens x 32 heads over 1,000 keys 19.7 us, parts of 128 21.8); 128 where that makes
//     more parts, up to 16 and as long as they come to 10,240 rows (32 new tokens x 32 heads over 700 keys 15.3 -> 13.1 us, over 2,500 18.5 -> 15.5)
struct CutRule { int parts, align, shift, round, min_cut; };
struct Cut { int parts, keys; };
__host__ __device__ inline Cut cut_keys(const CutRule& c, int n) {
    const int most = (n + c.round) >> c.shift, d = c.parts < most ? c.parts : most;
    if (d <= 1) return {1, n};
    const int keys = ((n - 1) / d + c.align) / c.align * c.align;                     // n / d rounded up, to the next multiple
    return n - keys < c.min_cut ? Cut{1, n} : Cut{(n - 1) / keys + 1, keys};
}

struct AttnPagedArgs {
    const bf16_t* q; bf16_t* out;
    const char* kpool; const char* vpool; const uint8_t* kscale; const uint8_t* vscale;
    const int* table; const int* cu_q; const int* kv_len;
    float* part;                                     // [tile][kv head][parts]: ROWS * HD un-normalised outputs, ROWS * 2 (max, sum)
    int n_tok, B, n_pages, page_shift, max_pages, ld_table, nh, nkv, G, ldq, ldo;
    int tps;                                         // rows kernel: tiles per sequence; tile kernel: bound of the tiles of all of them
    CutRule cut;
    int class_bits;                                  // find_tile: 2^class_bits classes of 64 keys
    float scale_log2;                                // softmax scale * log2(e), > 0
};

// what a tile of query rows is: R0 .. R0 + rows - 1 of the n * G rows of its sequence
struct Tile {
    int b, tok0, n, row0, rows;                      // sequence, its first row in q, its new tokens, first packed row, packed rows
    int first;                                       // key that row 0 of the sequence sees last (kv_len - n)
    int n_vis;                                       // keys that the tile's last row sees (<= 0: none)
};
template <int ROWS>
__device__ __forceinline__ Tile make_tile(const AttnPagedArgs& p, int b, int ti) {
    Tile t;
    t.b = b;
    const int s = min(max(p.cu_q[b], 0), p.n_tok), e = min(max(p.cu_q[b + 1], s), p.n_tok);
    t.tok0 = s; t.n = e - s;
    t.row0 = ti * ROWS;
    t.rows = min(ROWS, t.n * p.G - t.row0);
    t.first = max(p.kv_len[b], 0) - t.n;             // (less than no keys: no row sees one either way, and the difference stays in 32 bits)
    t.n_vis = t.rows > 0 ? t.first + (t.row0 + t.rows - 1) / p.G + 1 : 0;
    return t;
}
// ---- K / V steps ------------------------------------------------------------------------------------------------------------------------
struct KvSource {
    const int* row;                                  // the sequence's page ids
    int n_pages, shift, nkv, kvh;
    // index (in keys of the pool) of the 16 keys that hold `key`, with the page id already loaded; a page that is none reads page 0 (the rows that see
    // it are made NaN at the end)
    __device__ __forceinline__ size_t group(int key, int page) const {
        const unsigned pg = (unsigned)page < (unsigned)n_pages ? (unsigned)page : 0u;
        return (((size_t)pg * nkv + kvh) << shift) + (key & ((1 << shift) - 1) & ~15);
    }
};

// R (16 | 8) rows of a 16-key group, from row `r0` of the tile image on, by LDS-DMA: PIECES of 1 KiB per matrix.  `off`: the lane's byte offsets from the
// group's first row (piece_row_col); `lds`: where the piece's rows start in the image.
template <int HD, int R> constexpr int PIECES = R * HD / 512;
template <int HD> __device__ __forceinline__ void piece_row_col(int i, int lane, int& row, int& col) {      // piece i of a group
    constexpr int NCB = HD / 16;
    const int blk = lane >> 3, cin = lane & 7, rbl = i * (8 / NCB) + blk / NCB, b0 = rbl & 1, b1 = (rbl >> 1) & 1;
    row = rbl * 4 + (cin >> 1);
    col = (((blk % NCB) ^ b0) << 4) + (((cin & 1) ^ b1) << 3);
}
template <bool NT> __device__ __forceinline__ void dma16(unsigned off, const char* base, unsigned lds) {
    // (from asm, as in attention.hip: with the builtin hipcc waits for every pending LDS-DMA in front of the next transposed read)
    if (NT) asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 nt" ::"v"(off), "s"(base), "s"(lds) : "memory", "m0");
    else asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds) : "memory", "m0");
}
template <int HD, int R>
__device__ __forceinline__ void piece_offsets(int r0, int lane, unsigned (&off)[PIECES<HD, R>]) {
#pragma unroll
    for (int i = 0; i < PIECES<HD, R>; ++i) {
        int row, col;
        piece_row_col<HD>((r0 & 15) * HD / 512 + i, lane, row, col);
        off[i] = (unsigned)((row * HD + col) * 2);
    }
}
template <bool NT, int N>
__device__ __forceinline__ void dma_rows(const char* base, unsigned lds, const unsigned (&off)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) dma16<NT>(off[i], base, __builtin_amdgcn_readfirstlane(lds + i * 1024));
}
// the same for the group that the last key is in (or lies in front of): rows behind it repeat it, so that nothing behind a sequence's end — stale
// pages may hold NaN — gets into the tile
template <int HD, int R>
__device__ __forceinline__ void dma_rows_clamped(const char* base, unsigned lds, int r0, int lim, int lane) {
#pragma unroll
    for (int i = 0; i < PIECES<HD, R>; ++i) {
        int row, col;
        piece_row_col<HD>((r0 & 15) * HD / 512 + i, lane, row, col);
        dma16<false>((unsigned)((min(row, lim) * HD + col) * 2), base, __builtin_amdgcn_readfirstlane(lds + i * 1024));
    }
}
// every LDS read of this wave has its data: what it read may be overwritten
__device__ __forceinline__ void lds_read_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
template <int N> __device__ __forceinline__ void wait_vm() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// A 16-key group as e4m3 codes through registers: NL loads of 16 codes a lane, K's units first, then V's.
template <int HD> struct Codes {
    static constexpr int UPM = HD, NL = 2 * UPM / 64;                // units of 16 codes per matrix; loads a lane
    u32x4 c[NL];
    uint8_t e[NL];
};
// a lane's unit: row block (of 4), row in it, column block.  Eight neighbouring lanes take four rows and the four of the row block after the next, whose halves
// lie the other way round in the image: their stores meet in no bank.  (Four rows of two column blocks: two lanes in every bank, 29 % of the LDS cycles of
// a mixed batch; 6 x 301 new tokens over 2,500 keys 120 -> 113 us, 2,048 over 16,384 531 -> 519.)  But a load takes half of 128-byte rows then,
// and the streaming ones (NT) fetch them twice: 32 x 4,000 keys 49.0 -> 64.9 us, so those take whole rows.
template <int HD, bool NT> __device__ __forceinline__ void code_unit(int w, int& rb, int& r, int& cb) {
    r = w & 3;
    if constexpr (NT && HD == 128) {
        cb = (w >> 2) & 7;
        rb = w >> 5;
    } else {
        rb = ((w >> 2) & 1) * 2 + ((w >> 3) & 1);
        cb = w >> 4;
    }
}
template <int HD, bool NT>
__device__ __forceinline__ void codes_load(Codes<HD>& c, const AttnPagedArgs& p, size_t at, int lim, int lane) {
#pragma unroll
    for (int j = 0; j < Codes<HD>::NL; ++j) {
        const int u = j * 64 + lane;
        const bool isv = u >= Codes<HD>::UPM;
        int rb, r, cb;
        code_unit<HD, NT>(u % Codes<HD>::UPM, rb, r, cb);
        const size_t key = at + min(rb * 4 + r, lim);
        const u32x4* src = reinterpret_cast<const u32x4*>((isv ? p.vpool : p.kpool) + key * HD + cb * 16);
        c.c[j] = NT ? __builtin_nontemporal_load(src) : *src;
        c.e[j] = (isv ? p.vscale : p.kscale)[key];
    }
}
template <int HD, bool NT>
__device__ __forceinline__ void codes_store(const Codes<HD>& c, bf16_t* imgk, bf16_t* imgv, int r0, int lane) {      // rows r0 .. of the tile's images
    constexpr int NCB = HD / 16;
#pragma unroll
    for (int j = 0; j < Codes<HD>::NL; ++j) {
        const int u = j * 64 + lane;
        int rb, r, cb;
        code_unit<HD, NT>(u % Codes<HD>::UPM, rb, r, cb);
        const int rbl = (r0 >> 2) + rb, b0 = rbl & 1, b1 = (rbl >> 1) & 1;
        bf16_t* d = (u >= Codes<HD>::UPM ? imgv : imgk) + (rbl * NCB + (cb ^ b0)) * 64 + r * 16;
        const float scale = exp2i((int)c.e[j] - 127);
        *reinterpret_cast<u32x4*>(d + b1 * 8) = e4m3_to_bf8(u32x2{c.c[j][0], c.c[j][1]}, scale);
        *reinterpret_cast<u32x4*>(d + (b1 ^ 1) * 8) = e4m3_to_bf8(u32x2{c.c[j][2], c.c[j][3]}, scale);
    }
}

// ---- 32 query rows of a wave ---------------------------------------------------------------------------------------------------------------
template <int HD> struct Rows {
    bf16x8 qf[HD / 16];                              // B operand of S^T: lane (r, h) holds q[row r][16 s + 8 h .. +7]
    f32x16 o[HD / 32];                               // O^T: lane = row, registers = columns
    float m, l;                                      // running maximum (log2 domain, scaled) and this half-wave's part of the sum
    int qi;                                          // last key the lane's row sees
    int qmin, qmax;                                  // over the wave's rows (uniform)
    bool odd;                                        // add_odd has something to do (uniform)
};
template <int HD>
__device__ __forceinline__ void rows_init(Rows<HD>& st, const AttnPagedArgs& p, const Tile& t, int kvh, int wave_row, int lane) {
    const int r = lane & 31, h = lane >> 5;
    const int R = t.row0 + min(wave_row + r, t.rows - 1);          // (lanes behind the tile's last row repeat it)
    const int tok = R / p.G, g = R - tok * p.G;
    const bf16_t* qp = p.q + (size_t)(t.tok0 + tok) * p.ldq + (kvh * p.G + g) * HD + 8 * h;
#pragma unroll
    for (int s = 0; s < HD / 16; ++s) st.qf[s] = *reinterpret_cast<const bf16x8*>(qp + 16 * s);
#pragma unroll
    for (int d = 0; d < HD / 32; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) st.o[d][e] = 0.f;
    st.m = -INFINITY; st.l = 0.f; st.odd = false;
    st.qi = t.first + tok;
    st.qmin = t.first + (t.row0 + min(wave_row, t.rows - 1)) / p.G;
    st.qmax = t.first + (t.row0 + min(wave_row + 31, t.rows - 1)) / p.G;
}

// V values that are not finite, in a step that some row does not see all of: P is 0 there, and 0 * NaN would be NaN.  attend32 takes them out of such
// a step (clear_odd) and this adds them to the rows that do see them, at the end.  step0, step0 + stride ..: the wave's steps below k1.
template <int HD, bool FP8>
__device__ __forceinline__ void add_odd(Rows<HD>& st, const AttnPagedArgs& p, const KvSource& src, int step0, int stride, int k1, int lane) {
    const int h = lane >> 5;
#pragma unroll 1
    for (int kb = step0; kb < k1; kb += stride) {
        if (kb + 31 <= st.qmin) continue;                // (every row saw these: they went through the product)
#pragma unroll 1
        for (int key = kb; key < min(kb + 32, k1); ++key) {
            const size_t at = src.group(key, src.row[key >> src.shift]) + (key & 15);
            const float scale = FP8 ? exp2i((int)p.vscale[at] - 127) : 1.f;
#pragma unroll
            for (int d = 0; d < HD / 32; ++d)
#pragma unroll
                for (int g4 = 0; g4 < 4; ++g4) {
                    const int col = 32 * d + 8 * g4 + 4 * h;
                    u32x2 w;
                    if constexpr (FP8) {
                        const u32x4 x = e4m3_to_bf8(u32x2{*reinterpret_cast<const unsigned*>(p.vpool + at * HD + col), 0u}, scale);
                        w = u32x2{x[0], x[1]};
                    } else {
                        w = *reinterpret_cast<const u32x2*>(p.vpool + (at * HD + col) * 2);
                    }
                    const float x[4] = {bflo(w[0]), bfhi(w[0]), bflo(w[1]), bfhi(w[1])};
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        st.o[d][4 * g4 + e] += key <= st.qi && !(fabsf(x[e]) < INFINITY) ? x[e] : 0.f;
                }
        }
    }
}
// values whose exponent field is all ones -> 0; true if there was one in any lane
template <int ND>
__device__ __forceinline__ bool clear_odd(bf16x8 (&vf)[2][ND]) {
    typedef __attribute__((ext_vector_type(2))) unsigned short u16x2;
    const u16x2 limit = {0x7f7f, 0x7f7f}, one = {1, 1};
    u16x2 top = {0, 0};
#pragma unroll
    for (int sp = 0; sp < 2; ++sp)
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            const u32x4 w = __builtin_bit_cast(u32x4, vf[sp][d]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const unsigned x = w[j] & 0x7f807f80u;
                top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, x));
            }
        }
    if (!__any(top[0] == 0x7f80 || top[1] == 0x7f80)) return false;
#pragma unroll
    for (int sp = 0; sp < 2; ++sp)
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            u32x4 w = __builtin_bit_cast(u32x4, vf[sp][d]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const unsigned x = w[j] & 0x7f807f80u;
                const u16x2 odd = __builtin_elementwise_sub_sat(__builtin_bit_cast(u16x2, x), limit);       // 1: not finite
                w[j] &= __builtin_bit_cast(unsigned, (u16x2)(odd - one));
            }
            vf[sp][d] = __builtin_bit_cast(bf16x8, w);
        }
    return true;
}

// the upper halves of floats: bf16, rounded towards 0
__device__ __forceinline__ float cut_bf(float x) { return __builtin_bit_cast(float, __builtin_bit_cast(unsigned, x) & 0xffff0000u); }
__device__ __forceinline__ unsigned cut_bf2(float lo, float hi) {
    return __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, hi), __builtin_bit_cast(unsigned, lo), 0x07060302);
}

// one step of 32 keys: rows `sub` * 32 .. of the images, keys kbase ..
// FINE: P goes through the second product as two bf16, cut off and rest, which leaves 2^-16 of a term where one bf16 leaves 2^-8: the output has
// no error but its own rounding then (relative to 64 bits 0.0017 instead of 0.0023).  The rest is taken from P (1 + 2^-20): positive wherever P is, so that
// an infinite V makes it infinite and not 0 * inf.  Single steps wait for memory and pay little for it:
// 32 x 4,000 keys e4m3 49.6 -> 50.0 us, bf16 93.2 -> 94.7, 1 x 700 bf16 11.0 -> 11.5, 64 x 2,000 at head dim 64 e4m3 25.5 -> 26.7.  The tiles
// are bound by the matrix pipes, where it would be half as much work again.
template <int HD, bool FINE>
__device__ __forceinline__ void attend32(Rows<HD>& st, const bf16_t* sK, const bf16_t* sV, int sub, int kbase, float scale_log2, int lane) {
    constexpr int NS = HD / 16, ND = HD / 32;
    const int r = lane & 31, h = lane >> 5;
    bf16x8 kf[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s) kf[s] = row_frag<HD>(sK, 32 * sub + r, s, h);
    __builtin_amdgcn_sched_barrier(0);               // every read in flight before the first MFMA
    f32x16 sc;
#pragma unroll
    for (int e = 0; e < 16; ++e) sc[e] = 0.f;
#pragma unroll
    for (int s = 0; s < NS; ++s) sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[s], st.qf[s], sc, 0, 0, 0);
    bf16x8 vf[2][ND];
#pragma unroll
    for (int sp = 0; sp < 2; ++sp)
#pragma unroll
        for (int d = 0; d < ND; ++d) vf[sp][d] = tr_frag<HD>(sV, 32 * sub, sp, d, lane);
    const bool edge = kbase + 31 > st.qmin;          // (uniform) some row does not see all of the step
    if (edge) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int key = kbase + (e & 3) + 8 * (e >> 2) + 4 * h;
            sc[e] = key <= st.qi ? sc[e] : -INFINITY;
        }
        if (clear_odd<ND>(vf)) st.odd = true;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int e = 0; e < 16; ++e) mx = fmaxf(mx, sc[e]);
    mx = xhalf_max(mx) * scale_log2;
    if (!__all(mx - st.m <= RESCALE_THR)) {          // the reference maximum follows only where it has grown by more than 2^8
        const float m_new = fmaxf(st.m, mx);
        const float alpha = fast_exp2(st.m - (m_new == -INFINITY ? 0.f : m_new));
        st.l *= alpha;
        st.m = m_new;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) st.o[d][e] *= alpha;
    }
    const float m_ref = st.m == -INFINITY ? 0.f : st.m;
#pragma unroll
    for (int e = 0; e < 16; ++e) sc[e] = fast_exp2(sc[e] * scale_log2 - m_ref);
    float rs[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) rs[g] = (sc[4 * g] + sc[4 * g + 1]) + (sc[4 * g + 2] + sc[4 * g + 3]);
    st.l += (rs[0] + rs[1]) + (rs[2] + rs[3]);
    bf16x8 pf[2];
#pragma unroll
    for (int sp = 0; sp < 2; ++sp) {
        if constexpr (FINE) {
            u32x4 w;
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = cut_bf2(sc[8 * sp + 2 * j], sc[8 * sp + 2 * j + 1]);
            pf[sp] = __builtin_bit_cast(bf16x8, w);
        } else {
            pf[sp] = acc_to_frag(sc, 8 * sp);
        }
    }
#pragma unroll
    for (int d = 0; d < ND; ++d) {
        st.o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[0][d], pf[0], st.o[d], 0, 0, 0);
        st.o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[1][d], pf[1], st.o[d], 0, 0, 0);
    }
    if constexpr (FINE) {
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[e] = __builtin_fmaf(sc[e], 1.f + 0x1p-20f, -cut_bf(sc[e]));
#pragma unroll
        for (int sp = 0; sp < 2; ++sp) pf[sp] = acc_to_frag(sc, 8 * sp);
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            st.o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[0][d], pf[0], st.o[d], 0, 0, 0);
            st.o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[1][d], pf[1], st.o[d], 0, 0, 0);
        }
    }
}

// the first of the keys k0 .. k1 - 1 that lies on a page that is none, by all threads of the block (0x7fffffff: all pages are); *sh is set
// behind the next barrier
template <int THREADS>
__device__ __forceinline__ void scan_pages(const AttnPagedArgs& p, const int* row, int k0, int k1, int* sh) {
    const int last = k1 > k0 ? (k1 - 1) >> p.page_shift : -1;
    for (int i = (k0 >> p.page_shift) + threadIdx.x; i <= last; i += THREADS)
        if ((unsigned)row[i] >= (unsigned)p.n_pages) atomicMin(sh, i << p.page_shift);
}

// ---- short chunks: tiles of up to 32 rows; a block's NW waves take every NW-th step of 32 keys ------------------------------------------------------------
// (Cutting all sequences' keys into equal shares, whatever tiles they belong to, was measured too: 45.7 us against 45.8 for 32 x 1,000..4,000
// keys, and 64.5 against 57.2 where all are 4,000 long: finding a share's place and a second tile per block cost what the balance gains.)
// NW: as many waves as their images leave room for on a compute unit (128 KB for all but e4m3 at dim 64, two blocks there), two a SIMD but for bf16 at dim 128
// (eight waves with one buffer each there: 106.4 us against 104.6 for 32 x 4,000 keys, 97.4 against 94.5 for 4 x 32,768)
constexpr int rows_waves(int head_dim, bool fp8) { return head_dim == 128 && !fp8 ? 4 : 8; }
template <int HD, bool FP8>
__global__ __launch_bounds__(64 * rows_waves(HD, FP8), rows_waves(HD, FP8) / 4) void attn_paged_rows_kernel(AttnPagedArgs p) {
    constexpr int NW = rows_waves(HD, FP8), STRIDE = 32 * NW;      // keys between two steps of a wave
    extern __shared__ __attribute__((aligned(16))) char smem[];
    __shared__ int s_bad;
    __shared__ float s_ml[NW][RROWS][2];
    constexpr int IMG = 32 * HD;                     // elements of a step's K (or V) image
    constexpr int NBUF = FP8 ? 1 : 2;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    bf16_t* img = reinterpret_cast<bf16_t*>(smem) + wave * NBUF * 2 * IMG;            // [buffer][K | V]
    const unsigned img_lds = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)LDS_PTR(img));
    unsigned off[PIECES<HD, 16>];
    piece_offsets<HD, 16>(0, lane, off);
    int bid = blockIdx.x;
    const int s = bid % p.cut.parts; bid /= p.cut.parts;
    const int kvh = bid % p.nkv; bid /= p.nkv;
    const int b = bid / p.tps;
    for (int ti = bid % p.tps;; ti += p.tps) {       // (a sequence has more tiles than p.tps only where the caller's max_q was too small)
        const Tile t = make_tile<RROWS>(p, b, ti);
        if (t.rows <= 0) return;
        const int kmax = p.max_pages << p.page_shift;
        const int n_keys = min(t.n_vis, kmax);
        const Cut cut = ti < p.tps ? cut_keys(p.cut, n_keys) : Cut{1, n_keys};
        const int parts = cut.parts, chunk = cut.keys;
        if (s >= parts) continue;
        const int k0 = s * chunk, k1 = min(n_keys, k0 + chunk);
        float* part = parts > 1 ? p.part + ((size_t)((b * p.tps + ti) * p.nkv + kvh) * p.cut.parts + s) * (RROWS * (HD + 2)) : nullptr;
        const int last = k1 - 1;
        const KvSource src{p.table + (size_t)t.b * p.ld_table, p.n_pages, p.page_shift, p.nkv, kvh};
        if (tid == 0) s_bad = t.n_vis > kmax ? kmax : 0x7fffffff;
        Rows<HD> st;
        rows_init<HD>(st, p, t, kvh, 0, lane);
        const int key0 = k0 + 32 * wave;
        // page ids of the wave's next 32 steps, two groups each: lane 2 i + g.  Waited for here, once in 32 steps: a wait inside the steps would be a wait for
        // the DMA in flight.
        int pages = 0;
        auto look = [&](int key) {
            const int i = (key - key0) / STRIDE;
            if ((i & 31) == 0) {
                pages = src.row[min(key + (lane >> 1) * STRIDE + (lane & 1) * 16, last) >> p.page_shift];
                arrived(pages);
            }
            return i & 31;
        };
        auto dma_step = [&](int key, int buf) {
            const int i = look(key);
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const int kb = key + 16 * g, kc = min(kb, last & ~15);
                const size_t at = src.group(kc, __builtin_amdgcn_readlane(pages, 2 * i + g)) * (HD * 2);
                const unsigned dst = img_lds + (buf * 2 * IMG + g * 16 * HD) * 2;
                if (kb + 15 <= last) {
                    dma_rows<true>(p.kpool + at, dst, off);
                    dma_rows<true>(p.vpool + at, dst + IMG * 2, off);
                } else {
                    const int lim = kb > last ? 0 : last - kc;              // (a group behind the last key: 16 copies of a key that is there)
                    dma_rows_clamped<HD, 16>(p.kpool + at, dst, 0, lim, lane);
                    dma_rows_clamped<HD, 16>(p.vpool + at, dst + IMG * 2, 0, lim, lane);
                }
            }
        };
        if constexpr (FP8) {
            // (one step's codes on their way in registers; three, at one block a CU, were slower: 52.8 us against 45.8 for 32 x 1,000..4,000 keys.  A lone wave
            // spends 1.3 us a step, 0.65 of it in attend32 and 0.37 in the conversion: it is a second wave on the SIMD that hides them)
            Codes<HD> c[2];
            auto load_step = [&](int key) {
                const int i = look(key);
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    const int kb = key + 16 * g, kc = min(kb, last & ~15);
                    codes_load<HD, true>(c[g], p, src.group(kc, __builtin_amdgcn_readlane(pages, 2 * i + g)), kb > last ? 0 : min(last - kc, 15), lane);
                }
            };
            if (key0 < k1) load_step(key0);
#pragma unroll 1
            for (int key = key0; key < k1; key += STRIDE) {
#pragma unroll
                for (int g = 0; g < 2; ++g) codes_store<HD, true>(c[g], img, img + IMG, 16 * g, lane);
                if (key + STRIDE < k1) load_step(key + STRIDE);
                attend32<HD, true>(st, img, img + IMG, 0, key, p.scale_log2, lane);
            }
        } else {
#pragma unroll
            for (int i = 0; i < HD / 16; ++i) arrived(st.qf[i]);
            if (key0 < k1) dma_step(key0, 0);
            int buf = 0;
#pragma unroll 1
            for (int key = key0; key < k1; key += STRIDE) {
                if (key + STRIDE < k1) {
                    lds_read_done();                 // (the other buffer, in the step before)
                    dma_step(key + STRIDE, buf ^ 1);
                    // this step's pieces have landed when only the next one's are still out
                    wait_vm<4 * PIECES<HD, 16>>();
                } else {
                    dma_wait();
                }
                attend32<HD, true>(st, img + buf * 2 * IMG, img + buf * 2 * IMG + IMG, 0, key, p.scale_log2, lane);
                buf ^= 1;
            }
        }
        if (st.odd) add_odd<HD, FP8>(st, p, src, k0 + 32 * wave, STRIDE, k1, lane);
        __syncthreads();                             // the images are dead; s_bad is set
        scan_pages<64 * NW>(p, src.row, k0, k1, &s_bad);
        // the waves' rows, un-normalised, through LDS
        const int r = lane & 31, h = lane >> 5;
        const float l = st.l + __shfl_xor(st.l, 32, 64);
        if (h == 0) { s_ml[wave][r][0] = st.m; s_ml[wave][r][1] = l; }
        float* acc = reinterpret_cast<float*>(smem) + (size_t)wave * RROWS * HD;
        if (r < t.rows)
#pragma unroll
            for (int d = 0; d < HD / 32; ++d)
#pragma unroll
                for (int g4 = 0; g4 < 4; ++g4)
                    *reinterpret_cast<f32x4*>(acc + r * HD + 32 * d + 8 * g4 + 4 * h) =
                        f32x4{st.o[d][4 * g4], st.o[d][4 * g4 + 1], st.o[d][4 * g4 + 2], st.o[d][4 * g4 + 3]};
        __syncthreads();
        const int bad = s_bad;
        for (int i = tid; i < t.rows * (HD / 4); i += 64 * NW) {
            const int row = i / (HD / 4), c4 = (i % (HD / 4)) * 4;
            float m = -INFINITY;
#pragma unroll
            for (int w = 0; w < NW; ++w) m = fmaxf(m, s_ml[w][row][0]);
            const float mu = m == -INFINITY ? 0.f : m;
            f32x4 a = {0.f, 0.f, 0.f, 0.f};
            float ls = 0.f;
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const float f = fast_exp2(s_ml[w][row][0] - mu);
                const f32x4 x = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(smem) + ((size_t)w * RROWS + row) * HD + c4);
                ls += s_ml[w][row][1] * f;
#pragma unroll
                for (int e = 0; e < 4; ++e) a[e] += f == 0.f ? 0.f : x[e] * f;            // (a wave without keys has zeros: never 0 * inf)
            }
            const int R = t.row0 + row, tok = R / p.G;
            if (t.first + tok >= bad) ls = __builtin_nanf("");
            if (part) {
                *reinterpret_cast<f32x4*>(part + row * HD + c4) = a;
                if (c4 == 0) { part[RROWS * HD + row * 2] = m; part[RROWS * HD + row * 2 + 1] = ls; }
            } else {
                const float inv = ls == 0.f ? 0.f : 1.f / ls;
                bf16_t* d = p.out + (size_t)(t.tok0 + tok) * p.ldo + (kvh * p.G + R - tok * p.G) * HD + c4;
                *reinterpret_cast<u32x2*>(d) = u32x2{pack_bf2(a[0] * inv, a[1] * inv), pack_bf2(a[2] * inv, a[3] * inv)};
            }
        }
        __syncthreads();                             // (the next tile's images and s_bad)
    }
}

// ---- long chunks: 128 or 64 rows a block -----------------------------------------------------------------------------------------------------------
// Sum over the lanes up to and including each (lane 63: all).
__device__ __forceinline__ int wave_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);      // row_shr 1, 2, 4, 8: within rows of 16
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);      // row_bcast 15: rows 1 and 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);      // row_bcast 31: rows 2 and 3
    return x;
}
__device__ __forceinline__ int wave_total(int x) { return __builtin_amdgcn_readlane(wave_scan(x), 63); }
// one sequence a lane: its tiles (0 behind the last sequence) and its keys, as far as they are ranked (at least 0)
struct Seq { int n, len; };
template <int TROWS> __device__ __forceinline__ Seq load_seq(const AttnPagedArgs& p, int b) {
    const int i = min(b, p.B - 1), s0 = p.cu_q[i], e0 = p.cu_q[i + 1], keys = p.kv_len[i];
    const int s = min(max(s0, 0), p.n_tok), rows = (min(max(e0, s), p.n_tok) - s) * p.G;
    return {b < p.B ? (rows + TROWS - 1) / TROWS : 0, min(max(keys, 0), (64 << p.class_bits) - 1)};
}
// The tile of a rank, 64 sequences after the other (the first 64 in `q`), of these the tile with the most keys first, in classes of 64 keys; within a class by sequence.
// A sequence's tiles are TROWS / G keys apart.  -1: there are fewer tiles.  (Ranked by their sequences' lengths only: 8 prompts of 314..1,111 tokens at head dim 64 32.5
// us against 27.0, 64 of 1,111 290 against 269; tiles of single steps ranked by half their keys: 24 sequences, a quarter of them with 301 new tokens, 89 us against 86.)
template <int TROWS> __device__ __forceinline__ int find_tile(const AttnPagedArgs& p, Seq q, int rank, int lane, int* ti) {
    const float per_key = (float)p.G / TROWS;
    for (int b0 = 0;;) {
        const Seq next = load_seq<TROWS>(p, b0 + 64 + lane);
        const int total = wave_total(q.n);
        if (rank < total) {
            if (p.B == 1) {
                *ti = total - 1 - rank;
                return 0;
            }
            auto least = [&](int c) {                // this sequence's tiles of class c or above
                const int over = q.len - 64 * c;
                return c == 0 ? q.n : over < 0 ? 0 : min(q.n, (int)fminf((float)over * per_key, 0x1p30f) + 1);
            };
            int c = 0;                               // the rank's class: the highest that has more than `rank` tiles in it and above it
            for (int bit = p.class_bits - 1; bit >= 0; --bit)
                if (wave_total(least(c | 1 << bit)) > rank) c |= 1 << bit;
            const int above = least(c + 1), here = least(c) - above;
            rank -= wave_total(above);
            const int upto = wave_scan(here), k = above + rank - (upto - here);      // (k-th from the sequence's last tile)
            const int who = __ffsll((long long)__ballot(rank < upto)) - 1;
            *ti = __builtin_amdgcn_readlane(q.n - 1 - k, who);
            return b0 + who;
        }
        rank -= total;
        b0 += 64;
        if (b0 >= p.B) return -1;
        q = next;
    }
}
// The rank of an XCD's block `pos`, of N.  Blocks start in order, the first 32 on a compute unit each, the next 32 on the same ones in the same order, while there is
// room (SLOTS blocks a unit); later ones where a block has ended.  So of every 64 the second half goes backwards: the longest shares its unit with the shortest; where
// the second half is not full, the longest are alone.  (2,048 tokens over 16,384 keys 512 -> 509 us, e4m3 548 -> 539; 4 x 512 over 3,000 e4m3 108.7 -> 107.)
template <int SLOTS> __device__ __forceinline__ int deal(int pos, int N) {
    const int base = pos & ~63, n = min(N - base, 64), i = pos & 63, k = n - 32;
    if (base >= 32 * SLOTS || k <= 0) return pos;
    return base + (i >= 32 ? n - 1 - (i - 32) : i < k ? 64 - n + i : i - k);
}

// KS 1: the waves own 32 rows each (128 a block).  KS 2: two own 32 rows each (64 a block) for the first half of every tile's keys, two the same rows for the
// second; they meet at the end.  Half the chain of steps a wave goes through, for twice the K / V traffic: for few tiles of unequal length.
template <int HD, bool FP8, int KS>
__global__ __launch_bounds__(256, 2) void attn_paged_tile_kernel(AttnPagedArgs p) {
    extern __shared__ __attribute__((aligned(16))) char smem_raw[];
    __shared__ int s_bad;
    bf16_t* smem = reinterpret_cast<bf16_t*>(smem_raw);            // [2 stages][K tile | V tile]
    constexpr int TILE = 64 * HD, TROWS = 128 / KS, R = 16;        // R: rows of a tile that a wave stages
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wrow = KS == 1 ? wave * 32 : (wave & 1) * 32, kg = KS == 1 ? 0 : wave >> 1;
    // The workgroups of one XCD (every eighth) share the keys of as few (kv head, part) units as possible in its L2: whole units to an XCD where they can
    // be dealt evenly, every X-th tile of a unit to each of its X XCDs where there are fewer, else contiguous runs of (unit, tile).
    const int units = p.nkv * p.cut.parts, xcd = blockIdx.x & 7, i8 = blockIdx.x >> 3;
    int pos, unit, x = 0, X = 1;                     // the unit's XCDs take every X-th tile, this one those of rank x, x + X ..
    bool whole = true;
    if (units % 8 == 0) {
        unit = xcd * (units / 8) + i8 / p.tps;
        pos = i8 % p.tps;
    } else if (8 % units == 0) {
        X = 8 / units;
        unit = xcd / X;
        x = xcd % X;
        pos = i8;
    } else {
        const int run = (units * p.tps + 7) / 8;
        const int v = xcd * run + i8;
        if (i8 >= run || v >= units * p.tps) return;
        unit = v / p.tps;
        pos = v % p.tps;
        whole = false;
    }
    const Seq seq = load_seq<TROWS>(p, lane);
    int f = pos * X + x;
    if (whole && p.B <= 64) {                        // (more sequences: more tiles than start at once)
        const int total = min(wave_total(seq.n), p.tps), N = (total - x + X - 1) / X;
        if (pos >= N) return;
        f = deal<HD == 128 || FP8 ? 2 : 4>(pos, N) * X + x;
    }
    if (f >= p.tps) return;                          // (more tiles than that only where cu_q does not ascend)
    const int s = unit % p.cut.parts, kvh = unit / p.cut.parts;
    int ti = 0;
    const int b = __builtin_amdgcn_readfirstlane(find_tile<TROWS>(p, seq, f, lane, &ti));
    if (b < 0) return;
    ti = __builtin_amdgcn_readfirstlane(ti);
    const Tile t = make_tile<TROWS>(p, b, ti);
    const int kmax = p.max_pages << p.page_shift;
    const int n_keys = min(t.n_vis, kmax);
    const Cut cut = cut_keys(p.cut, n_keys);
    const int parts = cut.parts, chunk = cut.keys;
    if (s >= parts) return;
    const int k0 = s * chunk, k1 = min(n_keys, k0 + chunk), last = k1 - 1;
    const KvSource src{p.table + (size_t)b * p.ld_table, p.n_pages, p.page_shift, p.nkv, kvh};
    if (tid == 0) s_bad = t.n_vis > kmax ? kmax : 0x7fffffff;
    const bool active = wrow < t.rows;
    Rows<HD> st;
    rows_init<HD>(st, p, t, kvh, wrow, lane);
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) arrived(st.qf[i]);
    const int r0 = wave * R;                         // this wave's rows of every tile: within one 16-key group, so on one page
    unsigned off[PIECES<HD, R>];
    piece_offsets<HD, R>(r0, lane, off);
    const unsigned smem_lds = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)LDS_PTR(smem));
    const int tiles = k1 > k0 ? (k1 - k0 + 63) >> 6 : 0;
    int pages = 0;                                   // page ids of this wave's rows of the next 64 tiles (waited for once in 4,096 keys)
    Codes<HD> c;
    auto issue = [&](int i) {                        // tile i
        if ((i & 63) == 0) {
            pages = src.row[min(k0 + 64 * (i + lane) + (r0 & ~15), last) >> p.page_shift];
            arrived(pages);
        }
        const int kb = k0 + 64 * i + (r0 & ~15), kc = min(kb, last & ~15);
        const size_t at = src.group(kc, __builtin_amdgcn_readlane(pages, i & 63));
        if constexpr (FP8) {
            codes_load<HD, false>(c, p, at, kb > last ? 0 : min(last - kc, 15), lane);
        } else {
            const unsigned dst = smem_lds + ((i & 1) * 2 * TILE + r0 * HD) * 2;
            if (kb + 15 <= last) {
                dma_rows<false>(p.kpool + at * (HD * 2), dst, off);
                dma_rows<false>(p.vpool + at * (HD * 2), dst + TILE * 2, off);
            } else {
                const int lim = kb > last ? 0 : last - kc;
                dma_rows_clamped<HD, R>(p.kpool + at * (HD * 2), dst, r0, lim, lane);
                dma_rows_clamped<HD, R>(p.vpool + at * (HD * 2), dst + TILE * 2, r0, lim, lane);
            }
        }
    };
    auto land = [&](int i) {                         // this wave's rows of tile i are in LDS
        if constexpr (FP8) {
            bf16_t* img = smem + (i & 1) * 2 * TILE;
            codes_store<HD, false>(c, img, img + TILE, r0, lane);
            if (i + 1 < tiles) issue(i + 1);         // (the codes go out a whole tile ahead)
        } else {
            dma_wait();
        }
    };
    if (tiles > 0) {
        issue(0);
        land(0);
    }
    __syncthreads();
    scan_pages<256>(p, src.row, k0, k1, &s_bad);
#pragma unroll 1
    for (int i = 0; i < tiles; ++i) {
        const bf16_t* sK = smem + (i & 1) * 2 * TILE;
        if (!FP8 && i + 1 < tiles) issue(i + 1);     // (its stage was read up to the last barrier)
        const int k = k0 + 64 * i;
        if (active) {
            if constexpr (KS == 2) {
                if (k + 32 * kg <= st.qmax) attend32<HD, false>(st, sK + 32 * HD * kg, sK + TILE + 32 * HD * kg, 0, k + 32 * kg, p.scale_log2, lane);
            } else {
#pragma unroll
                for (int sub = 0; sub < 2; ++sub)
                    if (k + 32 * sub <= st.qmax) attend32<HD, false>(st, sK, sK + TILE, sub, k + 32 * sub, p.scale_log2, lane);
            }
        }
        if (i + 1 < tiles) land(i + 1);
        __syncthreads();
    }
    if (tiles == 0) __syncthreads();                 // (s_bad)
    // ---- epilogue: this wave's 32 rows
    if (active && st.odd) add_odd<HD, FP8>(st, p, src, k0 + 32 * kg, 32 * KS, min(k1, st.qmax + 1), lane);
    const int r = lane & 31, h = lane >> 5, rows = min(32, t.rows - wrow);
    float l = st.l + __shfl_xor(st.l, 32, 64);
    if constexpr (KS == 2) {                         // the second half's waves hand their rows over, register by register, in the dead stages
        f32x4* o2 = reinterpret_cast<f32x4*>(smem_raw) + (wave & 1) * (HD * 32 / 4 + 64) + lane;
        if (kg == 1) {
#pragma unroll
            for (int d = 0; d < HD / 32; ++d)
#pragma unroll
                for (int g4 = 0; g4 < 4; ++g4)
                    o2[(d * 4 + g4) * 64] = f32x4{st.o[d][4 * g4], st.o[d][4 * g4 + 1], st.o[d][4 * g4 + 2], st.o[d][4 * g4 + 3]};
            o2[HD / 32 * 4 * 64] = f32x4{st.m, l, 0.f, 0.f};
        }
        __syncthreads();
        if (kg == 1) return;
        const f32x4 ml = o2[HD / 32 * 4 * 64];
        const float m = fmaxf(st.m, ml[0]), mu = m == -INFINITY ? 0.f : m;
        const float f0 = fast_exp2(st.m - mu), f1 = fast_exp2(ml[0] - mu);
        st.m = m;
        l = l * f0 + ml[1] * f1;
#pragma unroll
        for (int d = 0; d < HD / 32; ++d)
#pragma unroll
            for (int g4 = 0; g4 < 4; ++g4) {
                const f32x4 x = o2[(d * 4 + g4) * 64];
#pragma unroll
                for (int e = 0; e < 4; ++e)          // (a half that weighs nothing adds nothing: never 0 * inf)
                    st.o[d][4 * g4 + e] = (f0 == 0.f ? 0.f : st.o[d][4 * g4 + e] * f0) + (f1 == 0.f ? 0.f : x[e] * f1);
            }
    }
    if (!active) return;
    if (st.qi >= s_bad) l = __builtin_nanf("");
    if (parts > 1) {
        float* part = p.part + ((size_t)(f * p.nkv + kvh) * p.cut.parts + s) * (TROWS * (HD + 2));
        if (r < rows) {
            float* d = part + (size_t)(wrow + r) * HD;
#pragma unroll
            for (int dd = 0; dd < HD / 32; ++dd)
#pragma unroll
                for (int g4 = 0; g4 < 4; ++g4)
                    *reinterpret_cast<f32x4*>(d + 32 * dd + 8 * g4 + 4 * h) =
                        f32x4{st.o[dd][4 * g4], st.o[dd][4 * g4 + 1], st.o[dd][4 * g4 + 2], st.o[dd][4 * g4 + 3]};
            if (h == 0) *reinterpret_cast<f32x2*>(part + TROWS * HD + (wrow + r) * 2) = f32x2{st.m, l};
        }
        return;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    // rows through a slab of the wave's own in the dead stages: whole rows leave, 16 bytes a lane
    constexpr int PITCH = HD + 8, LPR = HD / 8, RPI = 64 / LPR;
    bf16_t* slab = smem + (KS == 2 ? 64 * HD * 2 + 1024 : 0) + wave * 32 * PITCH;      // (KS 2: behind the rows handed over)
#pragma unroll
    for (int d = 0; d < HD / 32; ++d)
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4)
            *reinterpret_cast<u32x2*>(slab + r * PITCH + 32 * d + 8 * g4 + 4 * h) =
                u32x2{pack_bf2(st.o[d][4 * g4] * inv, st.o[d][4 * g4 + 1] * inv), pack_bf2(st.o[d][4 * g4 + 2] * inv, st.o[d][4 * g4 + 3] * inv)};
    const int lr = lane / LPR, lc = (lane % LPR) * 8;
#pragma unroll
    for (int it = 0; it < 32 / RPI; ++it) {
        const int row = it * RPI + lr;
        const u32x4 x = *reinterpret_cast<const u32x4*>(slab + row * PITCH + lc);
        const int RR = t.row0 + wrow + row, tok = RR / p.G;
        if (row < rows) *reinterpret_cast<u32x4*>(p.out + (size_t)(t.tok0 + tok) * p.ldo + (kvh * p.G + RR - tok * p.G) * HD + lc) = x;
    }
}

// ---- joining parts: out = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s.  One wave a row, the lanes holding the parts' maxima and sums; part s is
// at at(s): HD outputs of the row, `ml` floats behind them its maximum and sum.
template <int HD, class At>
__device__ __forceinline__ void join_parts(int parts, At at, size_t ml, bf16_t* dst, int lane) {
    constexpr int C = HD / 64;
    float m = -INFINITY;
    for (int s = lane; s < parts; s += 64) m = fmaxf(m, at(s)[ml]);
    m = wave_max(m);
    const float mu = m == -INFINITY ? 0.f : m;
    float l = 0.f, a[C];
#pragma unroll
    for (int c = 0; c < C; ++c) a[c] = 0.f;
    for (int s0 = 0; s0 < parts; s0 += 64) {
        float f = 0.f;
        if (s0 + lane < parts) {
            const f32x2 v = *reinterpret_cast<const f32x2*>(at(s0 + lane) + ml);
            f = fast_exp2(v[0] - mu);
            l += v[1] * f;
        }
        const int n = min(parts - s0, 64);
        for (int i0 = 0; i0 < n; i0 += 8) {          // eight parts' loads in flight
            float x[8][C];
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int c = 0; c < C; ++c) x[i][c] = at(s0 + min(i0 + i, n - 1))[lane * C + c];
#pragma unroll
            for (int i = 0; i < 8; ++i) {            // (a part that weighs nothing adds nothing: never 0 * inf)
                const float fs = i0 + i < n ? __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), (i0 + i) & 63)) : 0.f;
#pragma unroll
                for (int c = 0; c < C; ++c) a[c] += fs == 0.f ? 0.f : x[i][c] * fs;
            }
        }
    }
    l = wave_sum(l);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (C == 2) *reinterpret_cast<unsigned*>(dst + lane * C) = pack_bf2(a[0] * inv, a[C - 1] * inv);
    else dst[lane] = f2bf(a[0] * inv);
}

// a block takes every gridDim.y-th group of four rows of a tile
template <int HD, int ROWS>
__global__ __launch_bounds__(256) void attn_paged_join_kernel(AttnPagedArgs p) {
    constexpr int STRIDE = ROWS * (HD + 2);
    const int lane = threadIdx.x & 63, tile = blockIdx.x / p.nkv, kvh = blockIdx.x % p.nkv;
    int b = tile / p.tps, ti = tile % p.tps;
    if constexpr (ROWS != RROWS) b = find_tile<ROWS>(p, load_seq<ROWS>(p, lane), tile, lane, &ti);
    if (b < 0) return;
    const Tile t = make_tile<ROWS>(p, b, ti);
    const int parts = cut_keys(p.cut, min(t.n_vis, p.max_pages << p.page_shift)).parts;
    if (parts == 1) return;                          // written by the attention itself
    const float* base = p.part + (size_t)(tile * p.nkv + kvh) * p.cut.parts * STRIDE;
    for (int row = blockIdx.y * 4 + (threadIdx.x >> 6); row < t.rows; row += gridDim.y * 4) {
        const int R = t.row0 + row, tok = R / p.G;
        join_parts<HD>(parts, [&](int s) { return base + (size_t)s * STRIDE + row * HD; }, (size_t)ROWS * HD + row * 2 - row * HD,
                       p.out + (size_t)(t.tok0 + tok) * p.ldo + (kvh * p.G + R - tok * p.G) * HD, lane);
    }
}

// ---- host: which kernel, and how many parts
struct Shape { int ks, tps, rows, class_bits; CutRule cut; long tiles, part_floats; };      // ks 0: the rows kernel
Shape pick_shape(int n_tok, int B, int nkv, int G, int HD, bool fp8, long max_keys, int max_q, int max_kv) {
    Shape sh{};
    const long mq = max_q > 0 && max_q < n_tok ? max_q : n_tok;
    const long keys = max_kv > 0 && max_kv < max_keys ? max_kv : max_keys;
    // 64-row tiles where 128-row ones would leave compute units without a second block: 512 tokens x 4 heads a kv head over 8,192 keys 137 -> 116 us, one
    // sequence of 64 over 20,000 52 -> 46 us; but 2,048 tokens over 16,384 keys 518 -> 560 us, 24 mixed sequences 103 -> 111 us
    sh.ks = mq * G <= RROWS ? 0 : ((long)n_tok * G / 128 + B) * nkv < 512 ? 2 : 1;
    const int rows = sh.ks ? 128 / sh.ks : RROWS;
    for (sh.class_bits = 0; sh.class_bits < 24 && (64L << sh.class_bits) <= keys; ++sh.class_bits) {}
    sh.tps = (int)(sh.ks ? (long)n_tok * G / rows + B : (mq * G + RROWS - 1) / RROWS);
    sh.rows = (int)(mq * G < rows ? mq * G : rows);      // rows of a tile, as far as the caller knows
    sh.tiles = sh.ks ? sh.tps : (long)sh.tps * B;
    const long units = sh.tiles * nkv, slots = sh.ks || (HD == 64 && fp8) ? 512 : 256;      // blocks that are resident at a time
    long parts = units > 0 ? slots / units : 1;
    parts = parts < 1 ? 1 : parts > MAX_PARTS ? MAX_PARTS : parts;
    const int round = 32 * rows_waves(HD, fp8);
    long few = 10240 / ((long)n_tok * G * nkv);
    few = few < 16 ? few : 16;                       // (the join takes 8 parts at a time)
    const long coarse = parts < keys / 512 ? parts : keys / 512;
    if (!sh.ks) sh.cut = CutRule{(int)parts, round, round == 256 ? 8 : 7, round - 1, 700};
    else if (few > coarse) sh.cut = CutRule{(int)(parts < few ? parts : few), 64, 7, 0, 400};
    else sh.cut = CutRule{(int)parts, 64, 9, 0, 0};
    sh.cut.parts = cut_keys(sh.cut, (int)keys).parts;
    sh.part_floats = sh.cut.parts > 1 ? units * sh.cut.parts * rows * (HD + 2) : 0;
    return sh;
}

template <int HD, int ROWS>
void launch_join(hipStream_t st, const AttnPagedArgs& p, const Shape& sh) {
    const long n = sh.tiles * p.nkv, most = (sh.rows + 3) / 4, y = (4095 + n) / n;      // a group of four rows a block, up to some 4,096 blocks
    hipLaunchKernelGGL((attn_paged_join_kernel<HD, ROWS>), dim3((unsigned)n, (unsigned)(y < most ? y : most)), dim3(256), 0, st, p);
}
template <int HD, bool FP8, int KS>
void launch_tile(hipStream_t st, const AttnPagedArgs& p, const Shape& sh) {
    // two stages; behind the loop the waves' rows (KS 2: 64 rows in fp32 with their maxima and sums, and the slabs)
    constexpr size_t stages = 2 * 2 * 64 * HD * 2, tail = KS == 2 ? 64 * HD * 4 + 2048 + 2 * 32 * (HD + 8) * 2 : 4 * 32 * (HD + 8) * 2, lds = stages > tail ? stages : tail;
    static const hipError_t once = hipFuncSetAttribute((const void*)attn_paged_tile_kernel<HD, FP8, KS>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    (void)once;
    const int units = p.nkv * sh.cut.parts;              // (the kernel's three ways to deal them to the 8 XCDs)
    const long blocks = 8 % units == 0 ? 8L * cdiv(sh.tps, 8 / units) : 8L * cdiv((long)units * sh.tps, 8);
    hipLaunchKernelGGL((attn_paged_tile_kernel<HD, FP8, KS>), dim3((unsigned)blocks), dim3(256), lds, st, p);
    if (sh.cut.parts > 1) launch_join<HD, 128 / KS>(st, p, sh);
}
template <int HD, bool FP8>
void launch(hipStream_t st, const AttnPagedArgs& p, const Shape& sh) {
    if (sh.ks == 2) return launch_tile<HD, FP8, 2>(st, p, sh);
    if (sh.ks == 1) return launch_tile<HD, FP8, 1>(st, p, sh);
    constexpr int NW = rows_waves(HD, FP8);
    const size_t lds = NW * RROWS * HD * 4 * (FP8 ? 1 : 2);           // images (e4m3: one buffer of 32 rows K | V in bf16), at the end the waves' rows in fp32
    static const hipError_t once = hipFuncSetAttribute((const void*)attn_paged_rows_kernel<HD, FP8>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    (void)once;
    hipLaunchKernelGGL((attn_paged_rows_kernel<HD, FP8>), dim3((unsigned)(sh.tiles * p.nkv * sh.cut.parts)), dim3(64 * NW), lds, st, p);
    if (sh.cut.parts > 1) launch_join<HD, RROWS>(st, p, sh);
}

int check_sizes(int n_tokens, int B, int n_heads, int n_kv_heads, int max_pages, int page_size) {
    MOLLY_CHECK(n_tokens >= 0 && B >= 0 && max_pages >= 0, "attn_paged: n_tokens=%d B=%d max_pages=%d", n_tokens, B, max_pages);
    MOLLY_CHECK(n_heads > 0 && n_kv_heads > 0 && n_heads % n_kv_heads == 0, "attn_paged: n_heads=%d not a multiple of n_kv_heads=%d", n_heads, n_kv_heads);
    MOLLY_CHECK((long)max_pages * page_size <= MAX_KEYS, "attn_paged: %d pages of %d keys a sequence, more than 2^31 - 2^15 - 1: keys are 32-bit", max_pages, page_size);
    MOLLY_CHECK((long)n_tokens * n_heads / n_kv_heads <= 0x1fffffffL && ((long)n_tokens * n_heads / 32 + 2L * B * n_kv_heads) * MAX_PARTS <= 0x7fffffffL,
                "attn_paged: n_tokens=%d x n_heads=%d, B=%d: more tiles than one call takes", n_tokens, n_heads, B);
    return 0;
}

}  // namespace

extern "C" int molly_attn_paged_workspace(int n_tokens, int B, int n_heads, int n_kv_heads, int head_dim, int page_size, int max_pages, int e4m3,
                                          int max_q, int max_kv) {
    if (n_tokens <= 0 || B <= 0 || page_size <= 0 || check_sizes(n_tokens, B, n_heads, n_kv_heads, max_pages, page_size)) return 0;
    const Shape sh = pick_shape(n_tokens, B, n_kv_heads, n_heads / n_kv_heads, head_dim, e4m3 != 0, (long)max_pages * page_size, max_q, max_kv);
    return sh.part_floats <= 0x7fffffffL ? (int)sh.part_floats : 0;
}

extern "C" int molly_attn_paged(void* stream, const void* q, void* out, const void* kpool, const void* vpool, const void* kscale_or_null,
                                const void* vscale_or_null, const int* block_table, const int* cu_q, const int* kv_len, int n_tokens, int B,
                                int n_pages, int page_size, int max_pages, int ld_table, int n_heads, int n_kv_heads, int head_dim, int ldq,
                                int ldo, float scale, int max_q, int max_kv, float* workspace, long workspace_floats) {
    MOLLY_ENTER();
    if (int rc = check_pool("attn_paged", kpool, vpool, kscale_or_null, vscale_or_null, n_pages, page_size, n_kv_heads, head_dim)) return rc;
    if (int rc = check_sizes(n_tokens, B, n_heads, n_kv_heads, max_pages, page_size)) return rc;
    MOLLY_CHECK(ld_table >= max_pages, "attn_paged: ld_table=%d for max_pages=%d", ld_table, max_pages);
    MOLLY_CHECK(scale > 0.f && scale < INFINITY, "attn_paged: scale=%g must be positive", (double)scale);
    if (n_tokens == 0 || B == 0) return 0;
    MOLLY_CHECK(q && out && cu_q && kv_len && (block_table || max_pages == 0), "attn_paged: q, out, block_table, cu_q, kv_len required");
    MOLLY_CHECK(aligned16(q) && aligned16(out) && ldq % 8 == 0 && ldo % 8 == 0 && ldq >= n_heads * head_dim && ldo >= n_heads * head_dim,
                "attn_paged: q / out rows must be 16-byte aligned and hold n_heads * head_dim values (ldq=%d ldo=%d)", ldq, ldo);
    MOLLY_CHECK(aligned16(workspace), "attn_paged: the workspace must be 16-byte aligned");
    AttnPagedArgs p{};
    p.q = (const bf16_t*)q; p.out = (bf16_t*)out; p.kpool = (const char*)kpool; p.vpool = (const char*)vpool;
    p.kscale = (const uint8_t*)kscale_or_null; p.vscale = (const uint8_t*)vscale_or_null;
    p.table = block_table; p.cu_q = cu_q; p.kv_len = kv_len; p.n_tok = n_tokens; p.B = B;
    p.n_pages = n_pages; p.page_shift = log2_exact(page_size); p.max_pages = max_pages; p.ld_table = ld_table;
    p.nh = n_heads; p.nkv = n_kv_heads; p.G = n_heads / n_kv_heads; p.ldq = ldq; p.ldo = ldo; p.scale_log2 = scale * LOG2E;
    Shape sh = pick_shape(n_tokens, B, n_kv_heads, p.G, head_dim, kscale_or_null != nullptr, (long)max_pages * page_size, max_q, max_kv);
    if (!workspace || workspace_floats < sh.part_floats) sh.cut.parts = 1;
    p.part = workspace; p.tps = sh.tps; p.cut = sh.cut; p.class_bits = sh.class_bits;
    hipStream_t st = (hipStream_t)stream;
    if (head_dim == 128) {
        if (kscale_or_null) launch<128, true>(st, p, sh);
        else launch<128, false>(st, p, sh);
    } else {
        if (kscale_or_null) launch<64, true>(st, p, sh);
        else launch<64, false>(st, p, sh);
    }
    MOLLY_LAUNCH_CHECK();
    return 0;
}
