"""Prefill + KV-cache decode for `OmicsOne.generate` (reference: src/model/omics_one.py:187-233 -> HF `generate` with
`inputs_embeds`, DynamicCache, sampling processors).  Prefill reuses the training forward kernels (flash attention over the
left-padded prompt, positions = cumsum(mask)-1 as HF does: HF:generation/utils.py:751-773) and writes every layer's
post-RoPE K and V into a token-major cache; each decode step is M = batch GEMMs + one `molly_attn_decode` per layer.
Token selection (temperature / top-k / top-p / repetition penalty, HF logits processors) runs on the [B, V] logits with
torch ops — a few KB of work per step, not a kernel target; presence / frequency penalties, biases and masks of allowed tokens are one kernel
(`molly_process_logits`).

kv_cache="paged" | "paged_e4m3" keeps K and V in pages (molly_amd.paged): no padding in the cache nor in the prompt's rows, the prompt in chunks of
`prefill_chunk` tokens a sequence, attention over the pages for chunks and decode steps alike (`molly_attn_paged`), e4m3 at half the bytes.
"""
from __future__ import annotations

from typing import Optional

import os

import torch

from . import ops

BF16 = torch.bfloat16


class GenerationSession:
    def __init__(self, model, max_new_tokens: int, use_graph: bool = None, kv_cache: str = "dense", prefill_chunk: Optional[int] = None,
                 page_size: int = 64):
        """kv_cache: 'dense' (one [B, T + max_new] rectangle a layer), 'paged' or 'paged_e4m3'; prefill_chunk: most prompt tokens of a sequence taken at a
        time (paged caches; None: the whole prompt): the prefill's activations are those of that many."""
        import os
        if kv_cache not in ("dense", "paged", "paged_e4m3"):
            raise ValueError(f"GenerationSession: kv_cache must be 'dense', 'paged' or 'paged_e4m3', got {kv_cache!r}")
        if prefill_chunk is not None and (kv_cache == "dense" or prefill_chunk < 1):
            raise ValueError("GenerationSession: prefill_chunk is a positive number of tokens, for the paged caches")
        self.kv_cache, self.prefill_chunk, self.page_size = kv_cache, prefill_chunk, page_size
        self.paged = None                               # PagedKVCache of a paged session
        self.use_graph = (os.environ.get("MOLLY_DECODE_GRAPH", "1") != "0") if use_graph is None else use_graph
        self.m = model
        self.rt = model._runtime()
        self.eng = self.rt.llm
        self.max_new = max_new_tokens

    # ---- prefill -------------------------------------------------------------------------------------------------
    @torch.no_grad()
    def prefill(self, input_ids, attention_mask, omic_ids, omic_info_list) -> torch.Tensor:
        """Returns the logits of the last prompt position [B, V] (fp32)."""
        with ops.use_gemm_context(self.rt.gemm_ctx):
            return self._prefill(input_ids, attention_mask, omic_ids, omic_info_list)

    def _prefill(self, input_ids, attention_mask, omic_ids, omic_info_list) -> torch.Tensor:
        m, rt, e = self.m, self.rt, self.eng
        B, T = input_ids.shape
        dev = rt.dev
        self.B, self.T = B, T
        self.Tmax = T + self.max_new
        lo, hi = m._kv_range(attention_mask, B, T, dev)
        mask = attention_mask.cpu().long() if attention_mask is not None else torch.ones(B, T, dtype=torch.long)
        pos = (mask.cumsum(1) - 1).clamp(min=0)                              # HF: position_ids = cumsum(mask)-1, pads -> 0/1
        self.lo = lo if lo is not None else torch.zeros(B, dtype=torch.int32, device=dev)
        self.n_valid = mask.sum(1).to(torch.int32).to(dev)                    # next position id per sample
        # the session's GEMM scratch is sized BEFORE its first GEMM (the launcher's split-K choices look at how much there is: a
        # workspace that grew between the prefill and a later one of the same shape could cut the second differently)
        ops.ensure_gemm_workspace(32 * 4 * max(B, 8) * max(2 * e.ff, e.nqkv), dev)
        st = m._stage(input_ids, None, None, omic_ids, omic_info_list, want_sort=False)
        if self.kv_cache != "dense":
            hs = e.prompt_rows(B * T)                                          # (the layers' rows are the chunks', not the rectangle's)
            m._embed_and_inject(st, False, out=hs)
            return self._prefill_paged(hs, mask, pos)
        hs, _ = m._embed_and_inject(st, False)
        e.reserve(B * T, B, T, training=False)
        # rope tables must cover prompt + generated positions
        from .qwen3 import rope_tables
        self.cos, self.sin = rope_tables(self.Tmax, e.hd, e.cfg.rope_theta, dev, e.rope_table_dtype)
        positions = pos.reshape(-1).to(torch.int32).to(dev)
        L, nkvd = e.L, e.nkv * e.hd
        self.kc = torch.zeros(L, B, self.Tmax, nkvd, dtype=BF16, device=dev)
        self.vc = torch.zeros(L, B, self.Tmax, nkvd, dtype=BF16, device=dev)
        rows = (torch.arange(B)[:, None] * self.Tmax + torch.arange(T)[None, :]).reshape(-1).to(torch.int32).to(dev)
        a = e.A[0]
        x = hs
        nq = e.nh * e.hd
        nk_ = e.nkv * e.hd
        if e.lora is not None:
            self.lt = torch.empty(B * T, e.lora.rp, dtype=BF16, device=dev)
        for i in range(L):
            w = e.W[i]
            ops.rmsnorm_fwd(x, w["ln1"], e.cfg.rms_norm_eps, out=a["xn"])
            ops.gemm_nt(a["xn"], w["qkv"], out=a["qkv"])
            self._lora(i, "q_proj", a["xn"], a["qkv"][:, :nq])
            self._lora(i, "k_proj", a["xn"], a["qkv"][:, nq:nq + nk_])
            self._lora(i, "v_proj", a["xn"], a["qkv"][:, nq + nk_:])
            # q/k-norm + rotary + the cache write of the whole prompt (row b * Tmax + t) in one launch
            ops.norm_rope_fwd(a["qkv"], a["qk"], e.nh, e.nkv, e.hd, T, w["qn"], w["kn"], self.cos, self.sin,
                              positions=positions, eps=e.cfg.rms_norm_eps,
                              kcache=self.kc[i].view(B * self.Tmax, nkvd), vcache=self.vc[i].view(B * self.Tmax, nkvd), slot=rows)
            ops.attn_fwd(a["qk"][:, :nq], a["qk"][:, nq:], a["qkv"][:, e.nqk:], B, T, e.nh, e.nkv, e.hd, e.hd ** -0.5, True,
                         lo, hi, out=a["attn"], lse=False)
            self._layer_tail(i, a, x, e.x_out)
            x = e.x_out
        last = x.view(B, T, e.h)[:, T - 1, :].contiguous()                    # left-padded prompts end at T-1
        self.cur_len = T
        self._alloc_step(B)
        return self._head(last)

    def _layer_tail(self, i, a, x, out):
        """From the attention's output to the layer's: o-projection + residual, norm, SwiGLU, down-projection + residual."""
        e = self.eng
        w = e.W[i]
        ops.gemm_nt(a["attn"], w["o"], out=a["x2"], res=x)
        self._lora(i, "o_proj", a["attn"], a["x2"])
        ops.rmsnorm_fwd(a["x2"], w["ln2"], e.cfg.rms_norm_eps, out=a["xn2"])
        if e.fused_swiglu:                                              # (no live adapters) SwiGLU in the gate|up GEMM's epilogue, as in training
            ops.gemm_gate_up_swiglu(a["xn2"], w["gu"], a["gu"], a["act"])
        else:
            ops.gemm_nt(a["xn2"], w["gu"], out=a["gu"])
            self._lora(i, "gate_proj", a["xn2"], a["gu"][:, :e.ff])
            self._lora(i, "up_proj", a["xn2"], a["gu"][:, e.ff:])
            ops.swiglu_fwd(a["gu"], out=a["act"])
        ops.gemm_nt(a["act"], w["down"], out=out, res=a["x2"])
        self._lora(i, "down_proj", a["act"], out)

    def _prefill_paged(self, hs, mask, pos) -> torch.Tensor:
        """The prompts' tokens without their padding, `prefill_chunk` of every sequence at a time, through the layers and into the pages.  The layers' activations
        are those of the largest chunk: only the embeddings (hs) have a row for every place of the prompts' rectangle."""
        from .paged import PagedKVCache
        from .qwen3 import rope_tables
        e, dev = self.eng, self.rt.dev
        B, T = mask.shape
        n_valid = mask.sum(1).tolist()
        if min(n_valid) == 0:
            raise ValueError("generate: a prompt without tokens")
        L, nq, nk = e.L, e.nh * e.hd, e.nkv * e.hd
        most = max(n_valid) + self.max_new
        self.cos, self.sin = rope_tables(most, e.hd, e.cfg.rope_theta, dev, e.rope_table_dtype)
        need = [-(-(n + self.max_new) // self.page_size) for n in n_valid]
        self.paged = PagedKVCache(L, sum(need), e.nkv, e.hd, self.page_size, "bf16" if self.kv_cache == "paged" else "e4m3", dev)
        self.need, self.own = need, list(need)                                # pages that the sequence in a row needs; that the row owns
        pages = [self.paged.allocate(n + self.max_new) for n in n_valid]
        self.table = self.paged.block_table(pages)
        # places of every sequence's tokens in the pools, [B, pages * page size] (behind the last page: none)
        at = self.table.cpu()
        places = torch.where(at[:, :, None] < 0, -1, at[:, :, None] * self.page_size + torch.arange(self.page_size, dtype=torch.int32)).flatten(1)
        self.places = places.to(dev)
        cols = [mask[b].nonzero().flatten() for b in range(B)]                # the columns that hold tokens
        chunk = self.prefill_chunk or max(n_valid)
        most_rows = sum(min(chunk, n) for n in n_valid)                       # (the first chunk's: no later one has more)
        if e.lora is not None:
            self.lt = torch.empty(max(most_rows, B), e.lora.rp, dtype=BF16, device=dev)
        scratch = e.prefill_rows(most_rows, None if self.prefill_chunk is None else B * chunk)
        last = torch.empty(B, e.h, dtype=BF16, device=dev)
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)        # noqa: E731
        for c0 in range(0, max(n_valid), chunk):
            new = [max(0, min(n - c0, chunk)) for n in n_valid]
            n = sum(new)
            rows = torch.cat([b * T + cols[b][c0:c0 + k] for b, k in enumerate(new)]).to(torch.int32).to(dev)
            positions = torch.cat([pos[b, cols[b][c0:c0 + k]] for b, k in enumerate(new)]).to(torch.int32).to(dev)
            slot = torch.cat([places[b, c0:c0 + k] for b, k in enumerate(new)]).to(torch.int32).to(dev)
            cu = [0]
            for k in new:
                cu.append(cu[-1] + k)
            cu_q, kv_len = i32(cu), i32([min(c0 + chunk, m) for m in n_valid])
            a = {k: scratch[k][:n] for k in ("xn", "qkv", "qk", "attn", "x2", "xn2", "gu", "act")}
            x, out = scratch["x"][:n], scratch["out"][:n]
            ops.copy_rows(hs, x, n, src_idx32=rows)
            for i in range(L):
                w = e.W[i]
                ops.rmsnorm_fwd(x, w["ln1"], e.cfg.rms_norm_eps, out=a["xn"])
                ops.gemm_nt(a["xn"], w["qkv"], out=a["qkv"])
                self._lora(i, "q_proj", a["xn"], a["qkv"][:, :nq])
                self._lora(i, "k_proj", a["xn"], a["qkv"][:, nq:nq + nk])
                self._lora(i, "v_proj", a["xn"], a["qkv"][:, nq + nk:])
                self._attend_paged(i, a["qkv"], a["qk"], a["attn"], slot, positions, cu_q, kv_len, max(new), min(c0 + chunk, max(n_valid)))
                self._layer_tail(i, a, x, out)
                x, out = out, x
            done = [b for b, m in enumerate(n_valid) if c0 < m <= c0 + chunk]  # their last token was in this chunk
            if done:
                ops.copy_rows(x, last, len(done), src_idx32=i32([cu[b + 1] - 1 for b in done]), dst_idx32=i32(done))
        self.cur_len = T
        self._alloc_step(B)
        self.hi.copy_(self.n_valid + 1)                                        # keys once the step's own token is in the pages
        self.cu_one = torch.arange(B + 1, dtype=torch.int32, device=dev)
        self.max_kv = most
        floats = ops.attn_paged_workspace(B, B, e.nh, e.nkv, e.hd, self.page_size, self.table.shape[1], self.kv_cache == "paged_e4m3", 1, most)
        self.dec_ws = torch.empty(max(floats, 4), dtype=torch.float32, device=dev)
        return self._head(last)

    def _attend_paged(self, i, qkv, qk, attn, slot, positions, cu_q, kv_len, max_q, max_kv, workspace=None):
        """One layer's q/k-norm, rotary and cache write in one launch, then attention over the pages."""
        e = self.eng
        w, nq = e.W[i], e.nh * e.hd
        pools = self.paged.layer(i)
        q = ops.paged_kv_append(qkv[:, nq:e.nqk], qkv[:, e.nqk:], slot=slot, q=qkv[:, :nq], q_out=qk[:, :nq], qw=w["qn"], kw=w["kn"], cos=self.cos,
                                sin=self.sin, positions=positions, eps=e.cfg.rms_norm_eps, **pools)
        ops.attn_paged(q, block_table=self.table, cu_q=cu_q, kv_len=kv_len, n_heads=e.nh, max_q=max_q, max_kv=max_kv, out=attn, workspace=workspace,
                       **pools)

    def _lora(self, i, mod, x, y):
        """live (un-merged) adapter: y += s * (x A^T) B^T, no dropout at inference (PEFT eval mode)."""
        lo = self.eng.lora
        if lo is None:
            return
        t = self.lt[:x.shape[0]]
        ops.gemm_nt(x, lo.A[i][mod], out=t)
        if lo.scale != 1.0:
            ops.scale_(t, lo.scale)
        ops.gemm_nt(t, lo.B[i][mod], out=y, accumulate=True)

    def _alloc_step(self, B):
        e, dev = self.eng, self.rt.dev
        z = lambda *s: torch.empty(*s, dtype=BF16, device=dev)
        self.s = dict(x=z(B, e.h), xn=z(B, e.h), qkv=z(B, e.nqkv), qk=z(B, e.nqk), attn=z(B, e.nh * e.hd), x2=z(B, e.h),
                      xn2=z(B, e.h), gu=z(B, 2 * e.ff), act=z(B, e.ff), hn=z(B, e.h))
        # static per-step state (device): token ids, position ids, cache slot and visible-key bound of the step's token
        self.tok = torch.zeros(B, dtype=torch.int64, device=dev)
        # (three rows of ONE tensor: the step advances them with one launch)
        self.state = torch.empty(3, B, dtype=torch.int32, device=dev)
        self.pos, self.slot, self.hi = self.state[0], self.state[1], self.state[2]
        self.pos.copy_(self.n_valid)                                           # position id = number of valid tokens so far
        self.slot.copy_(torch.arange(B, device=dev, dtype=torch.int32) * self.Tmax + self.cur_len)
        self.hi.fill_(self.cur_len + 1)
        self.logits = torch.empty(B, e.V, dtype=torch.float32, device=dev)
        self._graph, self._graph_ws, self._graph_ws_ptr, self._steps_done = None, None, 0, 0
        self.dec_ws = ops.attn_decode_workspace(B, e.nh, e.hd, dev)
        # decode GEMMs are M = B rows against whole weight matrices: the library splits K over the chip and needs slab space
        ops.ensure_gemm_workspace(32 * 4 * max(B, 8) * max(2 * e.ff, e.nqkv), dev)

    def _head(self, x):
        e = self.eng
        hn = ops.rmsnorm_fwd(x, e.norm_w, e.cfg.rms_norm_eps)
        return ops.gemm_nt(hn, e.head, out_dtype=torch.float32)

    # ---- one decode step ------------------------------------------------------------------------------------------
    def _step_body(self) -> torch.Tensor:
        """All device work of one step, reading/writing only the session's static tensors (tok, pos, slot, hi, caches), so
        the launch sequence is identical every step and can be replayed from a hipGraph."""
        e, s, B = self.eng, self.s, self.B
        nq, nkvd = e.nh * e.hd, e.nkv * e.hd
        ops.copy_rows(e.embed, s["x"], B, src_idx64=self.tok)
        x = s["x"]
        eps = e.cfg.rms_norm_eps
        # merged or no adapters: the launches behind a projection fold into it where the decode-row GEMM takes the shape (batch 17..64 on
        # the larger matrices) — residual + next RMSNorm behind o / down, SwiGLU behind gate|up — and the cache appends into norm + rope
        fuse = e.lora is None and os.environ.get("MOLLY_DECODE_FUSE", "1") != "0"
        H = x.shape[1]
        if self.paged is not None:                      # the places of the step's tokens
            self.slot.copy_(torch.gather(self.places, 1, self.pos.long()[:, None]).squeeze(1))
        f_qkv = self.paged is None and fuse and ops.gemm_rows_tail_supported(B, nq + 2 * nkvd, H, "qkv")
        # (the fused attention is built for groups of 1 / 2 / 4 / 8 query heads per KV head: other ratios take the plain path)
        f_att = (f_qkv and e.hd in (64, 128) and e.nh % e.nkv == 0 and e.nh // e.nkv in (1, 2, 4, 8)
                 and os.environ.get("MOLLY_DECODE_FUSE_ATTN", "1") != "0")
        f_o = fuse and ops.gemm_rows_tail_supported(B, H, nq, "norm")
        f_gu = fuse and ops.gemm_rows_tail_supported(B, 2 * e.ff, H, "swiglu")
        f_dn = fuse and ops.gemm_rows_tail_supported(B, H, e.ff, "norm")
        normed = False                                  # s["xn"] already holds ln1(x) of the layer about to run
        for i in range(e.L):
            w = e.W[i]
            if not normed:
                ops.rmsnorm_fwd(x, w["ln1"], eps, out=s["xn"])
            if self.paged is None:
                kc_i, vc_i = self.kc[i].view(B * self.Tmax, nkvd), self.vc[i].view(B * self.Tmax, nkvd)
            if f_att:                                   # projection as K-slice slabs; everything up to the attention output in ONE launch
                slabs, n_slabs = ops.gemm_rows_slabs(s["xn"], w["qkv"])
                ops.attn_decode_qkv(slabs, n_slabs, w["qn"], w["kn"], self.cos, self.sin, self.pos, eps, self.kc[i], self.vc[i], self.slot,
                                    s["attn"], self.lo, self.hi, B, self.Tmax, e.nh, e.nkv, e.hd, e.hd ** -0.5, kv_len_hint=self.Tmax,
                                    workspace=self.dec_ws)
            elif f_qkv:                                 # projection + q/k-norm + rotary + cache append: GEMM and one tail launch
                ops.gemm_rows_qkv(s["xn"], w["qkv"], s["qk"], e.nh, e.nkv, e.hd, w["qn"], w["kn"], self.cos, self.sin, self.pos, eps,
                                  kc_i, vc_i, self.slot)
            else:
                ops.gemm_nt(s["xn"], w["qkv"], out=s["qkv"])
                self._lora(i, "q_proj", s["xn"], s["qkv"][:, :nq])
                self._lora(i, "k_proj", s["xn"], s["qkv"][:, nq:nq + nkvd])
                self._lora(i, "v_proj", s["xn"], s["qkv"][:, nq + nkvd:])
                if self.paged is not None:
                    self._attend_paged(i, s["qkv"], s["qk"], s["attn"], self.slot, self.pos, self.cu_one, self.hi, 1, self.max_kv, self.dec_ws)
                elif fuse:
                    ops.norm_rope_fwd(s["qkv"], s["qk"], e.nh, e.nkv, e.hd, 1, w["qn"], w["kn"], self.cos, self.sin, positions=self.pos,
                                      eps=eps, kcache=kc_i, vcache=vc_i, slot=self.slot)
                else:
                    ops.norm_rope_fwd(s["qkv"], s["qk"], e.nh, e.nkv, e.hd, 1, w["qn"], w["kn"], self.cos, self.sin,
                                      positions=self.pos, eps=eps)
                    ops.copy_rows(s["qk"][:, nq:], kc_i, B, dst_idx32=self.slot)
                    ops.copy_rows(s["qkv"][:, e.nqk:], vc_i, B, dst_idx32=self.slot)
            if not f_att and self.paged is None:
                ops.attn_decode(s["qk"], self.kc[i], self.vc[i], s["attn"], self.lo, self.hi, B, self.Tmax, e.nh, e.nkv, e.hd,
                                e.hd ** -0.5, kv_len_hint=self.Tmax, workspace=self.dec_ws)
            if f_o:
                ops.gemm_rows_norm(s["attn"], w["o"], s["x2"], w["ln2"], eps, s["xn2"], res=x)
            else:
                ops.gemm_nt(s["attn"], w["o"], out=s["x2"], res=x)
                self._lora(i, "o_proj", s["attn"], s["x2"])
                ops.rmsnorm_fwd(s["x2"], w["ln2"], eps, out=s["xn2"])
            if f_gu:
                ops.gemm_rows_swiglu(s["xn2"], w["gu"], None, s["act"])          # (gate | up itself is not needed again)
            else:
                ops.gemm_nt(s["xn2"], w["gu"], out=s["gu"])
                self._lora(i, "gate_proj", s["xn2"], s["gu"][:, :e.ff])
                self._lora(i, "up_proj", s["xn2"], s["gu"][:, e.ff:])
                ops.swiglu_fwd(s["gu"], out=s["act"])
            if f_dn:                                    # ... + the NEXT block's input norm (the final norm behind the last block)
                last = i + 1 == e.L
                ops.gemm_rows_norm(s["act"], w["down"], s["x"], e.norm_w if last else e.W[i + 1]["ln1"], eps,
                                   s["hn"] if last else s["xn"], res=s["x2"])
                normed = True
            else:
                ops.gemm_nt(s["act"], w["down"], out=s["x"], res=s["x2"])
                self._lora(i, "down_proj", s["act"], s["x"])
            x = s["x"]
        if not normed:
            ops.rmsnorm_fwd(x, e.norm_w, eps, out=s["hn"])
        ops.gemm_nt(s["hn"], e.head, out=self.logits)
        # advance the per-sample position / cache slot / visible-key bound for the next step (device-side, graph-replayable)
        self.state += 1
        return self.logits

    @torch.no_grad()
    def reorder(self, rows: torch.Tensor):
        """Row i of the session becomes what row rows[i] was (beam search: the cache follows the beams that continue — HF's
        `DynamicCache.reorder_cache`, HF:cache_utils.py).  In place, so the captured decode graph's pointers stay valid; only the
        filled part of the caches moves."""
        rows = rows.to(self.rt.dev).long()
        if bool((rows == torch.arange(rows.numel(), device=rows.device)).all()):
            return                                      # every beam stays where it is: nothing moves
        n = self.cur_len
        if self.paged is not None:
            # what the rows hold of their pages moves; a row's own page list stays (the captured graph's tables)
            need = [self.need[r] for r in rows.tolist()]
            for i, (n, own) in enumerate(zip(need, self.own)):
                if n > own:
                    raise ValueError(f"reorder: row {i} owns {own} pages, the sequence that is to move there needs {n}")
            self.need = need
            used = -(-int(self.hi.max()) // self.page_size)
            src, dst = self.table[rows, :used], self.table[:, :used]
            moved = (src != dst) & (src >= 0) & (dst >= 0)
            self.paged.copy_pages(src[moved].long(), dst[moved].long())
            for t in (self.pos, self.hi, self.lo, self.n_valid):
                t.copy_(t.index_select(0, rows))
            return
        # layer by layer: the temporary is one layer's filled cache (B x n x kv width), not all L of them — at Qwen3-8B with a 3 k-token
        # prompt and B * num_beams rows the whole-cache gather was a multi-GB allocation beside a cache sized for 3,072 new tokens
        for i in range(self.kc.shape[0]):
            self.kc[i, :, :n] = self.kc[i, :, :n].index_select(0, rows)
            self.vc[i, :, :n] = self.vc[i, :, :n].index_select(0, rows)
        for t in (self.pos, self.hi, self.lo, self.n_valid):
            t.copy_(t.index_select(0, rows))
        # (slot = row * Tmax + cur_len belongs to the ROW, not to the beam that moved into it)

    @torch.no_grad()
    def step(self, token_ids: torch.Tensor) -> torch.Tensor:
        """token_ids int64 [B] (the tokens chosen from the previous logits).  Returns next-token logits [B, V] fp32 (a
        buffer that the next step overwrites).  The first step runs eagerly (it also sizes workspaces and sets kernel
        attributes), the second is captured into a hipGraph, later steps replay it: the step's launches (7 per layer with merged adapters: round 4) become one."""
        assert self.cur_len < self.Tmax, "generation budget exhausted"
        with ops.use_gemm_context(self.rt.gemm_ctx):
            return self._step(token_ids)

    def _step(self, token_ids: torch.Tensor) -> torch.Tensor:
        self.tok.copy_(token_ids.to(self.rt.dev), non_blocking=True)
        self.cur_len += 1
        self._steps_done += 1
        if not self.use_graph or self._steps_done == 1:
            return self._step_body()
        # The captured launches carry the context's scratch pointers (split-K slabs, the decode-row tails' slabs, stream-K and
        # dynamic-fetch counters).  Another session or a training reserve() on the same model may have grown — i.e. replaced — that
        # scratch since the capture: the graph then keeps its own reference to the tensor it was captured with (`_graph_ws`, so a
        # replay in flight never reads freed memory) and is dropped and captured again before the next replay.
        ws = self.rt.gemm_ctx.ws
        if self._graph is not None and (ws is None or ws.data_ptr() != self._graph_ws_ptr):
            self._graph = None
        if self._graph is None:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                self._step_body()
            assert self.rt.gemm_ctx.ws is ws, "the GEMM scratch was replaced during graph capture"
            self._graph, self._graph_ws, self._graph_ws_ptr = g, ws, (ws.data_ptr() if ws is not None else 0)
            # capture does not execute: fall through to the replay
        self._graph.replay()
        return self.logits


def _process_logits(logits, generated, temperature, top_k, top_p, repetition_penalty):
    """HF logits processors in HF's order: repetition penalty, temperature, top-k, top-p."""
    if repetition_penalty and repetition_penalty != 1.0 and generated.shape[1] > 0:
        score = torch.gather(logits, 1, generated)
        score = torch.where(score < 0, score * repetition_penalty, score / repetition_penalty)
        logits = logits.scatter(1, generated, score)
    if temperature and temperature != 1.0:
        logits = logits / temperature
    if top_k:
        kth = torch.topk(logits, min(top_k, logits.shape[-1]))[0][..., -1, None]
        logits = logits.masked_fill(logits < kth, float("-inf"))
    if top_p is not None and top_p < 1.0:
        sl, si = torch.sort(logits, descending=False)
        cp = sl.softmax(-1).cumsum(-1)
        remove = cp <= (1 - top_p)
        remove[..., -1:] = False
        logits = logits.masked_fill(remove.scatter(1, si, remove), float("-inf"))
    return logits


class NoRepeatNGram:
    """HF `NoRepeatNGramLogitsProcessor` (HF:generation/logits_process.py, `_calc_banned_ngram_tokens`): a token is banned when it
    would complete an n-gram that already occurs in the row's generated sequence.  HF rebuilds the n-gram table of every row at every
    step; here it is kept per row and extended by the one n-gram each new token completes.  The reference passes
    `no_repeat_ngram_size` through to HF generate (src/model/omics_one.py:199-200, 227); with `inputs_embeds` and no `input_ids` HF's
    `input_ids` hold the GENERATED tokens only, so the prompt never contributes n-grams."""

    def __init__(self, n: int, batch: int):
        assert n >= 1
        self.n = n
        self.table = [dict() for _ in range(batch)]            # row -> {(n-1)-gram prefix: set of tokens that followed it}
        self.hist = [[] for _ in range(batch)]

    def push(self, tokens):
        """tokens: the B tokens just appended (python ints)."""
        n = self.n
        for b, t in enumerate(tokens):
            h = self.hist[b]
            h.append(int(t))
            if len(h) >= n:
                self.table[b].setdefault(tuple(h[len(h) - n:len(h) - 1]), set()).add(h[-1])

    def banned(self):
        """per row: the tokens that must not come next (HF: none while fewer than n - 1... tokens exist: cur_len + 1 < n)."""
        n, out = self.n, []
        for b, h in enumerate(self.hist):
            if len(h) + 1 < n:
                out.append(())
            else:
                out.append(tuple(self.table[b].get(tuple(h[len(h) + 1 - n:]), ())))
        return out

    def apply(self, logits: torch.Tensor) -> torch.Tensor:
        rows, cols = [], []
        for b, toks in enumerate(self.banned()):
            rows += [b] * len(toks)
            cols += list(toks)
        if rows:
            logits = logits.clone()
            logits[torch.tensor(rows, device=logits.device), torch.tensor(cols, device=logits.device)] = float("-inf")
        return logits


def allowed_bits(allowed, vocab: int, device) -> torch.Tensor:
    """int32 [rows, ceil(vocab / 32)] for ops.process_logits: bit v % 32 of word v // 32 set for every v in allowed[row]."""
    rows, words = len(allowed), (vocab + 31) // 32
    on = torch.zeros(rows, words * 32, dtype=torch.bool)
    for r, ids in enumerate(allowed):
        ids = torch.as_tensor(ids, dtype=torch.int64).reshape(-1).cpu()
        if ids.numel() == 0:
            raise ValueError(f"generate: no token is allowed in row {r}")
        if int(ids.min()) < 0 or int(ids.max()) >= vocab:
            raise ValueError(f"generate: an allowed token of row {r} lies outside the vocabulary of {vocab}")
        on[r, ids] = True
    w = (on.view(rows, words, 32).long() << torch.arange(32)).sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32).to(device)


def _require_a_token(logits, unfinished):
    """-> logits [rows, V], with an error where an unfinished row has no token left (every score -inf).  A row that has ended says its pad token whatever
    its scores are: without one they become zeros, for the draw that is not used."""
    dead = logits.amax(1) == float("-inf")
    if not bool(dead.any()):
        return logits
    if bool((dead & unfinished).any()):
        raise ValueError(f"generate: no token is left in row {int((dead & unfinished).nonzero()[0])}: what is allowed is banned by min_new_tokens, "
                         "no_repeat_ngram_size or logit_bias")
    return logits.masked_fill(dead[:, None], 0.0)


def _bias_row(logit_bias, vocab: int, device) -> torch.Tensor:
    """{token: bias} or a [vocab] tensor -> fp32 [vocab]"""
    if torch.is_tensor(logit_bias):
        if tuple(logit_bias.shape) != (vocab,):
            raise ValueError(f"generate: logit_bias must have one value for each of {vocab} tokens, got {tuple(logit_bias.shape)}")
        return logit_bias.to(device=device, dtype=torch.float32).contiguous()
    b = torch.zeros(vocab)
    for t, x in logit_bias.items():
        if not 0 <= int(t) < vocab:
            raise ValueError(f"generate: logit_bias of token {t} outside the vocabulary of {vocab}")
        b[int(t)] = float(x)
    return b.to(device)


@torch.no_grad()
def generate(model, input_ids, attention_mask=None, omic_ids=None, omic_info_list=None, max_new_tokens=3072, do_sample=True,
             temperature=0.8, top_p=0.95, top_k=None, repetition_penalty=None, pad_token_id=None, eos_token_id=None,
             generator: Optional[torch.Generator] = None, no_repeat_ngram_size: Optional[int] = None, num_beams: int = 1,
             length_penalty: float = 1.0, early_stopping=False, min_new_tokens: int = 0, kv_cache: str = "dense",
             prefill_chunk: Optional[int] = None, presence_penalty: float = 0.0, frequency_penalty: float = 0.0, logit_bias=None,
             prefix_allowed_tokens_fn=None) -> torch.Tensor:
    """Returns the NEW tokens only, int64 [B, n_new] (what HF returns when called with inputs_embeds and no input_ids).
    min_new_tokens: HF's MinNewTokensLengthLogitsProcessor — the eos scores are -inf while fewer new tokens than that exist (it runs among
    the processors, in front of the warpers).
    kv_cache / prefill_chunk: GenerationSession.  presence_penalty, frequency_penalty (subtracted once / once an occurrence for every token generated
    so far), logit_bias ({token: added} or [V]) and prefix_allowed_tokens_fn(row, generated ids) -> allowed tokens (HF's) go, with the repetition
    penalty, through one kernel in front of the warpers (ops.process_logits).  A row that has not ended and of which they, the n-gram rule and
    min_new_tokens leave no token is a ValueError."""
    extra = bool(presence_penalty or frequency_penalty or logit_bias is not None or prefix_allowed_tokens_fn is not None)
    if num_beams and num_beams > 1:
        if min_new_tokens:
            raise NotImplementedError("generate: min_new_tokens together with molly_num_beams > 1 is not built")
        if extra or kv_cache != "dense" or prefill_chunk is not None:
            raise NotImplementedError("generate: the paged caches, presence / frequency penalties, biases and allowed tokens together with "
                                      "molly_num_beams > 1 are not built")
        return _generate_beams(model, input_ids, attention_mask, omic_ids, omic_info_list, max_new_tokens, do_sample, repetition_penalty,
                               pad_token_id, eos_token_id, no_repeat_ngram_size, int(num_beams), length_penalty, early_stopping,
                               temperature, top_k, top_p, generator)
    sess = GenerationSession(model, max_new_tokens, kv_cache=kv_cache, prefill_chunk=prefill_chunk)
    logits = sess.prefill(input_ids, attention_mask, omic_ids, omic_info_list)
    B = input_ids.shape[0]
    dev = logits.device
    bias = None if logit_bias is None else _bias_row(logit_bias, logits.shape[1], dev)
    # what can take a row's last token away (penalties and finite biases cannot)
    bans = prefix_allowed_tokens_fn is not None or (bias is not None and bool((bias == float("-inf")).any()))
    eos = None if eos_token_id is None else torch.as_tensor(eos_token_id, device=dev).reshape(-1)
    pad = pad_token_id if pad_token_id is not None else (int(eos[0]) if eos is not None else 0)
    out = torch.empty(B, 0, dtype=torch.int64, device=dev)
    unfinished = torch.ones(B, dtype=torch.bool, device=dev)
    # sampling with a top-k (the reference's inference settings: top_k 20) runs in ONE kernel per step: penalty, temperature,
    # top-k, top-p, softmax and the draw (csrc/sampling.hip).  Without a top-k the torch restatement below is used.
    fused = bool(do_sample and top_k and 1 <= top_k <= 1024 and logits.dtype == torch.float32)
    # The Philox stream is keyed by (seed, step, row).  The seed is DRAWN from the generator (or torch's global one), so it is
    # reproducible under manual_seed and — like torch.multinomial in the reference path — advances the generator's state:
    # two calls with one generator (inference.py passes one for the whole dataset) get independent samples.
    seed = 0
    if fused:
        gdev = generator.device if generator is not None else "cpu"
        seed = int(torch.randint(0, 1 << 62, (1,), generator=generator, device=gdev, dtype=torch.int64).item())
    ngram = NoRepeatNGram(int(no_repeat_ngram_size), B) if no_repeat_ngram_size else None
    for it in range(max_new_tokens):
        if ngram is not None:
            # HF's order: repetition penalty, then the n-gram ban, then the warpers; a banned logit is -inf and the penalty leaves -inf
            # where it is, so banning first gives the same scores
            logits = ngram.apply(logits)
        if min_new_tokens and it < min_new_tokens and eos is not None:
            logits = logits.clone()
            logits[:, eos] = float("-inf")
        penalty = repetition_penalty
        if extra:
            allowed = None
            if prefix_allowed_tokens_fn is not None:
                so_far = out.cpu()
                allowed = allowed_bits([prefix_allowed_tokens_fn(b, so_far[b]) for b in range(B)], logits.shape[1], dev)
            logits = ops.process_logits(logits, generated=out if out.shape[1] else None, repetition_penalty=float(repetition_penalty or 1.0),
                                        presence_penalty=float(presence_penalty), frequency_penalty=float(frequency_penalty), bias=bias, allowed=allowed)
            penalty = None                                  # (done)
            if bans:
                logits = _require_a_token(logits, unfinished)
        if fused:
            nxt = ops.sample_logits(logits, out if out.shape[1] else None, penalty, temperature, top_k, top_p,
                                    seed, it)
        else:
            lg = _process_logits(logits, out, temperature if do_sample else None, top_k if do_sample else None,
                                 top_p if do_sample else None, penalty)
            if do_sample:
                nxt = torch.multinomial(lg.softmax(-1), 1, generator=generator).squeeze(1)
            else:
                nxt = ops.argmax(lg) if lg.dtype == torch.float32 else lg.argmax(-1)
        nxt = torch.where(unfinished, nxt, torch.full_like(nxt, pad))
        out = torch.cat([out, nxt[:, None]], 1)
        if ngram is not None:
            ngram.push(nxt.tolist())
        if eos is not None:
            unfinished = unfinished & ~torch.isin(nxt, eos)
            if not bool(unfinished.any()):
                break
        if out.shape[1] == max_new_tokens:
            break
        logits = sess.step(nxt)
    return out


def _generate_beams(model, input_ids, attention_mask, omic_ids, omic_info_list, max_new_tokens, do_sample, repetition_penalty, pad_token_id,
                    eos_token_id, no_repeat_ngram_size, num_beams, length_penalty, early_stopping, temperature=None, top_k=None, top_p=None,
                    generator=None):
    """Beam search, this build's extension (`OmicsOne.generate(molly_num_beams=N)`; the reference's own `num_beams` parameter is dropped
    by its generate, src/model/omics_one.py:220-232, and is ignored here too).  Procedure = HF `_beam_search` (molly_amd/beam.py): the prompt rows
    repeated num_beams times through one prefill, then molly_amd.beam.beam_search over the decode session (logits from
    `GenerationSession.step`, the KV cache gathered by `GenerationSession.reorder`).  With do_sample=True this is HF's beam sampling:
    the warpers (temperature, top-k, top-p) act on the log-probabilities and the continuations are drawn by torch.multinomial — the
    same procedure; the random stream is the caller's generator on the GPU, so draws differ from a CPU run of HF."""
    from .beam import beam_search
    B, nb = input_ids.shape[0], num_beams
    rep = lambda t: None if t is None else t.repeat_interleave(nb, 0)
    rep_list = lambda l: None if l is None else [x for x in l for _ in range(nb)]
    omic_rep = rep(omic_ids) if torch.is_tensor(omic_ids) else rep_list(omic_ids)
    sess = GenerationSession(model, max_new_tokens)
    logits = sess.prefill(rep(input_ids), rep(attention_mask), omic_rep, rep_list(omic_info_list))
    eos = None if eos_token_id is None else [int(x) for x in torch.as_tensor(eos_token_id).reshape(-1).tolist()]

    def processors(generated, lp):
        # HF applies the processors to the log-probabilities in beam mode: repetition penalty, then the n-gram ban
        if repetition_penalty and repetition_penalty != 1.0 and generated.shape[1] > 0:
            lp = _process_logits(lp, generated, None, None, None, repetition_penalty)
        if no_repeat_ngram_size and generated.shape[1] + 1 >= no_repeat_ngram_size:
            ng = NoRepeatNGram(int(no_repeat_ngram_size), generated.shape[0])       # rows change beams every step: rebuilt, as HF does
            for t in range(generated.shape[1]):
                ng.push(generated[:, t].tolist())
            lp = ng.apply(lp)
        if do_sample:
            lp = _process_logits(lp, generated, temperature, top_k, top_p, None)
        return lp
    use_proc = (repetition_penalty and repetition_penalty != 1.0) or no_repeat_ngram_size or do_sample
    gen = generator
    if do_sample and generator is not None and generator.device.type != logits.device.type:
        gen = torch.Generator(device=logits.device).manual_seed(int(torch.randint(0, 1 << 62, (1,), generator=generator).item()))
    return beam_search(logits, sess.step, sess.reorder, B, nb, max_new_tokens, eos, pad_token_id, length_penalty, early_stopping,
                       processors if use_proc else None, do_sample=bool(do_sample), generator=gen)
