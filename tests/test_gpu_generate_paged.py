"""GPU: generation over the paged caches — store, attention of chunks and single tokens, logit processors, draw, as a user's call runs them —
against the oracle's full re-forward (teacher forcing) and against the dense cache."""
import pytest
import torch

from conftest import tiny_state_dict
from test_gpu_generate import _left_padded_batch
from test_gpu_model import build_tiny

pytestmark = pytest.mark.gpu


def _session(m, batch, **kw):
    from molly_amd.generate import GenerationSession
    s = GenerationSession(m, max_new_tokens=6, **kw)
    return s, s.prefill(*batch)


@pytest.mark.parametrize("kv_cache,chunk,page", [("paged", None, 64), ("paged", 50, 16), ("paged", 1000, 256), ("paged", 7, 32)])
def test_paged_decode_logits_match_oracle_reforward(tiny_meta, kv_cache, chunk, page):
    """The bound is the dense path's own (tests/test_gpu_generate.py: 3e-2 of the largest logit, bf16 weights and activations)."""
    from oracle import molly_ref as R
    m = build_tiny(tiny_meta)
    ids, mask, omic, info = _left_padded_batch(tiny_meta)
    sess, logits = _session(m, (ids, mask, omic, info), kv_cache=kv_cache, prefill_chunk=chunk, page_size=page)
    c = tiny_meta["config"]
    llm, dna, prot = R.cfgs_from_meta(c)
    sd = tiny_state_dict(tiny_meta)
    batch = {"input_ids": ids, "attention_mask": mask, "omic_ids": omic, "omic_info_list": info}
    new = torch.empty(2, 0, dtype=torch.long)
    for step in range(5):
        ref = R.generate_last_logits(sd, llm, dna, prot, batch, new, {"dna_rna": c["K"], "protein": c["K"]})
        err = (logits.float().cpu() - ref).abs().max().item()
        assert err <= 3e-2 * ref.abs().max().item(), (step, err)
        nxt = ref.argmax(-1)
        new = torch.cat([new, nxt[:, None]], 1)
        logits = sess.step(nxt)


@pytest.mark.parametrize("chunk", [None, 40])
def test_e4m3_cache_stays_near_the_bf16_one(tiny_meta, chunk):
    """K and V of both layers are off by at most 2^-4 of themselves; what else the residual stream carries is the same: 2 * 2 * 2^-4 of the logits'
    norm.  The graph's replays give the eager steps' bits."""
    m = build_tiny(tiny_meta)
    batch = _left_padded_batch(tiny_meta)
    a, la = _session(m, batch, kv_cache="paged", prefill_chunk=chunk)
    b, lb = _session(m, batch, kv_cache="paged_e4m3", prefill_chunk=chunk)
    e, le = _session(m, batch, kv_cache="paged_e4m3", prefill_chunk=chunk, use_graph=False)
    assert b.paged.k.numel() == b.paged.k.view(torch.uint8).numel() and a.paged.k.element_size() == 2
    for step in range(5):
        assert torch.equal(lb, le)
        assert (lb - la).norm() <= 2 * 2 * 2.0 ** -4 * la.norm(), step
        nxt = la.argmax(-1)
        la, lb, le = a.step(nxt), b.step(nxt), e.step(nxt)


@pytest.mark.parametrize("kv_cache", ["paged", "paged_e4m3"])
def test_paged_reorder(tiny_meta, kv_cache):
    """Rows that change places go on as they would have where they were: the same tokens give the same logits, row for row."""
    m = build_tiny(tiny_meta)
    ids, mask, omic, info = _left_padded_batch(tiny_meta)
    ids, mask, omic = (t[1:2].repeat(3, *[1] * (t.dim() - 1)) for t in (ids, mask, omic))
    batch = (ids, mask, omic, [info[1]] * 3)
    a, la = _session(m, batch, kv_cache=kv_cache, page_size=16)
    b, _ = _session(m, batch, kv_cache=kv_cache, page_size=16)
    first = la.topk(3, -1).indices[0]
    la, lb = a.step(first), b.step(first)                         # three continuations
    perm = torch.tensor([2, 0, 2])
    b.reorder(perm)
    for tok in (5, 17, 400):
        la = a.step(torch.tensor([tok + 1, 0, tok]))
        lb = b.step(torch.tensor([tok, tok + 1, tok]))            # rows 0 and 2 were row 2, row 1 was row 0
        assert torch.equal(lb[0], lb[2])
        tol = 2.0 ** -6 * la.abs().max()                          # (other rows of a batch, other tiles: roundings of bf16 in two layers)
        assert (lb[0] - la[2]).abs().max() <= tol and (lb[1] - la[0]).abs().max() <= tol


def test_paged_reorder_into_a_row_with_fewer_pages_is_refused(tiny_meta):
    """A row keeps the pages its prompt was given; a longer sequence does not fit into fewer of them."""
    m = build_tiny(tiny_meta)
    batch = _left_padded_batch(tiny_meta)
    n = batch[1].sum(1).tolist()
    assert n[0] != n[1]
    small, large = (0, 1) if n[0] < n[1] else (1, 0)
    a, la = _session(m, batch, kv_cache="paged", page_size=16)
    assert len(set(a.own)) == 2
    first = la.argmax(-1)
    state = a.state.clone()
    with pytest.raises(ValueError):
        a.reorder(torch.tensor([large, large]))
    assert torch.equal(a.state, state)
    a.reorder(torch.tensor([small, small]))                       # the shorter one fits into both, and both say the same from here on
    for tok in (int(first[small]), 9):
        l = a.step(torch.tensor([tok, tok]))
        assert torch.equal(l[0], l[1]) and torch.isfinite(l).all()


def test_live_adapters_with_a_paged_cache(tiny_meta):
    """Un-merged adapters (plain projections + rank-r additions) go the same way: paged and dense caches agree to bf16 (the bound of the test above)."""
    from molly_amd.lora import LoraConfig
    from test_gpu_lora import _build, _randomize_B
    m = _build(tiny_meta, train_llm=False, lora=LoraConfig(r=8, lora_alpha=16, lora_dropout=0.0))
    _randomize_B(m)
    batch = _left_padded_batch(tiny_meta)
    a, la = _session(m, batch)
    b, lb = _session(m, batch, kv_cache="paged", prefill_chunk=64)
    for _ in range(3):
        assert (la - lb).abs().max() <= 3e-2 * la.abs().max()
        nxt = la.argmax(-1)
        la, lb = a.step(nxt), b.step(nxt)


def test_generate_with_paged_cache_and_processors(tiny_meta):
    m = build_tiny(tiny_meta)
    ids, mask, omic, info = _left_padded_batch(tiny_meta)
    gen = lambda **kw: m.generate(ids, mask, omic, info, do_sample=False, max_new_tokens=8, **kw)  # noqa: E731
    m.text_config.eos_token_id = None
    plain = gen(molly_kv_cache="paged", molly_prefill_chunk=33)
    assert plain.shape == (2, 8) and torch.equal(plain, gen(molly_kv_cache="paged", molly_prefill_chunk=33))
    # a bias that outweighs everything; a frequency penalty that forbids repeats; rows that may only say some tokens
    assert (gen(molly_kv_cache="paged_e4m3", molly_logit_bias={77: 1e6}) == 77).all()
    once = gen(molly_frequency_penalty=1e4, molly_logit_bias={77: 1e3})
    assert all(len(set(r.tolist())) == 8 for r in once) and (once[:, 0] == 77).all()
    b = torch.zeros(1024)
    b[5] = 1e6
    assert (gen(molly_logit_bias=b, molly_presence_penalty=1.0) == 5).all()
    seen = []

    def fn(row, so_far):
        seen.append((row, so_far.tolist()))
        return [10 * row + 1, 10 * row + 2 + len(so_far)]
    out = gen(prefix_allowed_tokens_fn=fn, molly_kv_cache="paged")
    for r in range(2):
        assert all(t in (10 * r + 1, 10 * r + 2 + j) for j, t in enumerate(out[r].tolist()))
    assert seen[-1] == (1, out[1, :7].tolist())
    g = torch.Generator(device="cuda").manual_seed(0)
    s = m.generate(ids, mask, omic, info, do_sample=True, top_k=20, temperature=0.8, top_p=0.95, repetition_penalty=1.1, max_new_tokens=4, generator=g,
                   molly_kv_cache="paged_e4m3", molly_presence_penalty=0.3, prefix_allowed_tokens_fn=lambda r, x: range(100, 200))
    assert s.shape == (2, 4) and bool(((s >= 100) & (s < 200)).all())
    # fewer allowed tokens than top_k, as a tensor of any device
    few = torch.tensor([700, 3], device="cuda")
    s = m.generate(ids, mask, omic, info, do_sample=True, top_k=20, temperature=0.8, top_p=1.0, max_new_tokens=8, prefix_allowed_tokens_fn=lambda r, x: few)
    assert s.shape == (2, 8) and bool(((s == 700) | (s == 3)).all())


def test_refusals(tiny_meta):
    from molly_amd.generate import GenerationSession
    m = build_tiny(tiny_meta)
    ids, mask, omic, info = _left_padded_batch(tiny_meta)
    with pytest.raises(ValueError):
        GenerationSession(m, 4, kv_cache="int4")
    with pytest.raises(ValueError):
        GenerationSession(m, 4, prefill_chunk=16)
    with pytest.raises(ValueError):
        GenerationSession(m, 4, kv_cache="paged", page_size=48).prefill(ids, mask, omic, info)
    with pytest.raises(NotImplementedError):
        m.generate(ids, mask, omic, info, do_sample=False, max_new_tokens=4, molly_num_beams=2, molly_kv_cache="paged")
    with pytest.raises(NotImplementedError):
        m.generate(ids, mask, omic, info, do_sample=False, max_new_tokens=4, molly_num_beams=2, molly_presence_penalty=0.5)
    for bad in (lambda r, x: [], lambda r, x: [5000]):
        with pytest.raises(ValueError):
            m.generate(ids, mask, omic, info, do_sample=False, max_new_tokens=4, prefix_allowed_tokens_fn=bad)
    with pytest.raises(ValueError):
        m.generate(ids, mask, omic, info, do_sample=False, max_new_tokens=4, molly_logit_bias={5000: 1.0})


@pytest.mark.parametrize("how", [dict(do_sample=False), dict(do_sample=True, top_k=20, temperature=0.8, top_p=0.95), dict(do_sample=True, temperature=0.8, top_p=1.0)])
def test_a_row_without_a_token_is_an_error(tiny_meta, how):
    """What is allowed is banned by another rule: the same error for greedy, fused and plain draws; no error for a row that has ended."""
    m = build_tiny(tiny_meta)
    ids, mask, omic, info = _left_padded_batch(tiny_meta)
    gen = lambda **kw: m.generate(ids, mask, omic, info, generator=torch.Generator(device="cuda").manual_seed(0), **how, **kw)  # noqa: E731
    m.text_config.eos_token_id = 9
    with pytest.raises(ValueError, match="no token is left in row 1"):
        gen(max_new_tokens=4, min_new_tokens=2, prefix_allowed_tokens_fn=lambda r, x: [9] if r else range(50, 90))
    with pytest.raises(ValueError, match="no token is left"):     # 1, 2, 1, then 2 would make a pair that was there
        gen(max_new_tokens=4, no_repeat_ngram_size=2, prefix_allowed_tokens_fn=lambda r, x: [1 + len(x) % 2])
    b = torch.full((m.text_config.vocab_size,), -float("inf"))
    with pytest.raises(ValueError, match="no token is left in row 0"):
        gen(max_new_tokens=4, molly_logit_bias=b)
    b[70] = 0.0
    assert (gen(max_new_tokens=3, molly_logit_bias=b) == 70).all()
    # row 0 ends with its first token; that it may then say nothing but what is banned is nobody's business
    out = gen(max_new_tokens=3, no_repeat_ngram_size=1, prefix_allowed_tokens_fn=lambda r, x: [60 + len(x)] if r else [9])
    assert out[0].tolist() == [9, m.text_config.pad_token_id, m.text_config.pad_token_id] and out[1].tolist() == [60, 61, 62]


def test_prefill_chunk_bounds_the_activations(tiny_meta):
    """A layer's rows are those of the chunk: xn, x2, xn2, x, out | qkv | qk | attn | gate and up, act.  (The rest is the same for both: weights, pages, embeddings; a chunk's
    attention may take a few MB of scratch: a fifth of the difference is left for it.)"""
    from molly_amd.synth import synth_batch
    m = build_tiny(tiny_meta)
    c = tiny_meta["config"]
    B, T, chunk = 2, 4000, 96
    b = synth_batch(B, T, [("protein", 64)], seed=3, text_vocab=1000, special_ids={k: tuple(v) for k, v in c["special_ids"].items()}, pad_id=1000)
    batch = (b["input_ids"], None, b["omic_ids"], b["omic_info_list"])
    t = c["text"]
    hd, nh, nkv = t["head_dim"], t["num_attention_heads"], t["num_key_value_heads"]
    row = 2 * (5 * t["hidden_size"] + (nh + 2 * nkv) * hd + (nh + nkv) * hd + nh * hd + 3 * t["intermediate_size"])

    def run(k):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        s, logits = _session(m, batch, kv_cache="paged", prefill_chunk=k)
        return torch.cuda.max_memory_allocated(), logits
    run(chunk)                                                    # (what the encoders and the GEMMs keep)
    cut, lc = run(chunk)
    whole, lw = run(None)
    assert whole - cut >= 0.8 * row * B * (T - chunk), (whole, cut, row)
    assert m._runtime().llm.cap == 0                              # the decoder's own buffers for the whole rectangle were not asked for
    assert (lw - lc).abs().max() <= 3e-2 * lw.abs().max()
    # the rows are kept for the next prefill, and a chunk's replace a whole prompt's
    e = m._runtime().llm
    kept = {k: v.data_ptr() for k, v in e.chunk.items()}
    run(None)
    assert {k: v.data_ptr() for k, v in e.chunk.items()} == kept and e.chunk_rows == B * T
    run(chunk)
    assert e.chunk_rows == B * chunk == e.chunk["x"].shape[0]
    run(chunk // 2)
    assert e.chunk_rows == B * (chunk // 2)


@pytest.mark.parametrize("chunk", [None, 50])
def test_paged_prefill_in_the_decoder_s_own_rows(tiny_meta, chunk):
    """Behind a dense session (or a training step) the rows are there already: none are allocated beside them, and the logits are the same bits; a larger batch gets rows
    of its own, and the decoder's next allocation gives them up."""
    batch = _left_padded_batch(tiny_meta)
    m = build_tiny(tiny_meta)
    own, want = _session(m, batch, kv_cache="paged", prefill_chunk=chunk)
    e = m._runtime().llm
    assert e.cap == 0 and e.chunk_rows > 0 and e.prompt is not None
    _session(m, batch)                                            # dense
    assert e.cap == batch[0].numel() and e.chunk_rows == 0 and e.chunk is None and e.prompt is None
    shared, got = _session(m, batch, kv_cache="paged", prefill_chunk=chunk)
    assert e.chunk is None and e.prompt is None and torch.equal(got, want)
    tok = want.argmax(-1)
    assert torch.equal(shared.step(tok), own.step(tok))
    twice = tuple(torch.cat([t, t]) for t in batch[:3]) + (batch[3] * 2,)
    _, both = _session(m, twice, kv_cache="paged")
    assert e.chunk_rows == 2 * int(batch[1].sum()) and e.prompt.shape[0] == twice[0].numel() and e.cap == batch[0].numel()
    assert (both[:2] - want).abs().max() <= 3e-2 * want.abs().max() and (both[2:] - want).abs().max() <= 3e-2 * want.abs().max()
