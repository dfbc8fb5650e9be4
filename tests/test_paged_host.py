"""CPU: the paged cache's bookkeeping, the processors' host parts, and the refusals that need no GPU."""
import pytest
import torch

from molly_amd import _lib, ops
from molly_amd.generate import _bias_row, _require_a_token, allowed_bits
from molly_amd.paged import PagedKVCache


def test_page_bookkeeping():
    c = PagedKVCache(2, 10, 2, 64, page_size=16, dtype="e4m3", device="cpu")
    assert c.k.shape == (2, 10, 2, 16, 64) and c.k.dtype == torch.float8_e4m3fn and c.kscale.shape == (2, 10, 2, 16)
    assert c.layer(1)["kpool"].data_ptr() == c.k[1].data_ptr() and set(c.layer(0)) == {"kpool", "vpool", "kscale", "vscale"}
    a, b = c.allocate(33), c.allocate(16)
    assert len(a) == 3 and len(b) == 1 and len(set(a + b)) == 4 and c.allocate(0) == []
    t = c.block_table([a, b, []])
    assert t.dtype == torch.int32 and t.tolist() == [a, b + [-1, -1], [-1, -1, -1]]
    with pytest.raises(RuntimeError):
        c.allocate(16 * 7)
    c.free(a)
    for bad in (a[:1], [b[0], b[0]], [10], [-1]):
        with pytest.raises(ValueError):
            c.free(bad)
    assert sorted(c.allocate(16 * 9) + b) == list(range(10))
    for kw in (dict(dtype="int8"), dict(head_dim=96), dict(page_size=8), dict(page_size=48), dict(n_pages=0)):
        with pytest.raises(ValueError):
            PagedKVCache(**{**dict(n_layers=1, n_pages=4, n_kv_heads=1, head_dim=64, device="cpu"), **kw})


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
def test_copy_pages_reads_before_it_writes(dtype):
    c = PagedKVCache(2, 4, 1, 64, page_size=16, dtype=dtype, device="cpu")
    raw = c.k.view(torch.uint8) if dtype == "e4m3" else c.k
    for p in range(4):
        raw[:, p] = p + 1
    c.copy_pages(torch.tensor([0, 1]), torch.tensor([1, 0]))
    assert raw[:, :, 0, 0, 0].tolist() == [[2, 1, 3, 4]] * 2


def test_allowed_bits_and_bias():
    V = 70
    m = allowed_bits([[0, 31, 32, 69], range(V), torch.tensor([63])], V, "cpu")
    assert m.dtype == torch.int32 and m.shape == (3, 3)
    bits = [[v for v in range(96) if (int(m[r, v // 32]) >> (v % 32)) & 1] for r in range(3)]
    assert bits == [[0, 31, 32, 69], list(range(V)), [63]]
    for bad in ([[]], [[V]], [[-1]]):
        with pytest.raises(ValueError):
            allowed_bits(bad, V, "cpu")
    b = _bias_row({3: 1.5, 69: -2}, V, "cpu")
    assert b.dtype == torch.float32 and b[3] == 1.5 and b[69] == -2 and int((b != 0).sum()) == 2
    assert torch.equal(_bias_row(b.double(), V, "cpu"), b)
    for bad in ({V: 1.0}, {-1: 1.0}, torch.zeros(V + 1)):
        with pytest.raises(ValueError):
            _bias_row(bad, V, "cpu")


def test_rows_without_a_token_are_refused():
    inf = float("inf")
    x = torch.zeros(3, 7)
    x[0, 1:], x[2, :] = -inf, -inf
    on = torch.ones(3, dtype=torch.bool)
    with pytest.raises(ValueError, match="row 2"):
        _require_a_token(x, on)
    assert torch.equal(_require_a_token(x[:2], on[:2]), x[:2])
    y = _require_a_token(x, torch.tensor([True, True, False]))    # a row that has ended needs none
    assert torch.equal(y[:2], x[:2]) and not y[2].any()
    x[2, 3] = float("nan")                                        # (not finite for another reason: not this refusal's)
    _require_a_token(x, on)


def test_wrappers_refuse_host_tensors():
    k = torch.zeros(4, 64, dtype=torch.bfloat16)
    pool = torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16)
    i = torch.zeros(4, dtype=torch.int32)
    for f in (lambda: ops.paged_kv_append(k, k, pool, pool, i), lambda: ops.paged_kv_read(pool, pool, i),
              lambda: ops.attn_paged(k, pool, pool, i[None], i[:2], i[:1], 1), lambda: ops.process_logits(torch.zeros(2, 5))):
        with pytest.raises(RuntimeError, match="GPU"):
            f()


def test_entry_points_refuse_bad_arguments():
    """Checked on the host, in front of any launch: callable without a GPU (addresses are never dereferenced)."""
    L = _lib.lib()
    P = 1 << 20

    def rejects(name, text, *args):
        assert L.fn[name](None, *args) != 0 and text in L.last_error(), (name, L.last_error())

    def append(k=P, v=P, q=None, qo=None, kp=P, ks=None, vs=None, slot=P, n=4, pages=4, page=16, nq=0, nkv=2, hd=64, ldq=0, ldk=128, ldv=128, ldqo=0,
               cos=None, sin=None, pos=None, n_pos=0):
        return k, v, q, qo, kp, P, ks, vs, slot, n, pages, page, nq, nkv, hd, ldq, ldk, ldv, ldqo, None, None, cos, sin, pos, n_pos, 1e-6
    for kw, text in ((dict(hd=96), "head_dim=96"), (dict(page=48), "page_size=48"), (dict(page=8), "page_size=8"), (dict(pages=0), "n_pages=0"),
                     (dict(pages=1 << 28), "32-bit"), (dict(ks=P), "exponents"), (dict(kp=P + 8), "16-byte"), (dict(k=None), "required"),
                     (dict(ldk=120), "ldk=120"), (dict(ldv=132), "ldv=132"), (dict(q=P), "go together"), (dict(cos=P, sin=P), "go together"),
                     (dict(q=P, qo=P, nq=2, ldq=64, ldqo=128), "ldq=64"), (dict(n=-1), "n_rows=-1")):
        rejects("molly_paged_kv_append", text, *append(**kw))
    assert L.fn["molly_paged_kv_append"](None, *append(n=0)) == 0
    for args, text in (((P, P, None, None, P, 4, 4, 16, 2, 64, P, P, 64, 128), "ldk=64"), ((P, P, None, None, None, 4, 4, 16, 2, 64, P, P, 128, 128), "required")):
        rejects("molly_paged_kv_read", text, *args)

    def attn(out=P, n=8, B=2, pages=4, page=16, maxp=3, ldt=3, nh=4, nkv=2, hd=64, ldq=256, ldo=256, scale=1.0, cu=P, ws=None, wsf=0):
        return P, out, P, P, None, None, P, cu, P, n, B, pages, page, maxp, ldt, nh, nkv, hd, ldq, ldo, scale, 0, 0, ws, wsf
    for kw, text in ((dict(nh=3), "multiple"), (dict(nkv=0), "n_kv_heads=0"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
                     (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale"), (dict(ldt=2), "ld_table"), (dict(ldq=128), "ldq=128"),
                     (dict(out=P + 2), "16-byte"), (dict(n=-1), "n_tokens=-1"), (dict(cu=None), "required"), (dict(maxp=1 << 28, ldt=1 << 28), "32-bit"),
                     (dict(n=1 << 30), "more tiles"), (dict(ws=P + 4, wsf=100), "workspace")):
        rejects("molly_attn_paged", text, *attn(**kw))
    assert L.fn["molly_attn_paged"](None, *attn(n=0)) == 0 and L.fn["molly_attn_paged"](None, *attn(B=0)) == 0
    assert ops.attn_paged_workspace(1, 1, 16, 8, 128, 64, 6, False) == 0 and ops.attn_paged_workspace(1, 1, 16, 8, 128, 64, 1000, False) > 0
    assert ops.attn_paged_workspace(-1, 1, 16, 8, 128, 64, 1000, False) == 0 and ops.attn_paged_workspace(1, 1, 15, 8, 128, 64, 1000, False) == 0

    def logits(x=P, out=P, rows=2, V=100, ldx=100, ldo=100, gen=None, n=0, ldg=0, rep=1.0, bias=None, ldb=0, allowed=None, ldm=0):
        return x, 0, out, rows, V, ldx, ldo, gen, None, n, ldg, rep, 0.0, 0.0, None, None, None, bias, ldb, allowed, ldm
    for kw, text in ((dict(V=0), "V=0"), (dict(ldx=99), "ld=99"), (dict(rows=70000), "rows=70000"), (dict(n=3), "3 generated"), (dict(gen=P, n=3, ldg=2), "ld=2"),
                     (dict(rep=0.0), "must be > 0"), (dict(bias=P, ldb=50), "ld_bias=50"), (dict(allowed=P, ldm=3), "ld_allowed=3"), (dict(x=None), "required")):
        rejects("molly_process_logits", text, *logits(**kw))
    assert L.fn["molly_process_logits"](None, *logits(rows=0)) == 0


def test_key_numbers_stay_in_32_bits():
    """The kernels count keys in ints and run ahead of the last one: the page lookup by 31 steps of 256 keys and 16, the end of the last part by what the parts
    were rounded up by.  At the largest table that is taken none of it passes 2^31 - 1; a larger one is refused."""
    L, P, most = _lib.lib(), 1 << 20, 0x7fffffff - 32768

    def call(page, pages):                                        # (no new tokens: nothing is launched, the sizes are checked)
        return L.fn["molly_attn_paged"](None, P, P, P, P, None, None, P, P, P, 0, 5, 4, page, pages, pages, 1, 1, 64, 64, 64, 1.0, 0, 0, None, 0)
    for page in (16, 32, 64, 128, 256):
        pages = most // page
        assert call(page, pages) == 0
        for p in (pages + 1, (0x7fffffff - 8192) // page, 0x7ffffe00 // page):
            assert call(page, p) != 0 and "32-bit" in L.last_error()
            assert ops.attn_paged_workspace(5, 5, 1, 1, 64, page, p, False, 1, 0) == 0
    keys = most // 16 * 16
    for parts in range(1, 65):
        for align, ahead in ((256, 31 * 256 + 16), (128, 31 * 128 + 16), (64, 63 * 64 + 48)):
            assert keys - 1 + ahead <= 0x7fffffff and keys + align <= 0x7fffffff
            part = ((keys - 1) // parts + align) // align * align                         # n / parts rounded up, to the next multiple
            assert -(-keys // part) * part <= 0x7fffffff


def test_no_rows_are_no_error():
    """An empty tensor has no address."""
    L, P = _lib.lib(), 1 << 20
    for q in (None, P):
        assert L.fn["molly_paged_kv_append"](None, None, None, q, q, P, P, None, None, None, 0, 4, 16, 2, 2, 64, 128, 128, 128, 128, P, P, P, P, None, 9, 1e-6) == 0
    assert L.fn["molly_paged_kv_read"](None, P, P, P, P, None, 0, 4, 16, 2, 64, None, None, 128, 128) == 0
    for page in (8, 48):                                          # (the pools are still looked at)
        assert L.fn["molly_paged_kv_read"](None, P, P, P, P, None, 0, 4, page, 2, 64, None, None, 128, 128) != 0


def test_positions_without_tables_are_refused():
    """Tables without rows have no address: they are not the same as none, the rows would go in unturned."""
    L, P = _lib.lib(), 1 << 20
    for cos, sin, pos, n_pos in ((None, None, P, 0), (None, None, P, 9), (P, P, P, 0), (P, None, P, 9), (None, P, None, 9)):
        assert L.fn["molly_paged_kv_append"](None, P, P, None, None, P, P, None, None, P, 4, 4, 16, 0, 2, 64, 0, 128, 128, 0, None, None, cos, sin, pos, n_pos, 1e-6) != 0
        assert "go together" in L.last_error()


def test_prefill_rows_behind_a_failed_allocation(monkeypatch):
    """Rows that could not be had are not taken for rows that are there; smaller ones are had afterwards."""
    from molly_amd.qwen3 import Qwen3Engine
    e = Qwen3Engine.__new__(Qwen3Engine)
    e.h, e.hd, e.nh, e.nkv, e.ff, e.nqkv, e.nqk, e.dev = 8, 4, 2, 1, 16, 16, 12, "cpu"
    e.cap, e.chunk_rows, e.chunk, e.prompt = 0, 0, None, None
    assert e.prefill_rows(8)["gu"].shape == (8, 32) and e.chunk_rows == 8 and e.prefill_rows(5) is e.chunk
    real = torch.empty

    def empty(rows, width, **kw):
        if rows > 100 and width > 16:
            raise torch.OutOfMemoryError("no")
        return real(rows, width, **kw)
    monkeypatch.setattr(torch, "empty", empty)
    with pytest.raises(torch.OutOfMemoryError):
        e.prefill_rows(1000)
    assert e.prefill_rows(20)["gu"].shape == (20, 32) and e.chunk_rows == 20
    assert e.prefill_rows(4, most=6)["act"].shape == (4, 16) and e.chunk_rows == 4
