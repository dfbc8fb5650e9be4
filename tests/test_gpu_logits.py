"""process_logits against its definition in 64 bits.  The result is float32: a handful of float32 operations on magnitudes below 64 and the one
rounding, so at most 2^-24 * 8 of the magnitudes summed."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ops():
    from molly_amd import ops as o
    return o


def reference(x, gen=None, n_gen=None, rep=1.0, pres=0.0, freq=0.0, bias=None, allowed=None):
    x = x.double().cpu().clone()
    rows, V = x.shape
    at = lambda p, r: float(p[r]) if torch.is_tensor(p) else float(p)  # noqa: E731
    for r in range(rows):
        if gen is not None:
            n = gen.shape[1] if n_gen is None else min(max(int(n_gen[r]), 0), gen.shape[1])
            ids = gen[r, :n].cpu()
            ids, c = torch.unique(ids[(ids >= 0) & (ids < V)], return_counts=True)
            y = x[r, ids]
            x[r, ids] = torch.where(y < 0, y * at(rep, r), y / at(rep, r)) - at(pres, r) - at(freq, r) * c
        if bias is not None:
            x[r] += (bias if bias.dim() == 1 else bias[r]).double().cpu()
        if allowed is not None:
            w = (allowed if allowed.dim() == 1 else allowed[r]).cpu().long()
            bits = torch.stack([(w >> j) & 1 for j in range(32)], 1).flatten()[:V]
            x[r, bits == 0] = -math.inf
    return x


def same(got, want):
    got = got.double().cpu()
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got[~fin & ~torch.isnan(want)], want[~fin & ~torch.isnan(want)])
    assert ((got - want).abs()[fin] <= 2.0 ** -21 * (want.abs()[fin] + 64)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,V,n", [(1, 1, 3), (1, 151936, 40), (3, 257, 0), (5, 4097, 9), (4, 8191, 5000), (2, 50257, 12000), (64, 1000, 33), (33, 32, 1)])
@pytest.mark.parametrize("per_row,bias,mask", [(False, None, None), (True, "one", "rows"), (True, "rows", "one"), (False, None, "rows")])
def test_process_logits(rows, V, n, dtype, per_row, bias, mask):
    g = torch.Generator(device=DEV).manual_seed(V + n)
    x = (6 * torch.randn(rows, V, generator=g, device=DEV)).to(dtype)
    ids = (torch.rand(rows, n, generator=g, device=DEV) ** 3 * V).long() if n else None
    n_gen = torch.randint(0, n + 1, (rows,), generator=g, device=DEV, dtype=torch.int32) if n else None
    pen = (1.3, 0.5, 0.1)
    if per_row:
        u = torch.rand(3, rows, generator=g, device=DEV)
        pen = (0.7 + u[0], u[1] - 0.5, 0.2 * u[2])
    b = None if bias is None else torch.randn(*((V,) if bias == "one" else (rows, V)), generator=g, device=DEV)
    W = (V + 31) // 32
    m = None if mask is None else torch.randint(-2 ** 31, 2 ** 31, (W,) if mask == "one" else (rows, W), generator=g, device=DEV).to(torch.int32)
    out = ops().process_logits(x, generated=ids, n_generated=n_gen, repetition_penalty=pen[0], presence_penalty=pen[1], frequency_penalty=pen[2], bias=b,
                               allowed=m)
    want = reference(x, ids, n_gen, *pen, b, m)
    same(out, want)
    if dtype == torch.float32:                                    # in place, the same bits
        y = x.clone()
        got = ops().process_logits(y, generated=ids, n_generated=n_gen, repetition_penalty=pen[0], presence_penalty=pen[1], frequency_penalty=pen[2],
                                   bias=b, allowed=m, out=y)
        assert got is y and torch.equal(y, out)


def test_edges():
    """Ids outside the vocabulary, the whole history one token, lengths out of range, values that are not finite, a mask that allows nothing."""
    V = 300
    x = torch.randn(4, V, device=DEV)
    x[0, 5], x[1, 5], x[2, 5], x[3, 5] = math.inf, -math.inf, math.nan, -0.0
    ids = torch.full((4, 700), 5, dtype=torch.int64, device=DEV)
    ids[:, 100:] = torch.tensor([-1, V, V + 2 ** 32 + 7, -2 ** 40], device=DEV)[:, None]
    n_gen = torch.tensor([700, 900, 3, -2], dtype=torch.int32, device=DEV)
    m = torch.full((4, 10), -1, dtype=torch.int32, device=DEV)
    m[1] = 0
    out = ops().process_logits(x, generated=ids, n_generated=n_gen, repetition_penalty=2.0, presence_penalty=0.25, frequency_penalty=0.5, allowed=m)
    same(out, reference(x, ids, n_gen, 2.0, 0.25, 0.5, None, m))
    assert (out[1] == -math.inf).all()
    assert ops().process_logits(x[:0]).shape == (0, V)


def test_strides_and_graph():
    rows, V = 6, 5001
    wide = torch.randn(rows, V + 7, device=DEV)
    x = wide[:, 3:3 + V]                                          # odd offset, odd stride
    ids = torch.randint(0, V, (rows, 50), device=DEV)[:, 5:45]
    ow = torch.full((rows, V + 11), 9.0, device=DEV)
    out = ow[:, 1:1 + V]
    kw = dict(generated=ids, repetition_penalty=1.2, frequency_penalty=0.3)
    assert ops().process_logits(x, out=out, **kw) is out
    same(out, reference(x, ids, None, 1.2, 0.0, 0.3))
    assert (ow[:, 0] == 9).all() and (ow[:, 1 + V:] == 9).all()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = ops().process_logits(x, **kw)
    for i in range(3):
        wide.copy_(torch.randn(rows, V + 7, device=DEV))
        eager = ops().process_logits(x, **kw)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, eager)
        same(got, reference(x, ids, None, 1.2, 0.0, 0.3))


def test_nothing_to_apply():
    """float32 logits come back as they are; bf16 ones, or ones with an `out`, are converted / copied."""
    x = torch.randn(3, 100, device=DEV)
    out = torch.empty_like(x)
    assert ops().process_logits(x, repetition_penalty=1.2, presence_penalty=0.5) is x
    assert ops().process_logits(x, out=out) is out and torch.equal(out, x)
    assert torch.equal(ops().process_logits(x.bfloat16()), x.bfloat16().float())


def test_refusals():
    o = ops()
    x = torch.randn(3, 100, device=DEV)
    ids = torch.zeros(3, 4, dtype=torch.int64, device=DEV)
    bad = [
        (RuntimeError, lambda: o.process_logits(x.cpu())),
        (ValueError, lambda: o.process_logits(x.half())),
        (ValueError, lambda: o.process_logits(x.t())),
        (ValueError, lambda: o.process_logits(x[:1].expand(3, 100))),
        (ValueError, lambda: o.process_logits(x, out=x.bfloat16())),
        (ValueError, lambda: o.process_logits(x, generated=ids.int())),
        (ValueError, lambda: o.process_logits(x, generated=ids[:2])),
        (ValueError, lambda: o.process_logits(x, n_generated=ids[:, 0].int())),
        (ValueError, lambda: o.process_logits(x, generated=ids, n_generated=ids[:, 0])),
        (ValueError, lambda: o.process_logits(x, repetition_penalty=x[:, 0].double())),
        (ValueError, lambda: o.process_logits(x, presence_penalty=x[0])),
        (ValueError, lambda: o.process_logits(x, bias=x[:2])),
        (ValueError, lambda: o.process_logits(x, bias=x[0].double())),
        (ValueError, lambda: o.process_logits(x, allowed=torch.zeros(3, dtype=torch.int32, device=DEV))),
        (ValueError, lambda: o.process_logits(x, bias=x[0].cpu())),
        (RuntimeError, lambda: o.process_logits(x, repetition_penalty=0.0)),
        (RuntimeError, lambda: o.process_logits(x, generated=ids[:1].expand(3, 4))),
    ]
    for i, (kind, f) in enumerate(bad):
        with pytest.raises(kind):
            f()
            pytest.fail(f"refusal {i} was accepted")
