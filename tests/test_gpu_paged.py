"""The paged cache and its attention against their definitions in 64 bits (tests/_paged_common.py).

Tolerances.  A value stored as bf16 is off by at most half a step, 2^-8 of it; e4m3 by 2^-4 of it, or by half a subnormal step, 2^-10 of the
head's scale.  In front of that rounding everything is float32 (2^-24 an operation, a few operations: 2^-20 of the magnitudes summed).
Attention rounds the probabilities to bf16 in front of the product with V (at most 2^-8 of every term: one bf16 in the tiles, two in the rows), its scores are float32 sums of dim products
(2^-24 * dim of |q| |k| * scale, below 2^-12 in the exponent for the values used here, so 2^-11 of a probability) and the result is rounded
once: (2^-8 + 2^-10) * sum p |v| + 2^-8 * |out|."""
import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import _paged_common as C  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ops():
    from molly_amd import ops as o
    return o


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


# ---- store and read ---------------------------------------------------------------------------------------------------------------
def store_inputs(n, nq, nkv, hd, seed, scale=1.0):
    g = gen(seed)
    x = (scale * torch.randn(n, (nq + 2 * nkv) * hd, generator=g, device=DEV)).bfloat16()
    q, k, v = x[:, :nq * hd], x[:, nq * hd:(nq + nkv) * hd], x[:, (nq + nkv) * hd:]
    qw, kw = ((1 + 0.2 * torch.randn(hd, generator=g, device=DEV)).bfloat16() for _ in range(2))
    ang = torch.arange(500, device=DEV, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(0, hd, 2, device=DEV, dtype=torch.float64) / hd)
    pos = torch.randint(0, 500, (n,), generator=g, device=DEV, dtype=torch.int32)
    return q, k, v, qw, kw, ang.cos().float(), ang.sin().float(), pos


def empty_pools(n_pages, nkv, page, hd, fp8):
    if fp8:
        k, v = (torch.full((n_pages, nkv, page, hd), 0x7f, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for _ in range(2))
        return k, v, *(torch.full((n_pages, nkv, page), 127, dtype=torch.uint8, device=DEV) for _ in range(2))
    k, v = (torch.full((n_pages, nkv, page, hd), math.nan, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    return k, v, None, None


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,nq,nkv,page", [(1, 4, 2, 16), (33, 3, 1, 64), (131, 0, 5, 32), (700, 16, 8, 256)])
@pytest.mark.parametrize("norm,rope", [(False, False), (True, False), (True, True)])
def test_append_and_read(n, nq, nkv, page, hd, fp8, norm, rope):
    q, k, v, qw, kw, cos, sin, pos = store_inputs(n, nq, nkv, hd, n + hd)
    n_pages = n // page + 3
    kp, vp, ks, vs = empty_pools(n_pages, nkv, page, hd, fp8)
    slot = torch.randperm(n_pages * page, generator=gen(7), device=DEV)[:n].to(torch.int32)
    if n > 1:
        slot[n // 2] = -1
    a = dict(qw=qw if norm and nq else None, kw=kw if norm else None)
    if rope:
        a.update(cos=cos, sin=sin, positions=pos)
    qo = ops().paged_kv_append(k, v, kp, vp, slot, kscale=ks, vscale=vs, q=q if nq else None, **a)
    kr, vr = ops().paged_kv_read(kp, vp, slot, kscale=ks, vscale=vs)
    live = (slot >= 0)[:, None, None]
    rp = (cos, sin, pos) if rope else ()
    slop = 2.0 ** -20 * 16                                        # heads have unit rms: magnitudes summed are below 16
    if nq:
        ref = C.turned(q, nq, a["qw"], *rp)
        assert ((qo.double().view(n, nq, hd) - ref).abs() <= 2.0 ** -8 * ref.abs() + slop).all()
    else:
        assert qo is None
    for got, x, w, r in ((kr, k, a["kw"], rp), (vr, v, None, ())):
        ref = torch.where(live, C.turned(x, nkv, w, *r), 0.0)
        got = got.double().view(n, nkv, hd)
        if not fp8:
            assert ((got - ref).abs() <= 2.0 ** -8 * ref.abs() + (slop if norm or rope else 0)).all()
            if not (w is not None or r):
                assert torch.equal(got, ref)
        elif w is None and not r:
            assert torch.equal(got, torch.where(live, C.quantise(ref)[0], 0.0))       # bf16 in, exact arithmetic: the very codes
        else:
            unit = torch.exp2(C.quantise(ref)[1].double() - 127)[..., None]
            assert ((got - ref).abs() <= 2.0 ** -4 * ref.abs() + 2.0 ** -10 * 2 * unit + slop).all()      # (2: the exponent may sit next to a border)
    # nothing else in the pools changed
    touched = torch.zeros(n_pages * page, dtype=torch.bool, device=DEV)
    touched[slot[slot >= 0].long()] = True
    rest = ~touched.view(n_pages, 1, page, 1).expand(n_pages, nkv, page, hd)
    for p in (kp, vp):
        assert torch.isnan(p.float()[rest]).all()


def test_append_codes_match_the_format():
    """Every bf16 magnitude class through the quantiser: subnormal heads, the largest values, zeros, infinities, NaN, ties."""
    hd = 64
    rows = [torch.linspace(-448, 448, hd), torch.linspace(0, 2.0 ** -20, hd), torch.zeros(hd), torch.linspace(-3e38, 3e38, hd),
            torch.linspace(1, 8, hd), torch.full((hd,), 1e-40), torch.arange(hd) / 16.0, -torch.arange(hd) * 1e-3, torch.full((hd,), 449.0)]
    k = torch.stack(rows).bfloat16().to(DEV)
    bad = k[:2].clone()
    bad[0, 3], bad[0, 9], bad[1, 0] = math.inf, math.nan, -math.inf
    k = torch.cat([k, bad])
    n = k.shape[0]
    kp, vp, ks, vs = empty_pools(1, 1, 16, hd, True)
    slot = torch.arange(n, device=DEV, dtype=torch.int32)
    ops().paged_kv_append(k, k, kp, vp, slot, kscale=ks, vscale=vs)
    val, e = C.quantise(k.double())
    assert torch.equal(ks[0, 0, :n], e)
    got = C.held(kp, ks)[0, 0, :n]
    assert torch.equal(torch.isnan(got), torch.isnan(val)) and torch.equal(got.nan_to_num(7.0), val.nan_to_num(7.0))
    kr, vr = ops().paged_kv_read(kp, vp, slot, kscale=ks, vscale=vs)
    assert torch.equal(kr.double().nan_to_num(7.0), val.bfloat16().double().nan_to_num(7.0)) and torch.equal(torch.isnan(kr), torch.isnan(vr))


@pytest.mark.parametrize("e", [1, 2, 3, 4, 100, 127, 246, 247])
def test_every_code_is_read_as_the_nearest_bf16(e):
    """Exactly what it stands for with exponent bytes of 3 .. 246; below, bf16's subnormals are coarser than the smallest codes; above, 2^128 is no bf16."""
    codes = torch.arange(256, dtype=torch.int32, device=DEV).to(torch.uint8)
    kp = torch.zeros(1, 1, 16, 128, dtype=torch.uint8, device=DEV)
    kp.view(-1)[:256] = codes
    kp, ks = kp.view(torch.float8_e4m3fn), torch.full((1, 1, 16), e, dtype=torch.uint8, device=DEV)
    kr, vr = ops().paged_kv_read(kp, kp, torch.arange(2, dtype=torch.int32, device=DEV), kscale=ks, vscale=ks)
    held = C.held(kp, ks).view(-1)[:256]
    want = held.cpu().float().bfloat16()                          # (float32 holds them all; one rounding)
    for got in (kr, vr):
        got = got.view(-1).cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got[~torch.isnan(want)], want[~torch.isnan(want)])
    fin = torch.isfinite(held.cpu())
    assert bool((want.double() == held.cpu())[fin].all()) == (3 <= e <= 246)


def test_append_without_queries_takes_their_gain_too():
    _, k, v, qw, kw, *_ = store_inputs(9, 4, 2, 64, 3)
    slot = torch.arange(9, device=DEV, dtype=torch.int32)
    kp, vp, _, _ = empty_pools(1, 2, 16, 64, False)
    kp2, vp2 = kp.clone(), vp.clone()
    assert ops().paged_kv_append(k, v, kp, vp, slot, qw=qw, kw=kw) is None
    ops().paged_kv_append(k, v, kp2, vp2, slot, kw=kw)
    assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in ((kp, kp2), (vp, vp2)))


@pytest.mark.parametrize("fp8", [False, True])
def test_append_and_read_of_no_rows(fp8):
    q, k, v, qw, kw, cos, sin, pos = store_inputs(3, 4, 2, 64, 3)
    kp, vp, ks, vs = empty_pools(1, 2, 16, 64, fp8)
    slot = torch.zeros(0, dtype=torch.int32, device=DEV)
    before = [p.view(torch.uint8).clone() for p in (kp, vp)]
    qo = ops().paged_kv_append(k[:0], v[:0], kp, vp, slot, kscale=ks, vscale=vs, q=q[:0], qw=qw, kw=kw, cos=cos, sin=sin, positions=pos[:0])
    kr, vr = ops().paged_kv_read(kp, vp, slot, kscale=ks, vscale=vs)
    assert qo.shape == (0, 256) and kr.shape == vr.shape == (0, 128)
    assert all(torch.equal(p.view(torch.uint8), b) for p, b in zip((kp, vp), before))


def test_tables_without_rows_are_refused():
    _, k, v, _, _, cos, sin, pos = store_inputs(3, 4, 2, 64, 3)
    kp, vp, _, _ = empty_pools(1, 2, 16, 64, False)
    with pytest.raises(RuntimeError, match="go together"):
        ops().paged_kv_append(k, v, kp, vp, torch.arange(3, device=DEV, dtype=torch.int32), cos=cos[:0], sin=sin[:0], positions=pos)
    assert torch.isnan(kp).all() and torch.isnan(vp).all()


def test_append_in_place_strided_and_bad_positions():
    n, nq, nkv, hd = 9, 4, 2, 64
    q, k, v, qw, kw, cos, sin, pos = store_inputs(n, nq, nkv, hd, 3)
    pos[4], pos[5] = 500, -1                                      # outside the tables
    kp, vp, _, _ = empty_pools(2, nkv, 16, hd, False)
    slot = torch.arange(n, device=DEV, dtype=torch.int32)
    want = ops().paged_kv_append(k, v, kp, vp, slot, q=q, qw=qw, kw=kw, cos=cos, sin=sin, positions=pos)
    wide = torch.zeros(n, nq * hd + 8, dtype=torch.bfloat16, device=DEV)
    qi = wide[:, :nq * hd]
    qi.copy_(q)
    got = ops().paged_kv_append(k, v, kp, vp, slot, q=qi, q_out=qi, qw=qw, kw=kw, cos=cos, sin=sin, positions=pos)
    assert got.data_ptr() == wide.data_ptr() and torch.equal(got.nan_to_num(9.0), want.nan_to_num(9.0)) and not wide[:, nq * hd:].any()
    isnan = torch.isnan(got).all(1)
    assert isnan[4] and isnan[5] and int(torch.isnan(got).any(1).sum()) == 2
    kr, vr = ops().paged_kv_read(kp, vp, slot)
    assert torch.isnan(kr[4:6]).all() and torch.isfinite(kr[:4]).all() and torch.equal(vr, v)


# ---- attention ----------------------------------------------------------------------------------------------------------------------
def layout(g, keys, page, spare=2):
    """block table with the pages of all sequences shuffled, and which places of the pool hold keys"""
    need = [-(-max(k, 0) // page) for k in keys]
    n_pages = sum(need) + spare
    order = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(keys), max(need + [1]) + 1), -1, dtype=torch.int32, device=DEV)
    live = torch.zeros(n_pages, page, dtype=torch.bool, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        for j in range(n):
            live[int(order[at + j]), : min(page, keys[b] - j * page)] = True
        at += n
    return table, n_pages, live


def poison(kp, vp, live):
    """what no sequence holds is NaN"""
    m = ~live[:, None, :, None].expand(kp.shape)
    if kp.dtype == torch.float8_e4m3fn:
        for p in (kp, vp):
            p.view(torch.uint8)[m] = 0x7f
    else:
        kp[m] = math.nan
        vp[m] = math.nan


def case(new, keys, nh, nkv, hd, page, fp8, seed=0):
    g = gen(seed)
    table, n_pages, live = layout(g, keys, page)
    kp, vp, ks, vs = C.pools(g, n_pages, nkv, page, hd, fp8, DEV)
    poison(kp, vp, live)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    q = torch.randn(cu[-1], nh * hd, generator=g, device=DEV).bfloat16()
    cu_t, len_t = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (cu, keys))
    return q, kp, vp, ks, vs, table, cu, keys, cu_t, len_t


def check(out, q, kp, vp, ks, vs, table, cu, keys, nh, scale=None):
    hd = kp.shape[-1]
    ref, mag = C.attend(q, C.held(kp, ks), C.held(vp, vs), table, cu, keys, nh, hd ** -0.5 if scale is None else scale)
    got = out.double().view(ref.shape)
    rows = torch.zeros(q.shape[0], dtype=torch.bool, device=DEV)
    rows[cu[0]:cu[-1]] = True
    got, ref, mag = got[rows], ref[rows], mag[rows]
    fin = torch.isfinite(ref)
    assert torch.equal(fin, torch.isfinite(got))
    err = (got - ref).abs()[fin]
    tol = ((2.0 ** -8 + 2.0 ** -10) * mag + 2.0 ** -8 * ref.abs())[fin] + 1e-30
    assert (err <= tol).all(), (float((err / tol).max()), float(err.max()))


SHAPES = [
    # new tokens, keys of each sequence; heads, kv heads
    ([1], [1], 4, 4),
    ([1], [37], 16, 8),
    ([1, 1, 1], [700, 1, 2050], 8, 2),
    ([1] * 5, [64, 63, 65, 128, 5], 5, 1),
    ([1, 1], [5000, 4001], 16, 2),
    ([3, 1, 2], [3, 400, 130], 8, 2),
    ([7], [7], 14, 2),
    ([40, 0, 1, 17], [300, 50, 1, 17], 6, 2),
    ([130], [1500], 16, 8),
    ([257, 5, 64], [257, 700, 64], 12, 4),
    ([1, 200, 1], [900, 1031, 77], 32, 8),
    ([300], [2600], 2, 2),
]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("hd,page", [(128, 64), (64, 16), (128, 16), (64, 128), (128, 256), (64, 32)])
@pytest.mark.parametrize("new,keys,nh,nkv", SHAPES)
def test_attn_paged(new, keys, nh, nkv, hd, page, fp8):
    q, kp, vp, ks, vs, table, cu, keys, cu_t, len_t = case(new, keys, nh, nkv, hd, page, fp8, seed=len(keys) + hd)
    out = ops().attn_paged(q, kp, vp, table, cu_t, len_t, nh, kscale=ks, vscale=vs, max_q=max(new), max_kv=max(keys))
    check(out, q, kp, vp, ks, vs, table, cu, keys, nh)
    # what the caller says of the lengths chooses the cut, not the result
    for mq, mk in ((0, 0), (1, 1), (100000, 1 << 20)):
        o2 = ops().attn_paged(q, kp, vp, table, cu_t, len_t, nh, kscale=ks, vscale=vs, max_q=mq, max_kv=mk)
        check(o2, q, kp, vp, ks, vs, table, cu, keys, nh)
    # the same bits twice
    assert torch.equal(out, ops().attn_paged(q, kp, vp, table, cu_t, len_t, nh, kscale=ks, vscale=vs, max_q=max(new), max_kv=max(keys)))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("new,keys,nh,nkv,hd", [([1, 1], [900, 40], 48, 1, 128), ([1], [6000], 71, 1, 64), ([2, 1], [70, 3000], 64, 2, 128)])
def test_attn_paged_more_query_heads_than_a_tile_of_single_steps_has_rows(new, keys, nh, nkv, hd, fp8):
    q, kp, vp, ks, vs, table, cu, keys, cu_t, len_t = case(new, keys, nh, nkv, hd, 32, fp8, seed=12)
    for mq, mk in ((max(new), max(keys)), (0, 0)):
        check(ops().attn_paged(q, kp, vp, table, cu_t, len_t, nh, kscale=ks, vscale=vs, max_q=mq, max_kv=mk), q, kp, vp, ks, vs, table, cu, keys, nh)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("kind", ["decode", "short", "mixed", "long"])
def test_attn_paged_many_sequences(kind, fp8):
    """More sequences than a wave has lanes, some without new tokens, lengths from none to thousands; few long ones over few heads."""
    import random
    r = random.Random(3)
    B = 150 if kind != "long" else 3
    keys = [int(5000 * r.random() ** 4) for _ in range(B)] if kind != "long" else [20000, 100, 9000]
    new = {"decode": [1] * B, "short": [r.choice([0, 1, 3, 7]) for _ in range(B)], "mixed": [r.choice([0, 1, 1, 40]) for _ in range(B)],
           "long": [1, 0, 2]}[kind]
    nh, nkv = (8, 2) if kind != "long" else (4, 1)
    q, kp, vp, ks, vs, table, cu, keys, cu_t, len_t = case(new, keys, nh, nkv, 64, 32, fp8, seed=6)
    o = ops()
    n, max_pages = q.shape[0], table.shape[1]
    floats = o.attn_paged_workspace(n, B, nh, nkv, 64, 32, max_pages, fp8, max(new), max(keys))
    outs = []
    for ws in (None, torch.full((max(floats, 1),), math.nan, device=DEV), torch.empty(16, device=DEV)):      # its own; the caller's; too small: uncut
        outs.append(o.attn_paged(q, kp, vp, table, cu_t, len_t, nh, kscale=ks, vscale=vs, max_q=max(new), max_kv=max(keys), workspace=ws))
        check(outs[-1], q, kp, vp, ks, vs, table, cu, keys, nh)
    assert torch.equal(outs[0], outs[1])
    for mq, mk in ((1, 1), (0, 0)):                               # hints that are wrong
        check(o.attn_paged(q, kp, vp, table, cu_t, len_t, nh, kscale=ks, vscale=vs, max_q=mq, max_kv=mk), q, kp, vp, ks, vs, table, cu, keys, nh)


@pytest.mark.parametrize("new,keys", [([1, 1], [2100, 33]), ([90, 3], [400, 3])])
def test_attn_paged_e4m3_is_bf16_of_the_held_values(new, keys):
    """The held values are exact in bf16, so both calls compute the same numbers: bit for bit where the keys go by in the same order (the tile kernel),
    within the bound of either where a block has another number of waves to deal them to (single steps: the sums are taken in another order, and the
    parts' maxima, which P is rounded against, differ)."""
    q, kp, vp, ks, vs, table, cu, keys, cu_t, len_t = case(new, keys, 8, 2, 128, 32, True, seed=5)
    a = ops().attn_paged(q, kp, vp, table, cu_t, len_t, 8, kscale=ks, vscale=vs, max_q=max(new), max_kv=max(keys))
    b = ops().attn_paged(q, C.held(kp, ks).bfloat16(), C.held(vp, vs).bfloat16(), table, cu_t, len_t, 8, max_q=max(new), max_kv=max(keys))
    for x in (a, b):
        check(x, q, kp, vp, ks, vs, table, cu, keys, 8)
    if max(new) * 4 > 32:
        assert torch.equal(a, b)


@pytest.mark.parametrize("fp8", [False, True])
def test_attn_paged_rows_that_see_nothing(fp8):
    """More new tokens than keys: the first rows see none; empty sequences, no sequences, no rows."""
    new, keys = [5, 3, 2, 0, 70], [3, 0, -4, 9, 10]
    q, kp, vp, ks, vs, table, cu, keys, cu_t, len_t = case(new, keys, 4, 2, 64, 16, fp8)
    out = ops().attn_paged(q, kp, vp, table, cu_t, len_t, 4, kscale=ks, vscale=vs, max_q=70)
    check(out, q, kp, vp, ks, vs, table, cu, keys, 4)
    assert not out[:2].any() and not out[5:10].any() and not out[10:70].any() and out[2].any() and out[70:].all(0).any()
    z = torch.zeros(0, 4 * 64, dtype=torch.bfloat16, device=DEV)
    assert ops().attn_paged(z, kp, vp, table, torch.zeros_like(cu_t), len_t, 4, kscale=ks, vscale=vs).shape == z.shape
    keep = torch.full_like(q, 3.0)
    ops().attn_paged(q, kp, vp, table[:0], cu_t[:1], len_t[:0], 4, kscale=ks, vscale=vs, out=keep)
    assert (keep == 3.0).all()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("new", [[1, 1, 2], [5, 3, 70], [1, 90, 200]])
def test_attn_paged_any_negative_number_of_keys_is_none(new, fp8):
    """kv_len - n of the smallest int is no small number."""
    q, kp, vp, ks, vs, table, cu, keys, cu_t, len_t = case(new, [40, 300, 200], 4, 2, 64, 16, fp8)
    good = ops().attn_paged(q, kp, vp, table, cu_t, len_t, 4, kscale=ks, vscale=vs, max_q=max(new))
    for few in (0, -1, -2 ** 31, -2 ** 31 + 1, -2 ** 31 + 60):
        len_t[0], len_t[2] = few, few
        out = ops().attn_paged(q, kp, vp, table, cu_t, len_t, 4, kscale=ks, vscale=vs, max_q=max(new))
        assert not out[: cu[1]].any() and not out[cu[2]:].any() and torch.equal(out[cu[1]:cu[2]], good[cu[1]:cu[2]])


def test_attn_paged_rows_outside_the_sequences_stay():
    q, kp, vp, ks, vs, table, cu, keys, cu_t, len_t = case([4, 30], [50, 30], 4, 2, 128, 16, False)
    pad = torch.cat([q[:3], q, q[:20]])
    for mq in (1, 30):
        out = torch.full_like(pad, 5.0)
        got = ops().attn_paged(pad, kp, vp, table, cu_t + 3, len_t, 4, max_q=mq, out=out)
        assert got is out and (out[:3] == 5.0).all() and (out[37:] == 5.0).all()
        check(out[3:37], q, kp, vp, ks, vs, table, cu, keys, 4)


@pytest.mark.parametrize("new,keys", [([1, 1], [300, 90]), ([100, 60], [300, 60])])
@pytest.mark.parametrize("bad", [-1, 1 << 30, "n_pages", "short"])
def test_attn_paged_pages_outside_the_pool(new, keys, bad):
    """A row with a visible key on a page that is none is NaN; the others are as they were."""
    q, kp, vp, ks, vs, table, cu, keys, cu_t, len_t = case(new, keys, 4, 2, 64, 32, False, seed=2)
    good = ops().attn_paged(q, kp, vp, table, cu_t, len_t, 4, max_q=max(new))
    first = 7 * 32                                                # the first key of sequence 0's page 7
    t = table.clone()
    if bad == "short":
        t = t[:, :7].contiguous()
    else:
        t[0, 7] = kp.shape[0] if bad == "n_pages" else bad
    out = ops().attn_paged(q, kp, vp, t, cu_t, len_t, 4, max_q=max(new))
    sees = torch.zeros(q.shape[0], dtype=torch.bool, device=DEV)
    for i in range(new[0]):
        sees[i] = keys[0] - new[0] + i >= first
    assert torch.isnan(out[sees]).all() and torch.equal(out[~sees], good[~sees])


@pytest.mark.parametrize("what", ["nan", "inf"])
@pytest.mark.parametrize("new,keys,nh,nkv", [([60], [200], 4, 2), ([150, 5], [150, 40], 8, 2), ([4], [300], 4, 1)])
def test_attn_paged_nothing_leaks_from_later_tokens(what, new, keys, nh, nkv):
    """The K and V of a token are NaN or infinite: only it and the rows behind it notice."""
    q, kp, vp, ks, vs, table, cu, keys, cu_t, len_t = case(new, keys, nh, nkv, 128, 16, False, seed=4)
    good = ops().attn_paged(q, kp, vp, table, cu_t, len_t, nh, max_q=max(new))
    j = keys[0] - new[0] // 2                                     # a key that the second half of the chunk sees
    x = math.nan if what == "nan" else math.inf
    kp[table[0, j // 16].long(), :, j % 16] = x
    vp[table[0, j // 16].long(), :, j % 16, ::3] = x
    out = ops().attn_paged(q, kp, vp, table, cu_t, len_t, nh, max_q=max(new))
    first = j - (keys[0] - new[0])
    assert torch.equal(out[:first], good[:first]) and torch.equal(out[new[0]:], good[new[0]:])
    assert not torch.isfinite(out[first:new[0]]).all(1).any()
    # V alone: the columns that are not finite in V, and only those
    kp[table[0, j // 16].long(), :, j % 16] = 0.5
    out = ops().attn_paged(q, kp, vp, table, cu_t, len_t, nh, max_q=max(new))
    check(out, q, kp, vp, ks, vs, table, cu, keys, nh)
    if what == "inf":
        assert (out.view(-1, nh, 128)[first:new[0], :, ::3] == math.inf).all()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new,keys,nh,nkv", [([1], [700], 16, 8), ([1, 1], [2050, 40], 8, 2), ([5], [900], 2, 2), ([150], [400], 8, 2)])
def test_attn_paged_infinite_values_that_every_row_sees(new, keys, nh, nkv, hd):
    """p * inf is inf with V's sign (two of opposite signs: NaN), as by the formula; the other columns are as they were."""
    q, kp, vp, ks, vs, table, cu, keys, cu_t, len_t = case(new, keys, nh, nkv, hd, 16, False, seed=8)
    a = dict(max_q=max(new), max_kv=max(keys))
    good = ops().attn_paged(q, kp, vp, table, cu_t, len_t, nh, **a).view(-1, nh, hd)
    for j, col, x in ((5, 0, math.inf), (130, 33, -math.inf), (7, 50, math.inf), (140, 50, -math.inf)):
        vp[table[0, j // 16].long(), :, j % 16, col] = x
    out = ops().attn_paged(q, kp, vp, table, cu_t, len_t, nh, **a).view(-1, nh, hd)
    own = out[:new[0]]
    assert (own[..., 0] == math.inf).all() and (own[..., 33] == -math.inf).all() and torch.isnan(own[..., 50]).all()
    rest = [c for c in range(hd) if c not in (0, 33, 50)]
    assert torch.equal(own[..., rest], good[:new[0]][..., rest]) and torch.equal(out[new[0]:], good[new[0]:])


def test_attn_paged_strides_scale_and_shared_pages():
    """q and out as parts of wider rows, a table that is a part of a wider one, a scale of one's own, sequences that share pages."""
    q, kp, vp, ks, vs, table, cu, keys, cu_t, len_t = case([3, 20, 1], [100, 97, 64], 8, 2, 64, 32, False, seed=8)
    table[1, :2] = table[0, :2]                                   # a common prefix of two pages
    wide = torch.zeros(q.shape[0], 3 * 512 + 8, dtype=torch.bfloat16, device=DEV)
    wide[:, 512:1024] = q
    tw = torch.full((3, 11), 99999, dtype=torch.int32, device=DEV)
    tw[:, 2:2 + table.shape[1]] = table
    ow = torch.full_like(wide, 2.0)
    for mq in (1, 20):
        ops().attn_paged(wide[:, 512:1024], kp, vp, tw[:, 2:2 + table.shape[1]], cu_t, len_t, 8, scale=0.3, max_q=mq, out=ow[:, 8:520])
        check(ow[:, 8:520], q, kp, vp, ks, vs, table, cu, keys, 8, scale=0.3)
        assert (ow[:, :8] == 2.0).all() and (ow[:, 520:] == 2.0).all()


@pytest.mark.parametrize("fp8", [False, True])
def test_pools_past_32_bits(fp8):
    """Pages whose values lie past 2^32 values and bytes: written, read back and attended to."""
    nkv, page, hd = 8, 256, 128
    n_pages = (1 << 32) // (nkv * page * hd) + 40                 # > 2^32 values
    kp = torch.empty(n_pages, nkv, page, hd, dtype=torch.uint8 if fp8 else torch.bfloat16, device=DEV)
    vp = torch.empty_like(kp)
    ks = vs = None
    if fp8:
        kp, vp = kp.view(torch.float8_e4m3fn), vp.view(torch.float8_e4m3fn)
        ks, vs = (torch.empty(n_pages, nkv, page, dtype=torch.uint8, device=DEV) for _ in range(2))
    keys = [300, 600]
    g = gen(1)
    k, v = (torch.randn(900, nkv * hd, generator=g, device=DEV).bfloat16() for _ in range(2))
    table = torch.tensor([[n_pages - 1, 3, 0], [n_pages - 7, n_pages - 3, 1]], dtype=torch.int32, device=DEV)
    slot = torch.cat([table[b].long().repeat_interleave(page)[:n] * page + torch.arange(n, device=DEV) % page for b, n in enumerate(keys)]).to(torch.int32)
    ops().paged_kv_append(k, v, kp, vp, slot, kscale=ks, vscale=vs)
    kr, vr = ops().paged_kv_read(kp, vp, slot, kscale=ks, vscale=vs)
    want = lambda x: C.quantise(x.double().view(900, nkv, hd))[0].flatten(1) if fp8 else x.double()  # noqa: E731
    assert torch.equal(kr.double(), want(k)) and torch.equal(vr.double(), want(v))
    ids = table[:, :3].flatten().long()
    small = torch.arange(6, device=DEV, dtype=torch.int32).view(2, 3)
    for new in ([1, 1], [200, 90]):
        cu = [0, new[0], new[0] + new[1]]
        q = torch.randn(cu[-1], 16 * hd, generator=g, device=DEV).bfloat16()
        cu_t, len_t = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (cu, keys))
        out = ops().attn_paged(q, kp, vp, table, cu_t, len_t, 16, kscale=ks, vscale=vs, max_q=max(new))
        sel = [None if t is None else t.view(torch.uint8)[ids].view(t.dtype) if t.dtype == torch.float8_e4m3fn else t[ids] for t in (kp, vp, ks, vs)]
        live = torch.zeros(6, page, dtype=torch.bool, device=DEV)
        for b, n in enumerate(keys):
            for j in range(3):
                live[3 * b + j, : max(0, min(page, n - j * page))] = True
        sel[0], sel[1] = sel[0].clone(), sel[1].clone()
        m = ~live[:, None, :, None].expand(sel[0].shape)
        for t in sel[:2]:
            (t.view(torch.uint8) if fp8 else t)[m] = 0
        if fp8:
            for t in sel[2:]:
                t[~live[:, None].expand(t.shape)] = 127
        check(out, q, *sel, small, cu, keys, 16)


def test_attn_paged_on_a_stream_and_in_graphs():
    """Two graphs captured from two calls, replayed in turn and at once with new contents, against eager results."""
    cs = [case([1, 1, 1], [3000, 40, 777], 16, 8, 128, 64, False, seed=1), case([33, 1], [1200, 90], 8, 2, 128, 64, True, seed=2)]
    nh = [16, 8]
    side = [torch.cuda.Stream() for _ in cs]

    def call(i):
        q, kp, vp, ks, vs, table, cu, keys, cu_t, len_t = cs[i]
        return ops().attn_paged(q, kp, vp, table, cu_t, len_t, nh[i], kscale=ks, vscale=vs, max_q=max(b - a for a, b in zip(cu, cu[1:])), max_kv=4096)
    torch.cuda.synchronize()
    eager = [call(0), call(1)]
    graphs, outs = [], []
    for i in range(2):
        with torch.cuda.stream(side[i]):
            assert torch.equal(call(i), eager[i])
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side[i]):
            outs.append(call(i))
        graphs.append(g)
    for rep in range(4):
        for i in range(2):
            cs[i][0].copy_(torch.randn(cs[i][0].shape, generator=gen(50 + rep), device=DEV).bfloat16())
            outs[i].zero_()
        eager = [call(0), call(1)]
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(side[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i], eager[i])
            check(outs[i], *cs[i][:8], nh[i])


def test_refusals():
    q, kp, vp, ks, vs, table, cu, keys, cu_t, len_t = case([2, 3], [40, 33], 4, 2, 64, 16, True)
    o = ops()
    bf = kp.float().bfloat16()
    k = torch.zeros(5, 128, dtype=torch.bfloat16, device=DEV)
    slot = torch.arange(5, device=DEV, dtype=torch.int32)
    cos = torch.zeros(10, 32, device=DEV)
    bad = [
        (ValueError, lambda: o.attn_paged(q, kp, vp, table, cu_t, len_t, 4)),                                     # e4m3 without exponents
        (ValueError, lambda: o.attn_paged(q, bf, bf, table, cu_t, len_t, 4, kscale=ks, vscale=vs)),               # bf16 with them
        (ValueError, lambda: o.attn_paged(q, kp, bf, table, cu_t, len_t, 4, kscale=ks, vscale=vs)),
        (ValueError, lambda: o.attn_paged(q, bf, bf, table, cu_t, len_t, 3)),                                     # 3 heads over 2
        (ValueError, lambda: o.attn_paged(q[:, :-64], bf, bf, table, cu_t, len_t, 4)),
        (TypeError, lambda: o.attn_paged(q.float(), bf, bf, table, cu_t, len_t, 4)),
        (ValueError, lambda: o.attn_paged(q, bf, bf, table.long(), cu_t, len_t, 4)),
        (ValueError, lambda: o.attn_paged(q, bf, bf, table, cu_t[:-1], len_t, 4)),
        (ValueError, lambda: o.attn_paged(q, bf, bf, table, cu_t, len_t.cpu(), 4)),
        (ValueError, lambda: o.attn_paged(q, bf.transpose(1, 2), bf.transpose(1, 2), table, cu_t, len_t, 4)),
        (RuntimeError, lambda: o.attn_paged(torch.zeros(5 * 256 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(5, 256), bf, bf, table, cu_t, len_t,
                                            4)),                                                                          # not 16-byte aligned
        (RuntimeError, lambda: o.attn_paged(q, bf, bf, table, cu_t, len_t, 4, scale=-1.0)),
        (RuntimeError, lambda: o.attn_paged(q, bf[:, :, :8].contiguous(), bf[:, :, :8].contiguous(), table, cu_t, len_t, 4)),     # pages of 8
        (RuntimeError, lambda: o.attn_paged(q[:, :128], bf[..., :32].contiguous(), bf[..., :32].contiguous(), table, cu_t, len_t, 4)),   # dim 32
        (RuntimeError, lambda: o.attn_paged(q.cpu(), bf.cpu(), bf.cpu(), table.cpu(), cu_t.cpu(), len_t.cpu(), 4)),
        (RuntimeError, lambda: o.attn_paged(q[:1].expand(5, 256), bf, bf, table, cu_t, len_t, 4)),                # rows on top of each other
        (ValueError, lambda: o.paged_kv_append(k, k[:4], bf, bf, slot)),
        (ValueError, lambda: o.paged_kv_append(k, k, bf, bf, slot[:4])),
        (ValueError, lambda: o.paged_kv_append(k, k, bf, bf, slot.long())),
        (ValueError, lambda: o.paged_kv_append(k, k, bf, bf, slot, cos=cos, sin=cos)),
        (ValueError, lambda: o.paged_kv_append(k, k, bf, bf, slot, cos=cos[:, :16], sin=cos[:, :16], positions=slot)),
        (ValueError, lambda: o.paged_kv_append(k, k, bf, bf, slot, q_out=k)),
        (ValueError, lambda: o.paged_kv_append(k, k, bf, bf, slot, q=k[:, :100])),
        (ValueError, lambda: o.paged_kv_append(k, k, bf, bf, slot, kw=k[0])),
        (TypeError, lambda: o.paged_kv_append(k.half(), k, bf, bf, slot)),
        (ValueError, lambda: o.paged_kv_read(bf, bf, slot, k_out=k[:4])),
        (ValueError, lambda: o.paged_kv_read(bf, bf, slot[None])),
        (TypeError, lambda: o.paged_kv_read(bf.half(), bf.half(), slot)),
    ]
    for i, (kind, f) in enumerate(bad):
        with pytest.raises(kind):
            f()
            pytest.fail(f"refusal {i} was accepted")
