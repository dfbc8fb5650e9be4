"""The operators of one serving step over a paged key/value cache, their plain forms and the cases they are measured at.

  store    new keys and values go into the pages of a cache (q/k-norm and rotary in the same pass where the path has them), as bf16 or as
           e4m3 with a power-of-two scale for each head of each token, and the rows of a list of places are read back
  attend   ragged chunks of new tokens (one token each: a decode step) attend causally to everything their sequence has in the pages
  choose   repetition / presence / frequency penalties, a bias and a mask of allowed tokens on the logits, in front of the draw

`run` computes them from elementary torch operations, or through `molly_amd.ops` where `own` is true.  Page pools are
[pages, kv heads, page size, head dim]; scales are the 8-bit exponent of a power of two (bias 127), [pages, kv heads, page size].
"""
import math
import random

import torch

own = False

EPS = 1e-6
THETA = 1.0e6
E4M3_MAX = 448.0


# ---- the cases -------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one user, a short answer: what a decode step's attention costs when latency is all there is
        dict(name="attend: one user", op="attend", kind="decode", batch=1, new=1, kv=700, heads=16, kv_heads=8, dim=128, page=64, cache="bf16", mix=1),
        # a full decode batch with a quantised cache, sequences of all lengths
        dict(name="attend: decode batch, e4m3", op="attend", kind="decode", batch=32, new=1, kv=4000, heads=32, kv_heads=8, dim=128, page=64, cache="e4m3", mix=2),
        # few long contexts: too few (sequence, head) pairs to fill the chip, so the key axis has to be cut
        dict(name="attend: long contexts", op="attend", kind="decode", batch=4, new=1, kv=32768, heads=16, kv_heads=8, dim=128, page=128, cache="bf16", mix=3),
        # chunked prefill of a long prompt: the largest call, bound by the matrix pipes
        dict(name="attend: prompt chunk", op="attend", kind="chunk", batch=1, new=2048, kv=16384, heads=32, kv_heads=8, dim=128, page=64, cache="bf16", mix=4),
        # continuous batching: a few sequences bring a chunk, the others one token; small pages, quantised
        dict(name="attend: mixed batch, e4m3", op="attend", kind="mixed", batch=24, new=301, kv=2500, heads=32, kv_heads=8, dim=128, page=16, cache="e4m3", mix=5),
        # whole prompts of ragged lengths at head dim 64
        dict(name="attend: ragged prompts", op="attend", kind="prompt", batch=8, new=1111, kv=1111, heads=16, kv_heads=4, dim=64, page=32, cache="bf16", mix=6),
        # the cache write of a decode step, with q/k-norm and rotary, quantised
        dict(name="store: decode step, e4m3", op="store", rows=32, heads=32, kv_heads=8, dim=128, page=64, cache="e4m3", norm=True, rope=True, mix=7),
        # the same for a prompt's rows
        dict(name="store: prompt", op="store", rows=8155, heads=16, kv_heads=8, dim=128, page=64, cache="bf16", norm=True, rope=True, mix=8),
        # finished keys and values moved into a quantised cache
        dict(name="store: rows, e4m3", op="store", rows=30011, heads=0, kv_heads=8, dim=128, page=16, cache="e4m3", norm=False, rope=False, mix=9),
        # one user's logits with a short history
        dict(name="choose: one row", op="choose", rows=1, vocab=151936, history=200, dtype="fp32", bias=False, mask=False, per_row=False),
        # a decode batch with everything on
        dict(name="choose: batch, all", op="choose", rows=32, vocab=151936, history=2000, dtype="fp32", bias=True, mask=True, per_row=True),
        # an odd vocabulary, half-width logits, long histories
        dict(name="choose: odd vocabulary, bf16", op="choose", rows=127, vocab=50257, history=6001, dtype="bf16", bias=False, mask=True, per_row=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        op = rng.choice(["attend", "attend", "attend", "store", "choose"])
        if op == "attend":
            heads, kv_heads = rng.choice([(16, 8), (32, 8), (16, 4), (16, 2), (12, 4), (14, 2), (4, 4), (5, 1), (20, 20)])
            c = dict(op=op, kind=rng.choice(["decode", "decode", "chunk", "mixed", "prompt"]), batch=_log(rng, 1, 64), new=1, kv=_log(rng, 1, 32768),
                     heads=heads, kv_heads=kv_heads, dim=rng.choice([64, 128]), page=rng.choice([16, 32, 64, 128]), cache=rng.choice(["bf16", "e4m3"]),
                     mix=rng.randrange(1 << 20))
            if c["kind"] == "prompt":
                c["new"] = c["kv"]
            elif c["kind"] != "decode":
                c["new"] = min(_log(rng, 2, 2048), c["kv"])
            # the plain form's scores, padded to the longest of everything, stay under 10 GB
            if c["batch"] * c["new"] * c["kv"] * heads > 2_200_000_000:
                continue
        elif op == "store":
            heads, kv_heads = rng.choice([(16, 8), (32, 8), (16, 2), (0, 8), (0, 4), (5, 1)])
            c = dict(op=op, rows=_log(rng, 1, 32768), heads=heads, kv_heads=kv_heads, dim=rng.choice([64, 128]), page=rng.choice([16, 32, 64, 128]),
                     cache=rng.choice(["bf16", "e4m3"]), norm=rng.random() < 0.6, rope=rng.random() < 0.6, mix=rng.randrange(1 << 20))
        else:
            c = dict(op=op, rows=_log(rng, 1, 128), vocab=_log(rng, 500, 160000), history=rng.choice([0, _log(rng, 1, 8000), _log(rng, 1, 8000)]),
                     dtype=rng.choice(["fp32", "bf16"]), bias=rng.random() < 0.5, mask=rng.random() < 0.5, per_row=rng.random() < 0.5)
        w, top = work(c), work(listed()[3])
        if w["bytes"] <= 16 * top["bytes"] and w["flops"] <= top["flops"]:
            return c


def _lengths(case):
    """(new tokens, keys including them) of every sequence: the same for every seed."""
    rng = random.Random(case["mix"])
    B, new, kv = case["batch"], case["new"], case["kv"]
    keys = [kv] + [rng.randint(max(1, kv // 4), kv) for _ in range(B - 1)]
    if case["kind"] == "decode":
        q = [1] * B
    elif case["kind"] == "chunk":
        q = [min(n, new) for n in keys]
    elif case["kind"] == "prompt":
        q = list(keys)
    else:
        q = [min(n, new) if b % 4 == 0 else 1 for b, n in enumerate(keys)]
    return q, keys


def work(case):
    if case["op"] == "attend":
        q, keys = _lengths(case)
        D, H, N = case["dim"], case["heads"], case["kv_heads"]
        per_key = 2 * N * (2 * D if case["cache"] == "bf16" else D + 1)
        pairs = sum(n * k - n * (n - 1) // 2 for n, k in zip(q, keys))
        return {"bytes": sum(keys) * per_key + 2 * sum(q) * H * D * 2, "flops": 4.0 * pairs * H * D}
    if case["op"] == "store":
        n, D, H, N = case["rows"], case["dim"], case["heads"], case["kv_heads"]
        held = 2 * N * (2 * D if case["cache"] == "bf16" else D + 1)                 # a token in the pages
        rows = 2 * 2 * H * D + 2 * N * D * 2                                          # q in and out, k and v in
        return {"bytes": n * (rows + held) + n * (held + 2 * N * D * 2) + 2 * 4 * n, "flops": 0.0}      # stored, then read back
    n, V = case["rows"], case["vocab"]
    b = n * V * ((4 if case["dtype"] == "fp32" else 2) + 4) + n * case["history"] * 8
    b += 4 * V if case["bias"] else 0
    b += n * ((V + 31) // 32) * 4 if case["mask"] else 0
    return {"bytes": b, "flops": 0.0}


# ---- the inputs ------------------------------------------------------------------------------------------------------------------
class State:
    pass


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _quantised(x):
    """e4m3 codes and exponents of x [..., dim]: the smallest power of two that brings the largest magnitude to 448 or less."""
    m, e = torch.frexp(x.abs().amax(-1))
    e = e - 9 + (m > 0.875).to(e.dtype)                                               # 448 = 0.875 * 2^9
    codes = torch.ldexp(x, -e[..., None]).to(torch.float8_e4m3fn)
    return codes, (e + 127).clamp(1, 254).to(torch.uint8)


def prepare(case, seed):
    def attend(case, g):
        s = State()
        q, keys = _lengths(case)
        D, H, N, page = case["dim"], case["heads"], case["kv_heads"], case["page"]
        need = [-(-k // page) for k in keys]
        pages = sum(need) + 3
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        table = torch.full((case["batch"], max(need)), -1, dtype=torch.int32)
        at = torch.zeros(case["batch"], max(need), dtype=torch.int64)
        first = 0
        for b, n in enumerate(need):
            table[b, :n] = 0
            at[b, :n] = torch.arange(first, first + n)
            first += n
        s.table = torch.where(table.cuda() < 0, -1, order[at.cuda()])                     # places behind a sequence's last page: none
        s.q = _normal(g, sum(q), H * D).to(torch.bfloat16)
        k, v = _normal(g, pages, N, page, D), _normal(g, pages, N, page, D)
        s.kscale = s.vscale = None
        if case["cache"] == "e4m3":
            (s.kpool, s.kscale), (s.vpool, s.vscale) = _quantised(k), _quantised(v)
        else:
            s.kpool, s.vpool = k.to(torch.bfloat16), v.to(torch.bfloat16)
        s.cu = torch.tensor([0] + torch.tensor(q).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
        s.kv_len = torch.tensor(keys, dtype=torch.int32, device="cuda")
        s.max_q, s.max_kv, s.heads, s.kv_heads, s.dim, s.page = max(q), max(keys), H, N, D, page
        return s

    def store(case, g):
        s = State()
        n, D, H, N, page = case["rows"], case["dim"], case["heads"], case["kv_heads"], case["page"]
        pages = n // page + 5
        x = _normal(g, n, (H + 2 * N) * D).to(torch.bfloat16)                             # one projection's rows: q | k | v
        s.q, s.k, s.v = x[:, :H * D], x[:, H * D:(H + N) * D], x[:, (H + N) * D:]
        order = torch.randperm(pages, generator=g, device="cuda")
        at = torch.arange(n, device="cuda") + 3
        slot = order[at // page] * page + at % page
        s.slot = torch.where(torch.arange(n, device="cuda") % 97 == 96, -1, slot).to(torch.int32)      # now and then a row of padding
        kind = torch.bfloat16 if case["cache"] == "bf16" else torch.uint8
        s.kpool, s.vpool = (torch.zeros(pages, N, page, D, dtype=kind, device="cuda") for _ in range(2))
        s.kscale = s.vscale = None
        if case["cache"] == "e4m3":
            s.kpool, s.vpool = s.kpool.view(torch.float8_e4m3fn), s.vpool.view(torch.float8_e4m3fn)
            s.kscale, s.vscale = (torch.zeros(pages, N, page, dtype=torch.uint8, device="cuda") for _ in range(2))
        s.qw = s.kw = s.cos = s.sin = s.positions = None
        if case["norm"]:
            s.qw, s.kw = ((1 + 0.1 * _normal(g, D)).to(torch.bfloat16) for _ in range(2))
        if case["rope"]:
            angle = torch.arange(8192, device="cuda", dtype=torch.float64)[:, None] * THETA ** (-torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D)
            s.cos, s.sin = angle.cos().float(), angle.sin().float()
            s.positions = torch.randint(0, 8192, (n,), generator=g, device="cuda", dtype=torch.int32)
        s.heads, s.kv_heads, s.dim, s.page = H, N, D, page
        return s

    def choose(case, g):
        s = State()
        n, V, L = case["rows"], case["vocab"], case["history"]
        s.logits = 4 * _normal(g, n, V)
        if case["dtype"] == "bf16":
            s.logits = s.logits.to(torch.bfloat16)
        s.generated = s.n_generated = s.bias = s.allowed = None
        if L:
            u = torch.rand(n, L, generator=g, device="cuda")
            s.generated = (V * u ** 4).long().clamp(max=V - 1)                             # a few tokens often, most of them rarely
            s.n_generated = (L - (torch.arange(n, device="cuda") * 7) % (L // 2 + 1)).to(torch.int32)
        if case["bias"]:
            s.bias = torch.where(torch.rand(V, generator=g, device="cuda") < 0.01, 5 * _normal(g, V), torch.zeros(V, device="cuda"))
        if case["mask"]:
            s.allowed = torch.randint(-(1 << 31), 1 << 31, (n, (V + 31) // 32), generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
        s.repetition, s.presence, s.frequency = 1.1, 0.4, 0.05
        if case["per_row"]:
            r = torch.rand(3, n, generator=g, device="cuda")
            s.repetition, s.presence, s.frequency = 1 + 0.3 * r[0], r[1] - 0.2, 0.2 * r[2]
        return s

    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"attend": attend, "store": store, "choose": choose}[case["op"]](case, g)
    s.op = case["op"]
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------------------
def run(s):
    if own:
        return _own(s)
    return {"attend": _attend, "store": _store, "choose": _choose}[s.op](s)


def _own(s):
    from molly_amd import ops
    if s.op == "attend":
        return ops.attn_paged(s.q, s.kpool, s.vpool, s.table, s.cu, s.kv_len, s.heads, kscale=s.kscale, vscale=s.vscale, max_q=s.max_q,
                              max_kv=s.max_kv)
    if s.op == "store":
        q = ops.paged_kv_append(s.k, s.v, s.kpool, s.vpool, s.slot, kscale=s.kscale, vscale=s.vscale, q=s.q if s.heads else None, qw=s.qw, kw=s.kw,
                                cos=s.cos, sin=s.sin, positions=s.positions, eps=EPS)
        k, v = ops.paged_kv_read(s.kpool, s.vpool, s.slot, kscale=s.kscale, vscale=s.vscale)
        return (q, k, v) if s.heads else (k, v)
    return ops.process_logits(s.logits, generated=s.generated, n_generated=s.n_generated, repetition_penalty=s.repetition,
                              presence_penalty=s.presence, frequency_penalty=s.frequency, bias=s.bias, allowed=s.allowed)


def _held(pool, scale, at):
    """The values that a pool holds at `at`."""
    if scale is None:
        return pool[at].float()
    return torch.ldexp(pool.view(torch.uint8)[at].view(torch.float8_e4m3fn).float(), scale[at].int()[..., None] - 127)


def _attend(s):
    B, D, N, G = s.kv_len.numel(), s.dim, s.kv_heads, s.heads // s.kv_heads
    n = s.cu[1:] - s.cu[:-1]
    i, key = torch.arange(s.max_q, device="cuda"), torch.arange(s.table.shape[1] * s.page, device="cuda")
    pages = s.table.clamp(min=0).long()
    k, v = (_held(p, c, pages).transpose(1, 2).reshape(B, N, -1, D) for p, c in ((s.kpool, s.kscale), (s.vpool, s.vscale)))
    at = (s.cu[:-1, None] + i).clamp(max=s.q.shape[0] - 1).long()
    q = s.q.float()[at].view(B, s.max_q, N, G, D).permute(0, 2, 1, 3, 4).reshape(B, N, s.max_q * G, D)
    x = torch.matmul(q, k.transpose(2, 3)).view(B, N, s.max_q, G, -1) * D ** -0.5
    seen = key <= ((s.kv_len - n)[:, None] + i)[..., None]                            # [B, new token, key]
    x = x.masked_fill(~seen[:, None, :, None], float("-inf"))
    p = torch.exp(x - x.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, N, s.max_q * G, -1), v).view(B, N, s.max_q, G, D).permute(0, 2, 1, 3, 4).reshape(B, s.max_q, -1)
    row = torch.arange(s.q.shape[0], device="cuda")
    b = torch.searchsorted(s.cu[1:].contiguous(), row.int(), right=True)
    return o[b, row - s.cu[b]].to(torch.bfloat16)


def _turned(s, x, heads, w):
    x = x.float().reshape(x.shape[0], heads, s.dim)
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()
    if s.cos is not None:
        c, t = s.cos[s.positions.long()][:, None], s.sin[s.positions.long()][:, None]
        a, b = x.chunk(2, -1)
        x = torch.cat([a * c - b * t, b * c + a * t], -1)
    return x


def _kept(s, x, pool, scale):
    """Rows x [n, kv heads, dim] into their places, and what those hold; a row without a place (slot -1) changes nothing and comes back as zeros."""
    live = s.slot >= 0
    slot = torch.where(live, s.slot, s.slot[0]).long()                                # (the first row is never one: it is written again, as it is)
    x = torch.where(live[:, None, None], x, x[:1])
    at = (slot // s.page, slice(None), slot % s.page)
    if scale is None:
        pool[at] = x.to(torch.bfloat16)
    else:
        codes, scale[at] = _quantised(x)
        pool.view(torch.uint8)[at] = codes.view(torch.uint8)
    return torch.where(live[:, None, None], _held(pool, scale, at), 0.0).flatten(1).to(torch.bfloat16)


def _store(s):
    k = _kept(s, _turned(s, s.k, s.kv_heads, s.kw), s.kpool, s.kscale)
    v = _kept(s, s.v.float().reshape(-1, s.kv_heads, s.dim), s.vpool, s.vscale)
    return (_turned(s, s.q, s.heads, s.qw).flatten(1).to(torch.bfloat16), k, v) if s.heads else (k, v)


def _choose(s):
    x = s.logits.float()
    n, V = x.shape
    column = lambda p: p[:, None] if torch.is_tensor(p) else p  # noqa: E731
    if s.generated is not None:
        live = torch.arange(s.generated.shape[1], device="cuda") < s.n_generated[:, None]
        count = torch.zeros(n, V, device="cuda").scatter_add_(1, s.generated, live.float())
        r = column(s.repetition)
        x = torch.where(count > 0, torch.where(x < 0, x * r, x / r) - column(s.presence), x) - column(s.frequency) * count
    if s.bias is not None:
        x = x + s.bias
    if s.allowed is not None:
        bit = torch.arange(V, device="cuda")
        x = x.masked_fill((s.allowed[:, bit // 32] >> (bit % 32).int()) & 1 == 0, float("-inf"))
    return x


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------------------
def exact(case, seed):
    def attend(s):
        cu, keys, G = s.cu.tolist(), s.kv_len.tolist(), s.heads // s.kv_heads
        out = torch.zeros(s.q.shape[0], s.heads, s.dim, dtype=torch.float64, device="cuda")
        for b, length in enumerate(keys):
            rows = s.q[cu[b]:cu[b + 1]].double().view(-1, s.heads, s.dim)
            new = rows.shape[0]
            used = s.table[b, : -(-length // s.page)].long()
            last = length - new + torch.arange(new, device="cuda")
            hidden = torch.arange(length, device="cuda")[None] > last[:, None]
            for h in range(s.kv_heads):
                kv = []
                for pool, scale in ((s.kpool, s.kscale), (s.vpool, s.vscale)):
                    x = pool[:, h][used] if scale is None else pool.view(torch.uint8)[:, h][used].view(torch.float8_e4m3fn)
                    x = x.double() if scale is None else x.double() * 2.0 ** (scale[:, h][used].double() - 127)[..., None]
                    kv.append(x.reshape(-1, s.dim)[:length])
                for j in range(h * G, (h + 1) * G):
                    score = (rows[:, j] @ kv[0].T) / math.sqrt(s.dim)
                    out[cu[b]:cu[b + 1], j] = torch.softmax(score.masked_fill(hidden, -math.inf), -1) @ kv[1]
        return out.flatten(1)

    def store(s):
        n, half = s.slot.numel(), s.dim // 2

        def head_rows(x, gain):
            y = x.double().reshape(n, -1, s.dim)
            if gain is not None:
                y = y / (y.pow(2).sum(-1, keepdim=True) / s.dim + EPS).sqrt() * gain.double()
            if s.cos is not None:
                z = torch.complex(y[..., :half], y[..., half:]) * torch.complex(s.cos.double(), s.sin.double())[s.positions.long()].unsqueeze(1)
                y = torch.cat([z.real, z.imag], -1)
            return y

        def kept(y):
            """What the cache holds of y, where it holds e4m3: codes have 3 bits behind the leading one, down to 2^-9."""
            if s.kscale is None:
                return y
            top = y.abs().amax(-1, keepdim=True)
            unit = torch.exp2(torch.ceil(torch.log2(top / E4M3_MAX)))
            unit = torch.where(top <= E4M3_MAX * unit / 2, unit / 2, torch.where(top > E4M3_MAX * unit, unit * 2, unit))      # (log2 is rounded)
            z = y / unit
            step = torch.exp2(torch.floor(torch.log2(z.abs().clamp(min=2.0 ** -6))) - 3)
            return torch.round(z / step) * step * unit                                     # (torch.round: to even)

        live = (s.slot >= 0)[:, None]
        k = kept(head_rows(s.k, s.kw)).flatten(1) * live
        v = kept(s.v.double().reshape(n, -1, s.dim)).flatten(1) * live
        return (head_rows(s.q, s.qw).flatten(1), k, v) if s.heads else (k, v)

    def choose(s):
        x = s.logits.double()
        n, V = x.shape
        per_row = [p.tolist() if torch.is_tensor(p) else [p] * n for p in (s.repetition, s.presence, s.frequency)]
        for r in range(n):
            if s.generated is not None:
                ids, times = torch.unique(s.generated[r, : int(s.n_generated[r])], return_counts=True)
                y = x[r, ids]
                x[r, ids] = y * per_row[0][r] ** torch.where(y < 0, 1.0, -1.0) - per_row[1][r] - per_row[2][r] * times
            if s.bias is not None:
                x[r] += s.bias.double()
            if s.allowed is not None:
                bits = torch.stack([(s.allowed[r].long() >> j) & 1 for j in range(32)], 1).flatten()[:V]
                x[r, bits == 0] = -math.inf
        return x

    return {"attend": attend, "store": store, "choose": choose}[case["op"]](prepare(case, seed))
