"""Inputs and 64-bit definitions shared by the tests of the paged cache (CPU and GPU)."""
import math

import torch


def quantise(x):
    """x [..., dim] float64 -> (values the cache holds, exponent bytes): the smallest power of two with amax <= 448 * 2^e over the finite values."""
    fin = torch.where(torch.isfinite(x), x, torch.zeros_like(x))
    m, e = torch.frexp(fin.abs().amax(-1))
    e = torch.where(m == 0, torch.full_like(e, -1000), e - 9 + (m > 0.875).to(e.dtype)).clamp(-126, 127)
    z = torch.where(torch.isfinite(x), torch.ldexp(x, -e[..., None].double()), torch.full_like(x, math.nan))
    step = torch.exp2(torch.floor(torch.log2(z.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(z / step) * step * torch.exp2(e[..., None].double()), (e + 127).to(torch.uint8)


def turned(x, heads, w=None, cos=None, sin=None, positions=None, eps=1e-6):
    """q/k-norm and rotary in float64: [n, heads, dim]."""
    y = x.double().reshape(x.shape[0], heads, -1)
    if w is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    if cos is not None:
        half = y.shape[-1] // 2
        c, s = cos.double()[positions.long()][:, None], sin.double()[positions.long()][:, None]
        y = torch.cat([y[..., :half] * c - y[..., half:] * s, y[..., half:] * c + y[..., :half] * s], -1)
    return y


def held(pool, scale=None):
    """the values a pool holds, float64"""
    return pool.double() if scale is None else pool.float().double() * torch.exp2(scale.double() - 127)[..., None]


def attend(q, kheld, vheld, table, cu, kv_len, n_heads, scale):
    """-> (out, sum_j p_j |v_j|) [n_tokens, n_heads, dim] float64 from held() pools; rows outside the sequences are NaN in both."""
    P, nkv, page, hd = kheld.shape
    G = n_heads // nkv
    out = torch.full((q.shape[0], n_heads, hd), math.nan, dtype=torch.float64, device=q.device)
    mag = out.clone()
    for b in range(len(kv_len)):
        s, e = cu[b], cu[b + 1]
        n, length = e - s, max(kv_len[b], 0)
        if n <= 0:
            continue
        used = table[b, : -(-length // page)].long() if length else table[b, :0].long()
        k = kheld[used].transpose(0, 1).reshape(nkv, -1, hd)[:, :length].repeat_interleave(G, 0)
        v = vheld[used].transpose(0, 1).reshape(nkv, -1, hd)[:, :length].repeat_interleave(G, 0)
        rows = q[s:e].double().view(n, n_heads, hd).transpose(0, 1)
        sc = rows @ k.transpose(1, 2) * scale
        seen = torch.arange(length, device=q.device)[None] <= (kv_len[b] - n + torch.arange(n, device=q.device))[:, None]
        sc = sc.masked_fill(~seen, -math.inf)
        p = torch.where(seen.any(-1)[None, :, None], torch.softmax(sc, -1), torch.zeros_like(sc)) if length else sc
        # what a row does not see has no part in it, whatever is there (0 * NaN)
        bad = ~torch.isfinite(v).all(-1)                                    # [heads, keys]
        clean = torch.where(torch.isfinite(v), v, torch.zeros_like(v))
        o = p @ clean
        for j in bad.any(0).nonzero().flatten().tolist():
            part = torch.where(torch.isfinite(v[:, None, j]), torch.zeros_like(o), p[:, :, j, None] * v[:, None, j])
            o = torch.where(seen[:, j][None, :, None], o + part, o)
        out[s:e] = o.transpose(0, 1)
        mag[s:e] = (p @ clean.abs()).transpose(0, 1)
    return out, mag


def pools(g, n_pages, nkv, page, hd, fp8, device):
    k, v = (torch.randn(n_pages, nkv, page, hd, generator=g, device=device) for _ in range(2))
    if not fp8:
        return k.bfloat16(), v.bfloat16(), None, None
    out = []
    for x in (k, v):
        val, e = quantise(x.double())
        out += [torch.ldexp(val, 127 - e.double()[..., None]).float().to(torch.float8_e4m3fn), e]
    return out[0], out[2], out[1], out[3]
