"""The 8-bit cache's operators in 64 bits, one sequence and head at a time: what the kernels are tested against."""
import math

import torch

TOP = {"int8": 127.0, "e4m3": 448.0}
DTYPE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def values(x8):
    return x8.to(torch.float32).double()


def nearest(x, kind):
    """float64 values rounded to the 8-bit type's values, ties to even."""
    top = TOP[kind]
    x = x.clamp(-top, top)
    if kind == "int8":
        return torch.round(x)
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), e.clamp(min=-5) - 4)
    return torch.round(x / step) * step


def scale_of(top, kind):
    """FP32 scale of a block whose largest value is `top` (float64)."""
    return (top / TOP[kind]).float().double()


def rotate(x, positions, inv_freq, factor, layout, inverse=False):
    """x [T, heads, d] float64."""
    f = torch.tensor(inv_freq, dtype=torch.float64, device=x.device)
    a = positions.double()[:, None] * f
    c, s = (a.cos() * factor)[:, None], (a.sin() * factor)[:, None]
    if inverse:
        s = -s
    n = f.numel()
    y = x.clone()
    i, j = (slice(0, n), slice(n, 2 * n)) if layout == "half" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    y[..., i] = x[..., i] * c - x[..., j] * s
    y[..., j] = x[..., i] * s + x[..., j] * c
    return y


def append(k8, scale, table, kv_len, q_start, q_len, x, kind):
    """x [T, hkv, d] float64 into pages: returns new (values float64, scale float64)."""
    page = k8.size(2)
    val, sc = values(k8), scale.double().clone()
    for b, (kv, r0, n) in enumerate(zip(kv_len, q_start, q_len)):
        if n == 0:
            continue
        old = kv - n
        for blk in range(old // page, -(-kv // page)):
            p = int(table[b, blk])
            n0, n1 = max(old - blk * page, 0), min(kv - blk * page, page)
            new = x[r0 + blk * page + n0 - old: r0 + blk * page + n1 - old].transpose(0, 1)     # [hkv, tokens, d]
            s_old = sc[p] if n0 > 0 else torch.zeros_like(sc[p])
            s_new = torch.maximum(s_old, scale_of(new.abs().amax((1, 2)), kind))
            safe = torch.where(s_new > 0, s_new, 1.0)[:, None, None]
            if n0 > 0:
                again = nearest(val[p, :, :n0] * s_old[:, None, None] / safe, kind)
                val[p, :, :n0] = torch.where((s_new == s_old)[:, None, None], val[p, :, :n0], again)
            val[p, :, n0:n1] = nearest(new / safe, kind)
            sc[p] = s_new
    return val, sc


def dense(val, scale, table_row, n):
    """First n tokens of a sequence [hkv, n, d]."""
    page = val.size(2)
    p = torch.tensor([int(x) for x in table_row[:-(-n // page)]], dtype=torch.int64, device=val.device)
    if n == 0:
        return val.new_zeros(val.size(1), 0, val.size(3))
    return (val[p] * scale[p][..., None, None]).transpose(0, 1).reshape(val.size(1), -1, val.size(3))[:, :n]


def attend(k, v, q, window, scale):
    """k, v [hkv, n, d], q [m, hq, d], the last m of the n tokens: (out, lse, weights [hkv, n], sum p |v|, max scale |q| |k|)."""
    hkv, n, d = k.shape
    m, hq, _ = q.shape
    g = hq // hkv
    qh = q.view(m, hkv, g, d).permute(1, 2, 0, 3)
    s = torch.einsum("hgqd,hkd->hgqk", qh, k) * scale
    size = torch.einsum("hgqd,hkd->hgqk", qh.abs(), k.abs()) * scale
    last = n - m + torch.arange(m, device=k.device)[:, None]
    at = torch.arange(n, device=k.device)
    hidden = (at > last) | ((at <= last - window) if window else torch.zeros_like(at > last))
    s = s.masked_fill(hidden, -math.inf)
    top = s.amax(-1, keepdim=True) if n else s.new_full((hkv, g, m, 1), -math.inf)
    top = torch.where(top > -math.inf, top, 0.0)
    e = (s - top).exp()
    tot = e.sum(-1, keepdim=True)
    p = e / torch.where(tot > 0, tot, 1.0)
    out = torch.einsum("hgqk,hkd->qhgd", p, v).reshape(m, hq, d)
    mag = torch.einsum("hgqk,hkd->qhgd", p, v.abs()).reshape(m, hq, d)
    lse = (tot.log() + top)[..., 0].permute(2, 0, 1).reshape(m, hq)
    most = float(size.masked_fill(hidden, 0.0).max()) if n and m else 0.0
    return out, lse, p.sum((1, 2)), mag, most


def kept(weights, n, budget, recent, sink):
    """Kept positions of one head: weights [n] (any order of equal ones: lowest position first)."""
    if n <= budget:
        return list(range(n))
    w = [math.inf if x != x else x for x in weights]
    nan = [x != x for x in weights]
    mid = sorted(range(sink, n - recent), key=lambda i: (not nan[i], -w[i], i))[:budget - sink - recent]
    return sorted(list(range(sink)) + mid + list(range(n - recent, n)))


def move(val, scale, table_row, keep, head, dest_row, kind):
    """One head's kept tokens into dest pages: {page: (values [tokens, d], scale)}."""
    page = val.size(2)
    out = {}
    for blk in range(-(-len(keep) // page)):
        src = keep[blk * page: (blk + 1) * page]
        pages = [int(table_row[i // page]) for i in src]
        q = torch.stack([val[p, head, i % page] for p, i in zip(pages, src)])
        s = torch.stack([scale[p, head] for p in pages]).double()
        if src == list(range(blk * page, blk * page + len(src))):
            out[int(dest_row[blk])] = (q, s[0])
            continue
        now = scale_of((q.abs().amax(1) * s).max(), kind)
        out[int(dest_row[blk])] = (nearest(q * s[:, None] / now, kind) if now > 0 else torch.zeros_like(q), now)
    return out
