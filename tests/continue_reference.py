"""Plain 64-bit statements of the operators that continue a prompt many times, on CPU tensors."""

from __future__ import annotations

import math

import torch

BS = 16


def rotate(y, mode, cos, sin, pos):
    """``y [rows, heads, dim]`` rotated by the tables' rows ``pos``."""

    if mode == 0:
        return y
    d = y.shape[-1]
    lo, hi = (torch.arange(d // 2), torch.arange(d // 2) + d // 2) if mode == 1 else (torch.arange(0, d, 2), torch.arange(1, d, 2))
    c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
    c1, c2, s1, s2 = (c[..., lo], c[..., hi], s[..., lo], s[..., hi]) if mode == 1 else (c, c, s, s)
    out = torch.empty_like(y)
    out[..., lo] = y[..., lo] * c1 - y[..., hi] * s1
    out[..., hi] = y[..., hi] * c2 + y[..., lo] * s2
    return out


def norm_append(qkv, table, slot, pos, q_w, k_w, cos, sin, mode, heads, kv_heads, eps):
    """q, k, v in 64 bits ``[rows, heads, dim]``, for q and k the size of what they are sums of, and the cache rows."""

    d = q_w.numel()
    x = qkv.double().view(qkv.shape[0], -1, d)
    w = torch.cat((q_w.double().expand(heads, d), k_w.double().expand(kv_heads, d)))
    y = x[:, : heads + kv_heads]
    y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * w
    p = torch.tensor(pos)
    z = rotate(y, mode, cos, sin, p)
    size = y.abs()
    if mode == 1:
        size = size + size.roll(d // 2, -1)
    elif mode == 2:
        size = size + size.view(*size.shape[:-1], d // 2, 2).flip(-1).flatten(-2)
    rows = [int(table[s, q // BS]) * BS + q % BS for s, q in zip(slot, pos)]
    return z[:, :heads], z[:, heads:], x[:, heads + kv_heads :], size, rows


def attend(q, pool, table_row, pos, scale, blocks):
    """One row ``q [heads, dim]`` over positions 0 .. pos of one layer's cache ``pool [2, rows, kv heads, dim]``; keys of
    blocks out of range are left out. Also sum p |v| / sum p."""

    at = torch.arange(pos + 1)
    ids = table_row.long()[at // BS]
    ok = (ids >= 0) & (ids < blocks)
    rows = (ids * BS + at % BS)[ok]
    h, d = q.shape
    hkv = pool.shape[2]
    k, v = pool[0, rows].double(), pool[1, rows].double()
    x = torch.einsum("hgd,lhd->hgl", q.double().view(hkv, h // hkv, d), k) * scale
    p = torch.softmax(x, -1)
    return torch.einsum("hgl,lhd->hgd", p, v).reshape(h, d), torch.einsum("hgl,lhd->hgd", p, v.abs()).reshape(h, d)


def sample(logits, u, t, k=0, p=1.0, m=0.0):
    """Token and log-probability of one row (Python floats are 64 bits)."""

    x = logits.double()
    x = torch.where(x.isnan(), -math.inf, x)
    top = x.max()
    if top == -math.inf:
        return -1, math.nan
    if not t > 0:
        return int((x == top).nonzero()[0]), 0.0
    w = torch.where(x == top, 1.0, torch.exp((x - top) / t)).nan_to_num(0.0)  # (-inf over an infinite temperature)
    order = sorted(range(x.numel()), key=lambda i: (-x[i].item(), i)) if x.numel() < 64 else torch.sort(x, descending=True, stable=True)[1].tolist()
    if k > 0:
        order = order[:k]
    idx = torch.tensor(order)
    sorted_w = w[idx]
    if p < 1:
        before = sorted_w.cumsum(0) - sorted_w
        keep = before < max(p, 0.0) * sorted_w.sum()
        keep[0] = True
        idx, sorted_w = idx[keep], sorted_w[keep]
    if m > 0:
        keep = sorted_w >= min(m, 1.0)
        idx = idx[keep]
    idx = idx.sort()[0]
    run = w[idx].cumsum(0)
    u = 0.0 if not u > 0 else u
    j = int((run > u * run[-1]).nonzero()[0]) if u < 1 else int((w[idx] > 0).nonzero()[-1])
    return int(idx[j]), float(torch.log(w[idx[j]] / run[-1]))
