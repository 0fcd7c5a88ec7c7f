"""Plain 64-bit statements of the 8-bit paged cache and its attention, for the tests (CPU)."""

from __future__ import annotations

import math

import torch

BS = 16


def block_scale(amax: float) -> float:
    """Smallest power of two s >= 2^-126 with amax <= 448 s."""

    if amax == 0.0:
        return 2.0**-126
    m, e = math.frexp(amax)  # amax = m 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    return 2.0 ** max(-126, e - 9 + (1 if m > 0.875 else 0))


def to_e4m3(v: torch.Tensor) -> torch.Tensor:
    """Nearest e4m3 value, ties to even, saturating at 448; NaN stays NaN."""

    a = v.abs().clamp(max=448.0)
    _, e = torch.frexp(a)
    step = torch.ldexp(torch.ones_like(a), (e - 1).clamp(min=-6) - 3)
    q = (torch.round(a / step) * step).clamp(max=448.0)
    return torch.where(v.isnan(), v, torch.copysign(q, v))


def rotate(x: torch.Tensor, mode: int, cos, sin, pos: int) -> torch.Tensor:
    """x [heads, dim] in fp64."""

    d = x.shape[-1]
    if mode == 1:
        h = d // 2
        return x * cos[pos].double() + torch.cat((-x[:, h:], x[:, :h]), -1) * sin[pos].double()
    if mode == 2:
        c, s = cos[pos].double(), sin[pos].double()
        a, b = x[:, 0::2], x[:, 1::2]
        return torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    return x


def append(qkv, codes, scales, table, slot, pos, cos, sin, bias, mode, heads):
    """Values ``codes`` [2, blocks, kv heads, 16, d] (fp64 code values, in place) and ``scales`` [2,
    blocks, kv heads] (fp64, in place) of one cache layer after the call, and the rotated q (fp64)."""

    hkv, d = codes.shape[2], codes.shape[4]
    n = len(pos)
    x = qkv.double().view(n, -1, d)
    q = torch.zeros(n, heads, d, dtype=torch.float64)
    i = 0
    while i < n:
        if pos[i] < 0:
            i += 1
            continue
        j = i
        while j < n and pos[j] >= 0 and slot[j] == slot[i] and pos[j] // BS == pos[i] // BS:
            j += 1
        new = []
        for r in range(i, j):
            qk = x[r, : heads + hkv]
            if bias is not None:
                qk = qk + bias.double().view(heads + hkv, d)
            qk = rotate(qk, mode, cos, sin, pos[r])
            q[r] = qk[:heads]
            new.append(torch.stack((qk[heads:], x[r, heads + hkv :])))
        new = torch.stack(new, 2)  # [2, hkv, rows, d]
        blk, off = int(table[slot[i], pos[i] // BS]), pos[i] % BS
        for kv in range(2):
            for h in range(hkv):
                v = new[kv, h]
                fin = v[v.isfinite()].abs()
                s = block_scale(float(fin.max()) if fin.numel() else 0.0)
                if off:
                    s = max(s, float(scales[kv, blk, h]))
                    old = codes[kv, blk, h, :off]
                    codes[kv, blk, h, :off] = to_e4m3(old * (float(scales[kv, blk, h]) / s))
                scales[kv, blk, h] = s
                codes[kv, blk, h, off : off + j - i] = to_e4m3(v / s)
        i = j
    return q


def attend(q, codes, scales, table_row, first, scale):
    """Rows q [n, heads, d] at positions first .. first + n - 1 over a row of the block table, causal:
    (output, sum of p |v| / sum of p) in fp64, [n, heads, d]."""

    n, hq, d = q.shape
    hkv = codes.shape[2]
    length = first + n
    pages = (length + BS - 1) // BS
    kv = codes[:, table_row[:pages].long()].double() * scales[:, table_row[:pages].long()].double()[..., None, None]
    k, v = kv.permute(0, 2, 1, 3, 4).reshape(2, hkv, -1, d)[:, :, :length]
    k, v = k.repeat_interleave(hq // hkv, 0), v.repeat_interleave(hq // hkv, 0)
    x = torch.einsum("nhd,hld->hnl", q.double(), k) * scale
    x = x.masked_fill(torch.arange(length)[None, :] > first + torch.arange(n)[:, None], -math.inf)
    p = torch.softmax(x, -1)
    return torch.einsum("hnl,hld->nhd", p, v), torch.einsum("hnl,hld->nhd", p, v.abs())
