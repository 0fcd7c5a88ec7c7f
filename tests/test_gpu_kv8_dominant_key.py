"""Attention over the 8-bit cache where one key takes the mass and its value is zero (an attention sink): the
output is the sum of many small weights.

Tolerance. 2^-8 of the value (bf16) and 2^-10 of A = sum p |v| / sum p, as in test_gpu_kv8. The weights of V are
f16, relative to their largest W = max p s_v, which stands at 2^7 or above: one below 2^-14 there is off by up to
half of f16's smallest step, 2^-25, so by 2^-32 W for a code of 1, and the output by 2^-32 W sum |code| / sum p.
"""

from __future__ import annotations

import math

import pytest
import torch

import continuous_depth_batching_b200.ops as ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BS = 16


def _cache(kv_heads, d, length, sink):
    """One row of ``length`` equal keys (codes 0) with positive values, and a key of ones at ``sink``, value 0."""

    g = torch.Generator().manual_seed(d + kv_heads + sink)
    blocks = -(-length // BS)
    codes = torch.zeros(1, 2, blocks, kv_heads, BS, d)
    codes[0, 1] = torch.randint(8, 28, codes[0, 1].shape, generator=g).float() * 16
    codes[0, 0, sink // BS, :, sink % BS] = 1.0
    codes[0, 1, sink // BS, :, sink % BS] = 0.0
    scales = torch.ones(1, 2, blocks, kv_heads)
    scales[0, 1] = 2.0**-6
    codes = codes.to(torch.float8_e4m3fn)
    return codes, scales, torch.arange(blocks, dtype=torch.int32)[None]


def _expect(q, codes, scales, length, scale):
    """Output, and what it may be off by, of one position that sees ``length`` keys: [heads, d]."""

    heads, d = q.shape
    hkv = codes.shape[3]
    k, v = codes[0].double().permute(0, 2, 1, 3, 4).reshape(2, hkv, -1, d)[:, :, :length].repeat_interleave(heads // hkv, 1)
    ks, vs = (s.repeat_interleave(BS, 1)[:, :length].repeat_interleave(heads // hkv, 0) for s in scales[0].double().transpose(1, 2))
    p = torch.softmax(torch.einsum("hd,hld->hl", q.double(), k) * ks * scale, -1)
    o, a = (torch.einsum("hl,hld->hd", p * vs, c) for c in (v, v.abs()))
    tiny = 2.0**-32 * (p * vs).amax(1)[:, None] * v.abs().sum(1)
    return o, 2.0**-8 * o.abs() + 2.0**-10 * a + tiny


def _queries(heads, group, d):
    return (1 + torch.arange(heads) % group / 64).bfloat16()[:, None].expand(heads, d)


@pytest.mark.parametrize("d,kv_heads,group", [(64, 16, 1), (128, 16, 1), (96, 16, 4), (128, 16, 4)])
@pytest.mark.parametrize("octaves", [12.0, 20.7, 24.3, 28.6])  # the others' weights: 2^-octaves of the large one's
@pytest.mark.parametrize("sink", [0, 1000])
def test_decode(d, kv_heads, group, octaves, sink):
    """As many segments as warps, so that each is one warp's."""

    rows, length, heads = 111, 2048, kv_heads * group
    codes, scales, table = _cache(kv_heads, d, length, sink)
    q = _queries(heads, group, d)
    scale = octaves * math.log(2.0) / d
    out = torch.empty(rows, heads * d, dtype=torch.bfloat16, device=DEV)
    torch.ops.cdb.kv8_decode_attention(
        q.reshape(1, -1).repeat(rows, 1).to(DEV), out, codes.to(DEV), scales.to(DEV), 0, table.to(DEV),
        torch.zeros(rows, dtype=torch.int32, device=DEV), torch.full((rows,), length - 1, dtype=torch.int32, device=DEV),
        heads, scale)
    torch.cuda.synchronize()
    assert ops.status_code() == 0
    want, tol = _expect(q, codes, scales, length, scale)
    off = (out.cpu().double().view(rows, heads, d) - want).abs()
    assert (off <= tol).all(), (off / tol).max()


@pytest.mark.parametrize("length,octaves", [(300, 20.7), (40_000, 24.3)])
def test_decode_of_one_row(length, octaves):
    """A row in one CTA and one in pieces over all of them."""

    d, heads = 128, 4
    codes, scales, table = _cache(2, d, length, 3)
    q = _queries(heads, 2, d)
    scale = octaves * math.log(2.0) / d
    out = torch.empty(1, heads * d, dtype=torch.bfloat16, device=DEV)
    torch.ops.cdb.kv8_decode_attention(
        q.reshape(1, -1).contiguous().to(DEV), out, codes.to(DEV), scales.to(DEV), 0, table.to(DEV),
        torch.zeros(1, dtype=torch.int32, device=DEV), torch.full((1,), length - 1, dtype=torch.int32, device=DEV), heads, scale)
    torch.cuda.synchronize()
    assert ops.status_code() == 0
    want, tol = _expect(q, codes, scales, length, scale)
    assert ((out.cpu().double().view(heads, d) - want).abs() <= tol).all()


@pytest.mark.parametrize("d,group", [(64, 1), (96, 2), (128, 1)])
@pytest.mark.parametrize("octaves", [12.0, 20.7, 24.3, 28.6])
@pytest.mark.parametrize("sink", [0, 1000])
def test_prefill(d, group, octaves, sink):
    length, n, heads = 5000, 130, 2 * group
    codes, scales, table = _cache(2, d, length, sink)
    q = _queries(heads, group, d)
    scale = octaves * math.log(2.0) / d
    first = length - n
    tiles = [(i, min(64, n - i), 0, first + i) for i in range(0, n, 64)]
    out = torch.empty(n, heads * d, dtype=torch.bfloat16, device=DEV)
    torch.ops.cdb.kv8_prefill_attention(
        q.reshape(1, -1).repeat(n, 1).to(DEV), out, codes.to(DEV), scales.to(DEV), 0, table.to(DEV),
        torch.tensor(tiles, dtype=torch.int32, device=DEV), heads, scale)
    torch.cuda.synchronize()
    assert ops.status_code() == 0
    for r in (0, 63, 64, 127, 128, 129):
        want, tol = _expect(q, codes, scales, first + r + 1, scale)
        off = (out[r].cpu().double().view(heads, d) - want).abs()
        assert (off <= tol).all(), (r, (off / tol).max())
