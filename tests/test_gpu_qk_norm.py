"""Norms of each head's query and key, rotation and append to the bf16 paged cache, against the formula in 64 bits.

Tolerance: one rounding to bf16 (2^-8 of the value), and the fp32 arithmetic before it: the mean of D <= 128 squares is
off by at most D / 2 roundings of 2^-24 relative (half of that after the square root), the rotation adds a few of
the pair's size: 2^-17 of the pair.
"""

from __future__ import annotations

import pytest
import torch

import continuous_depth_batching_b200.ops as ops
import continue_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
BS = 16
LAYOUTS = [(1, 1, 64), (4, 4, 128), (8, 2, 128), (6, 1, 96), (55, 55, 96), (32, 8, 64), (40, 8, 128), (3, 3, 64)]


def _tables(mode, d, positions):
    inv = 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    ang = torch.arange(positions, dtype=torch.float64)[:, None] * inv
    if mode == 1:
        ang = torch.cat((ang, ang), -1)
        return ang.cos().bfloat16(), ang.sin().bfloat16()
    return (ang.cos().float(), ang.sin().float()) if mode == 2 else (None, None)


def _near(got, want, size):
    assert ((got.double() - want).abs() <= 2.0**-8 * want.abs() + 2.0**-17 * size).all()


def _dev(t):
    return None if t is None else t.to(DEV)


@pytest.mark.parametrize("heads,kv,d", LAYOUTS)
@pytest.mark.parametrize("mode", [0, 1, 2])
@pytest.mark.parametrize("rows", [1, 2, 37, 300])
def test_against_the_formula(heads, kv, d, mode, rows):
    g = torch.Generator().manual_seed(heads * 7 + mode + rows)
    slots, width = 5, 30
    blocks = slots * width
    table = torch.randperm(blocks, generator=g).view(slots, width).int()
    # rows of several slots at places of their own; some are padding
    places = torch.randperm(slots * width * BS, generator=g)[:rows]
    slot, pos = (places // (width * BS)).tolist(), (places % (width * BS)).tolist()
    pad = [i for i in range(rows) if i % 7 == 3]
    for i in pad:
        slot[i], pos[i] = -1, -1
    all_heads = heads + 2 * kv
    qkv = torch.randn(rows, all_heads * d + 24, generator=g).bfloat16()
    qkv[::3] *= 30
    qkv[1::4] *= 1e-3
    q_w, k_w = (torch.randn(d, generator=g).bfloat16() for _ in range(2))
    cos, sin = _tables(mode, d, width * BS)
    pool = torch.randn(2, 2, blocks * BS + 5, kv, d, generator=g).bfloat16()
    dev_qkv, dev_pool = qkv.to(DEV), pool.to(DEV)
    view = dev_qkv[:, : all_heads * d]  # a row stride of its own
    q_out = torch.full((rows, heads * d + 8), 7.0, dtype=torch.bfloat16, device=DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    args = (dev_pool, 1, table.to(DEV), torch.tensor(slot, **i32), torch.tensor(pos, **i32), q_w.to(DEV), k_w.to(DEV), _dev(cos), _dev(sin), mode, heads, 1e-6)
    torch.ops.cdb.qk_norm_rope_append(view, q_out[:, : heads * d], *args)
    torch.cuda.synchronize()
    assert ops.status_code() == 0
    live = [i for i in range(rows) if pos[i] >= 0]
    q, k, v, size, at = ref.norm_append(qkv[live][:, : all_heads * d], table, [slot[i] for i in live], [pos[i] for i in live], q_w, k_w, cos, sin, mode, heads, kv,
                                        1e-6)
    got = q_out.cpu()
    _near(got[live][:, : heads * d].view(len(live), heads, d), q, size[:, :heads])
    assert (got[pad] == 7).all() and (got[:, heads * d :] == 7).all()
    new = dev_pool.cpu()
    _near(new[1, 0, at], k, size[:, heads:])
    assert torch.equal(new[1, 1, at].double(), v)
    want = pool.clone()
    want[1, :, at] = new[1, :, at]
    assert torch.equal(new, want)  # nothing else was written
    # without q; and over q's own columns
    again = pool.to(DEV)
    torch.ops.cdb.qk_norm_rope_append(view, None, again, *args[1:])
    torch.ops.cdb.qk_norm_rope_append(view, view, dev_pool, *args[1:])
    assert torch.equal(again, dev_pool)
    assert torch.equal(view[live][:, : heads * d], q_out[live][:, : heads * d])
    assert torch.equal(view.cpu()[pad], qkv[pad][:, : all_heads * d])
    assert torch.equal(view.cpu()[:, heads * d :], qkv[:, heads * d : all_heads * d])


def test_zero_and_large_rows():
    d, heads = 64, 2
    qkv = torch.zeros(3, 4 * d + 2 * d, dtype=torch.bfloat16)[:, : 4 * d].contiguous()
    qkv[1] = 1e15
    qkv[2, ::2] = 1e-20
    one = torch.ones(d, dtype=torch.bfloat16)
    i32 = dict(dtype=torch.int32, device=DEV)
    pool = torch.zeros(1, 2, 32, 1, d, dtype=torch.bfloat16, device=DEV)
    out = torch.empty(3, heads * d, dtype=torch.bfloat16, device=DEV)
    table = torch.tensor([[1, 0]], **i32)
    torch.ops.cdb.qk_norm_rope_append(qkv.to(DEV), out, pool, 0, table, torch.zeros(3, **i32), torch.tensor([0, 15, 16], **i32), one.to(DEV), one.to(DEV),
                                      None, None, 0, heads, 1e-5)
    q, k, _, size, at = ref.norm_append(qkv, table.cpu(), [0] * 3, [0, 15, 16], one, one, None, None, 0, heads, 1, 1e-5)
    _near(out.cpu().view(3, heads, d), q, size[:, :heads])
    _near(pool.cpu()[0, 0, at], k, size[:, heads:])


@pytest.mark.parametrize("what", ["slot", "position", "block", "angles"])
def test_indexes_out_of_range(what):
    d, n = 64, 3
    i32 = dict(dtype=torch.int32, device=DEV)
    slot, pos = torch.tensor([0, 1, 0], **i32), torch.tensor([3, 4, 20], **i32)
    table = torch.tensor([[2, 0, 3], [1, 3, 3]], **i32)
    positions = 64
    if what == "slot":
        slot[1] = 2
    elif what == "position":
        pos[1] = 48
    elif what == "block":
        table[1, 0] = 4
    else:
        positions, pos[1] = 21, 21
    cos, sin = (t.to(DEV) for t in _tables(2, d, positions))
    pool = torch.full((1, 2, 4 * BS + 3, 1, d), 5.0, dtype=torch.bfloat16, device=DEV)
    out = torch.full((n, d), 5.0, dtype=torch.bfloat16, device=DEV)
    qkv = torch.randn(n, 3 * d, device=DEV).bfloat16()
    w = torch.ones(d, dtype=torch.bfloat16, device=DEV)
    status = torch.ops.cdb._status_word(qkv)
    torch.ops.cdb.qk_norm_rope_append(qkv, out, pool, 0, table, slot, pos, w, w, cos, sin, 2, 1, 1e-6)
    torch.cuda.synchronize()
    assert ops.status_code() == 6
    status.zero_()
    assert (out[1] == 5).all() and (out[0] != 5).any() and (out[2] != 5).any()
    written = (pool[0, 0] != 5).flatten(1).any(1).nonzero()[:, 0].tolist()
    assert written == sorted([2 * BS + 3, 0 * BS + 4])


def test_no_rows():
    d = 64
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=DEV)  # noqa: E731
    i32 = dict(dtype=torch.int32, device=DEV)
    torch.ops.cdb.qk_norm_rope_append(z(0, 3 * d), z(0, d), z(1, 2, 16, 1, d), 0, torch.zeros(1, 1, **i32), torch.zeros(0, **i32), torch.zeros(0, **i32), z(d), z(d),
                                      None, None, 0, 1, 1e-6)
    assert ops.status_code() == 0


def test_a_cache_past_32_bits():
    """Rows whose offset passes 2^32 bytes and 2^31 elements, in the last layer of a large pool."""

    d, kv, heads = 128, 16, 16
    blocks = 2**31 // (2 * BS * kv * d) // 3 + 11
    pool = torch.empty(4, 2, blocks * BS, kv, d, dtype=torch.bfloat16, device=DEV)
    assert pool.numel() > 2**31
    g = torch.Generator().manual_seed(3)
    i32 = dict(dtype=torch.int32, device=DEV)
    table = torch.tensor([[blocks - 1, 0]], dtype=torch.int32)
    qkv = torch.randn(2, 3 * heads * d, generator=g).bfloat16()
    w = torch.ones(d, dtype=torch.bfloat16)
    torch.ops.cdb.qk_norm_rope_append(qkv.to(DEV), None, pool, 3, table.to(DEV), torch.zeros(2, **i32), torch.tensor([15, 16], **i32), w.to(DEV), w.to(DEV), None, None,
                                      0, heads, 1e-6)
    _, k, v, size, at = ref.norm_append(qkv, table, [0, 0], [15, 16], w, w, None, None, 0, heads, kv, 1e-6)
    _near(pool[3, 0, at].cpu(), k, size[:, heads:])
    assert torch.equal(pool[3, 1, at].cpu().double(), v)
