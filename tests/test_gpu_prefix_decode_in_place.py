"""Prefix decode attention over q's own columns, beside other columns of one buffer: the bits of a call with rows apart."""

from __future__ import annotations

import pytest
import torch

import continuous_depth_batching_b200.ops as ops
from continuous_depth_batching_b200 import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32 = dict(dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("heads,kv,d", [(4, 4, 128), (32, 8, 64), (6, 1, 96), (24, 2, 64)])
@pytest.mark.parametrize("sizes,prefix,extra", [([1], 0, 40), ([3, 40], 700, 60), ([150], 3000, 20), ([2, 1], 64, 9000)])
@pytest.mark.parametrize("sms", [None, 2, 11])
def test_in_place(heads, kv, d, sizes, prefix, extra, sms):
    """``sms``: how many the C entry point is told to use, so that small cases share too; None: the operator."""

    g = torch.Generator().manual_seed(sum(sizes) + heads)
    n, cols = sum(sizes), heads * d
    of = [i for i, s in enumerate(sizes) for _ in range(s)]
    pos = [prefix + int(x) for x in torch.randint(0, extra, (n,), generator=g)]
    shared, width = prefix // 16, (prefix + extra) // 16 + 1
    blocks = len(sizes) * shared + n * (width - shared)
    table = torch.empty(n, width, dtype=torch.int32)
    for i in range(n):
        table[i, :shared] = torch.arange(of[i] * shared, (of[i] + 1) * shared)
        table[i, shared:] = len(sizes) * shared + torch.arange(i * (width - shared), (i + 1) * (width - shared))
    pool = torch.randn(1, 2, blocks * 16, kv, d, generator=g).bfloat16().to(DEV)
    q = torch.randn(n, cols + 2 * kv * d, generator=g).bfloat16()
    table, slot, at = table.to(DEV), torch.arange(n, **I32), torch.tensor(pos, **I32)
    start, lens = torch.tensor([0, *sizes]).cumsum(0).int().to(DEV), torch.full((len(sizes),), prefix, **I32)

    def call(q, out):
        if sms is None:
            torch.ops.cdb.prefix_decode_attention(q, out, pool, 0, table, slot, at, start, lens, heads, d**-0.5)
            return
        floats = _lib.load().cdb_prefix_decode_workspace_floats(n, len(sizes), heads, kv, d, sms)
        ws = torch.empty(floats, device=DEV)
        _lib.call("cdb_prefix_decode_attention", _lib.ptr(q), q.stride(0), _lib.ptr(out), out.stride(0), _lib.ptr(pool), 1, pool.shape[2], 0, _lib.ptr(table),
                  table.stride(0), n, width, _lib.ptr(slot), _lib.ptr(at), n, _lib.ptr(start), _lib.ptr(lens), len(sizes), heads, kv, d, d**-0.5, sms, _lib.ptr(ws),
                  floats, _lib.ptr(torch.ops.cdb._status_word(q)), torch.cuda.current_stream().cuda_stream)

    apart = torch.empty(n, cols, dtype=torch.bfloat16, device=DEV)
    call(q.to(DEV), apart)
    over = q.to(DEV)
    call(over, over)
    beside = torch.cat((q.to(DEV)[:, :cols], torch.zeros(n, cols, dtype=torch.bfloat16, device=DEV)), 1)
    call(beside[:, :cols], beside[:, cols:])
    assert torch.equal(over[:, :cols], apart) and torch.equal(over[:, cols:].cpu(), q[:, cols:])
    assert torch.equal(beside[:, cols:], apart) and torch.equal(beside[:, :cols].cpu(), q[:, :cols])
    assert not apart.isnan().any() and ops.status_code() == 0
