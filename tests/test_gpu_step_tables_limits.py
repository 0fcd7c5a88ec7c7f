"""cdb_step_tables where its sums and positions pass 32 bits: what fits is written, the rest is reported."""

from __future__ import annotations

import pytest
import torch

from continuous_depth_batching_b200 import _lib

pytestmark = pytest.mark.gpu
I32 = dict(dtype=torch.int32, device="cuda")
MOST = 2**31 - 1


def _call(slots, seq_len, new_len, row_len, table, cap, tile_cap):
    n, p = slots.numel(), _lib.ptr
    ring, state = torch.arange(4, **I32), torch.tensor([0, 4, 4, 0], **I32)
    got = dict(row_len=row_len.clone(), state=torch.empty(4, **I32), granted=torch.empty(n, **I32),
               cu_q=torch.empty(n + 1, **I32), cu_k=torch.empty(n + 1, **I32), slot=torch.empty(cap, **I32),
               pos=torch.empty(cap, **I32), map=torch.empty(cap, dtype=torch.int64, device="cuda"))
    tiles = torch.full((tile_cap, 4), -7, **I32)
    status = torch.zeros(1, **I32)
    _lib.call("cdb_step_tables", p(slots), p(seq_len), p(new_len), p(row_len), n, p(table), table.stride(0),
              table.shape[0], table.shape[1], p(ring), 4, p(state), *map(p, list(got.values())), cap, p(tiles), tile_cap,
              p(status), torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    return {k: v.cpu() for k, v in got.items()}, tiles.cpu(), int(status.item())


@pytest.mark.parametrize("cap", [1000, 5000])  # one CTA, and a cluster of them
def test_more_tokens_than_32_bits_count(cap):
    """8192 requests, most of 2^19 tokens each: the sums wrap at the 4100th."""

    n, width = 8192, 1 << 15
    slots = torch.randperm(n, generator=torch.Generator().manual_seed(1)).int()
    new = torch.full((n,), 1 << 19, dtype=torch.int32)
    new[:4] = torch.tensor([100, 0, 700, 77])
    table = (torch.arange(n, **I32)[:, None] * 31 + torch.arange(width, **I32)) % 1000003
    held = torch.full((n,), width, **I32)
    got, tiles, status = _call(slots.cuda(), torch.zeros(n, **I32), new.cuda(), held, table, cap, 10)
    assert status == 6 and (tiles == 0).all()
    assert (got["granted"] == 1).all() and (got["row_len"] == width).all() and got["state"].tolist() == [0, 4, 4, 0]
    sums = torch.cat((torch.zeros(1, dtype=torch.int64), new.long().cumsum(0))).clamp(max=MOST)
    assert torch.equal(got["cu_q"].long(), sums) and torch.equal(got["cu_k"].long(), sums)
    first = torch.searchsorted(sums, torch.arange(cap), right=True) - 1
    slot, pos = slots[first].long(), torch.arange(cap) - sums[first]
    assert torch.equal(got["slot"].long(), slot) and torch.equal(got["pos"].long(), pos)
    assert torch.equal(got["map"], (slot * 31 + pos // 16) % 1000003 * 16 + pos % 16)


def test_positions_past_32_bits_are_refused():
    """A row of 2^27 and some blocks whose next tokens would lie behind position 2^31 - 1."""

    width = (1 << 27) + 8
    table = torch.zeros(2, width, **I32)
    table[1, 0] = 9
    got, tiles, status = _call(torch.tensor([0, 1], **I32), torch.tensor([MOST - 9, 3], **I32), torch.tensor([20, 2], **I32),
                               torch.tensor([width, 1], **I32), table, 30, 3)
    assert status == 6 and got["granted"].tolist() == [0, 1]
    assert got["cu_q"].tolist() == [0, 0, 2] and got["cu_k"].tolist() == [0, 0, 5]
    assert got["pos"].tolist() == [3, 4] + [-1] * 28 and got["map"].tolist() == [147, 148] + [-1] * 28
    assert tiles.tolist() == [[0, 2, 1, 3], [0] * 4, [0] * 4]
