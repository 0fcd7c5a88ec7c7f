"""Prefill attention over the 8-bit cache: blocks that all differ in scale, long lists, calls without rows.
Tolerance as in test_gpu_kv8: 2^-8 |o| + 2^-10 sum p |v| / sum p."""

from __future__ import annotations

import pytest
import torch

import continuous_depth_batching_b200.ops as ops
import kv8_reference as ref
from continuous_depth_batching_b200 import _lib
from continuous_depth_batching_b200.runner import OuroRunner

pytestmark = pytest.mark.gpu
DEV = "cuda"
BS = 16


def _cache(pages, kv_heads, d, seed):
    """``pages``: blocks of each slot."""

    g = torch.Generator().manual_seed(seed)
    blocks = sum(pages)
    codes = (torch.randn(1, 2, blocks, kv_heads, BS, d, generator=g) * 90).clamp(-448, 448).to(torch.float8_e4m3fn)
    scales = torch.exp2(torch.randint(-10, -4, (1, 2, blocks, kv_heads), generator=g).float())
    table = torch.full((len(pages), max(pages)), -1, dtype=torch.int32)
    ids = torch.randperm(blocks, generator=g).int()
    for i, n in enumerate(pages):
        table[i, :n], ids = ids[:n], ids[n:]
    return codes, scales, table, g


def _run(q, codes, scales, table, tiles, heads, rows=None):
    d = codes.shape[-1]
    out = torch.full((q.shape[0] if rows is None else rows, heads * d), 7.0, dtype=torch.bfloat16, device=DEV)
    torch.ops.cdb.kv8_prefill_attention(q.to(DEV), out, codes.to(DEV), scales.to(DEV), 0, table.to(DEV),
                                        torch.tensor(tiles, dtype=torch.int32, device=DEV).view(-1, 4), heads, d**-0.5)
    return out.cpu()


def _near(got, q, codes, scales, table_row, first, heads):
    n, d = q.shape[0], codes.shape[-1]
    o, a = ref.attend(q.view(n, heads, d), codes[0], scales[0], table_row, first, d**-0.5)
    assert ((got.double().view(n, heads, d) - o).abs() <= 2.0**-8 * o.abs() + 2.0**-10 * a).all()


@pytest.mark.parametrize("d", [64, 96, 128])
def test_scales_of_each_block_by_themselves(d):
    """V's scales differ by up to 2^20 from block to block, so one taken for its neighbour's shows; the same bits
    from call to call."""

    codes, scales, table, g = _cache([60], 2, d, d)
    scales[0, 1] = torch.exp2(torch.randint(-20, 1, scales[0, 1].shape, generator=g).float())
    q = torch.randn(200, 2 * d, generator=g).bfloat16()
    tiles = [(i, min(64, 200 - i), 0, 700 + i) for i in range(0, 200, 64)]
    got = _run(q, codes, scales, table, tiles, 2)
    _near(got, q, codes, scales, table[0], 700, 2)
    for _ in range(20):
        assert torch.equal(_run(q, codes, scales, table, tiles, 2), got)


def test_no_rows_and_a_padded_list():
    """q and out without rows, as a step without prompts has them: unused entries are skipped, others reported."""

    codes, scales, table, _ = _cache([2], 1, 64, 1)
    none = torch.empty(0, 64, dtype=torch.bfloat16)
    assert _run(none, codes, scales, table, [(0, 0, 0, 0)] * 3, 1).shape == (0, 64)
    assert ops.status_code() == 0
    codes, scales, table = codes.to(DEV), scales.to(DEV), table.to(DEV)
    status, tile = torch.zeros(1, dtype=torch.int32, device=DEV), torch.tensor([[0, 3, 0, 0]], dtype=torch.int32, device=DEV)
    p = _lib.ptr
    _lib.call("cdb_kv8_prefill_attention", None, 64, None, 64, 0, p(codes), p(scales), 1, 0, 2, p(table), 2, 1, 2, p(tile), 1,
              1, 1, 64, 0.125, p(status), torch.cuda.current_stream().cuda_stream)
    assert int(status.item()) == 6


@pytest.mark.parametrize("order", ["requests", "framework", "shuffled"])
@pytest.mark.parametrize("d", [64, 128])
def test_a_list_of_more_tiles_than_are_searched(d, order):
    """Some 450 tiles that all hold rows: neighbours pair, whatever stands between them is taken by itself."""

    n = 150
    g = torch.Generator().manual_seed(d)
    ctx = (torch.randint(0, 6, (n,), generator=g) * torch.tensor([16, 64, 23]).repeat(n // 3)).tolist()
    new = torch.randint(129, 190, (n,), generator=g).tolist()
    codes, scales, table, g = _cache([-(-(a + b) // BS) for a, b in zip(ctx, new)], 1, d, d + 1)
    slot = [s for s in range(n) for _ in range(new[s])]
    pos = [ctx[s] + i for s in range(n) for i in range(new[s])]
    tiles = OuroRunner.prefill_tiles(slot, pos)  # longest first
    if order == "requests":
        tiles = sorted(tiles)
    elif order == "shuffled":
        tiles = [tiles[i] for i in torch.randperm(len(tiles), generator=g).tolist()]
    assert len(tiles) == 3 * n
    q = torch.randn(len(slot), d, generator=g).bfloat16()
    out = _run(q, codes, scales, table, tiles, 1)
    assert ops.status_code() == 0
    row = 0
    for s in range(n):
        _near(out[row : row + new[s]], q[row : row + new[s]], codes, scales, table[s], ctx[s], 1)
        row += new[s]
