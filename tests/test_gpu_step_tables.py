"""cdb_step_tables against a plain sequential statement of it, and with the device allocator's own entry
points. Integers: everything has to be equal."""

from __future__ import annotations

import random

import pytest
import torch

import continuous_depth_batching_b200.ops  # noqa: F401  (registers torch.ops.cdb.*)
from continuous_depth_batching_b200 import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"
BS, TILE = 16, 64


def reference(slots, seq_len, new_len, row_len, table, ring, state, cap, tile_cap):
    head, avail, nb, peak = state
    table, row_len = [list(r) for r in table], list(row_len)
    granted, cu_q, cu_k, items, tiles = [], [0], [0], [], []
    for s, n in zip(slots, new_len):
        need = max(0, -(-(seq_len[s] + n) // BS) - row_len[s])
        ok = need <= avail and -(-(seq_len[s] + n) // BS) <= len(table[s])
        granted.append(int(ok))
        if not ok:
            cu_q.append(cu_q[-1])
            cu_k.append(cu_k[-1])
            continue
        for i in range(need):
            table[s][row_len[s] + i] = ring[(head + i) % nb]
        head, avail, row_len[s] = (head + need) % nb, avail - need, row_len[s] + need
        for i in range(0, n, TILE):
            tiles.append([cu_q[-1] + i, min(TILE, n - i), s, seq_len[s] + i])
        for p in range(seq_len[s], seq_len[s] + n):
            items.append((s, p, table[s][p // BS] * BS + p % BS))
        cu_q.append(cu_q[-1] + n)
        cu_k.append(cu_k[-1] + seq_len[s] + n)
    items += [(-1, -1, -1)] * (cap - len(items))
    tiles += [[0, 0, 0, 0]] * (tile_cap - len(tiles))
    return dict(table=table, row_len=row_len, state=[head, avail, nb, max(peak, nb - avail)], granted=granted, cu_q=cu_q,
                cu_k=cu_k, slot=[i[0] for i in items], pos=[i[1] for i in items], map=[i[2] for i in items], tiles=tiles)


def _case(seed, requests, max_ctx, max_new, spare, width_short=False, hold_more=False):
    rng = random.Random(seed)
    rows = requests + 5
    slots = rng.sample(range(rows), requests)
    seq_len = [rng.choice([0, 1, 15, 16, 17, rng.randint(0, max_ctx)]) for _ in range(rows)]
    new_len = [rng.choice([0, 1, 1, max_new, rng.randint(0, max_new)]) for _ in range(requests)]
    row_len = [-(-n // BS) + (rng.randint(0, 3) if hold_more else 0) for n in seq_len]
    width = max([row_len[s] for s in range(rows)] + [-(-(seq_len[s] + n) // BS) for s, n in zip(slots, new_len)])
    width -= 2 if width_short and width - 2 >= max(row_len) else 0
    need = sum(max(0, -(-(seq_len[s] + n) // BS) - row_len[s]) for s, n in zip(slots, new_len))
    free = max(0, need + spare)
    nb = sum(row_len) + free
    ids = list(range(nb))
    rng.shuffle(ids)
    table = [[-1] * width for _ in range(rows)]
    at = 0
    for s in range(rows):
        for i in range(row_len[s]):
            table[s][i] = ids[at]
            at += 1
    head = rng.randrange(max(1, nb))
    ring = [-1] * nb
    for i, b in enumerate(ids[at:]):
        ring[(head + i) % nb] = b
    return slots, seq_len, new_len, row_len, table, ring, [head, free, nb, nb - free]


def _run(slots, seq_len, new_len, row_len, table, ring, state, cap, tile_cap, in_place):
    t = lambda v, d=torch.int32: torch.tensor(v, dtype=d, device=DEV)  # noqa: E731
    n = len(slots)
    d_table, d_row, d_state = t(table).view(len(table), -1), t(row_len), t(state)
    o_row, o_state = (d_row, d_state) if in_place else (d_row.clone(), torch.zeros_like(d_state))
    granted, cu_q, cu_k = (torch.full((k,), -7, dtype=torch.int32, device=DEV) for k in (n, n + 1, n + 1))
    slot, pos = (torch.full((cap,), -7, dtype=torch.int32, device=DEV) for _ in range(2))
    rows = torch.full((cap,), -7, dtype=torch.int64, device=DEV)
    tiles = torch.full((tile_cap, 4), -7, dtype=torch.int32, device=DEV) if tile_cap is not None else None
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    p = _lib.ptr
    ins = [t(slots), t(seq_len), t(new_len), t(ring)]
    _lib.call("cdb_step_tables", p(ins[0]), p(ins[1]), p(ins[2]), p(d_row), n, p(d_table), d_table.stride(0),
              len(table), d_table.shape[1], p(ins[3]), len(ring), p(d_state), p(o_row), p(o_state), p(granted), p(cu_q),
              p(cu_k), p(slot), p(pos), p(rows), cap, p(tiles), tile_cap or 0, p(status),
              torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    got = dict(table=d_table.tolist(), row_len=o_row.tolist(), state=o_state.tolist(), granted=granted.tolist(),
               cu_q=cu_q.tolist(), cu_k=cu_k.tolist(), slot=slot.tolist(), pos=pos.tolist(), map=rows.tolist())
    if tiles is not None:
        got["tiles"] = tiles.tolist()
    return got, int(status.item())


@pytest.mark.parametrize("requests,max_ctx,max_new,spare,short,more", [
    (1, 100, 1, 0, False, False), (1, 0, 5000, 3, False, False), (256, 2000, 1, 0, False, False),
    (64, 1000, 500, 10, False, False), (33, 200, 700, -30, False, False), (40, 300, 90, -1000, False, False),
    (700, 60, 20, 5, False, True), (1500, 90, 9, 0, False, False), (30, 400, 200, 7, True, False),
    (4000, 40, 3, -200, False, False),
])
@pytest.mark.parametrize("in_place", [False, True])
def test_matches_sequential_statement(requests, max_ctx, max_new, spare, short, more, in_place):
    c = _case(requests + max_new, requests, max_ctx, max_new, spare, short, more)
    cap, tile_cap = sum(c[2]) + 37, sum(-(-n // TILE) for n in c[2]) + 5
    want = reference(*c, cap, tile_cap)
    got, status = _run(*c, cap, tile_cap, in_place)
    assert status == 0
    for k, v in want.items():
        assert got[k] == v, k


def test_no_requests_and_no_tokens():
    c = _case(3, 4, 50, 5, 2)
    got, status = _run([], c[1], [], *c[3:], 7, 2, False)
    assert status == 0 and got["cu_q"] == [0] and got["slot"] == [-1] * 7 and got["tiles"] == [[0] * 4] * 2
    assert got["table"] == c[4] and got["state"] == c[6] and got["row_len"] == c[3]
    got, status = _run(c[0], c[1], [0] * 4, *c[3:], 0, None, False)
    assert status == 0 and got["cu_q"] == [0] * 5 and got["granted"] == [1] * 4 and got["table"] == c[4]


def test_capacities_and_bad_requests_are_reported():
    c = list(_case(5, 6, 80, 40, 4))
    c[2] = [40, 3, 0, 17, 40, 1]
    total = sum(c[2])
    want = reference(*_grown(c), total, 20)
    got, status = _run(*_grown(c), total - 5, 20, False)  # five tokens too few
    assert status == 6
    assert got["map"] == want["map"][: total - 5] and got["table"] == want["table"]
    got, status = _run(*_grown(c), total, 1, False)
    assert status == 6 and got["tiles"] == [[0] * 4] and got["map"] == want["map"]
    bad = _grown(c)
    bad[0] = [len(c[1]) + 3] + bad[0][1:]  # no such slot
    bad[2] = bad[2][:3] + [-2] + bad[2][4:]  # a negative length
    got, status = _run(*bad, total, 20, False)
    assert status == 6 and got["granted"][0] == 0 and got["granted"][3] == 0
    keep = [1, 2, 4, 5]
    want = reference([bad[0][j] for j in keep], bad[1], [bad[2][j] for j in keep], *bad[3:], total, 20)
    assert got["table"] == want["table"] and got["map"] == want["map"] and got["state"] == want["state"]


def _grown(c):
    """The case with enough spare blocks and columns for any new lengths."""

    slots, seq_len, new_len, row_len, table, ring, state = c
    used = sum(row_len)
    free = list(range(used, used + 60))
    ids = iter(range(used))
    table = [[next(ids) if i < n else -1 for i in range(40)] for n in row_len]
    return [list(slots), seq_len, list(new_len), row_len, table, free + [-1] * used, [0, 60, used + 60, used]]


def test_blocks_taken_here_are_freed_by_the_allocator():
    """The ring, state and row lengths are those of cdb_block_alloc / cdb_block_free."""

    nb, rows, width = 50, 4, 12
    i32 = dict(dtype=torch.int32, device=DEV)
    ring, state, row_len = torch.empty(nb, **i32), torch.empty(4, **i32), torch.empty(rows, **i32)
    table = torch.full((rows, width), -1, **i32)
    sp = torch.cuda.current_stream().cuda_stream
    p = _lib.ptr
    _lib.call("cdb_block_pool_init", p(ring), p(state), p(row_len), rows, nb, sp)
    slots, seq_len = torch.tensor([2, 0], **i32), torch.zeros(rows, **i32)
    new = torch.tensor([100, 33], **i32)
    out = [torch.empty(k, **i32) for k in (2, 3, 3, 133, 133)]
    rows64, tiles = torch.empty(133, dtype=torch.int64, device=DEV), torch.empty(4, 4, **i32)
    torch.ops.cdb.step_tables(slots, seq_len, new, row_len, table, ring, state, row_len, state, *out, rows64, tiles)
    assert row_len.tolist() == [3, 0, 7, 0] and state.tolist() == [10, 40, 50, 10]
    assert table[2, :7].tolist() == list(range(7)) and table[0, :3].tolist() == [7, 8, 9]
    _lib.call("cdb_block_free", p(ring), p(state), p(row_len), p(table), width, p(slots), 1, sp)
    assert state.tolist() == [10, 47, 50, 10] and row_len.tolist() == [3, 0, 0, 0]
    seq_len.copy_(torch.tensor([33, 0, 0, 0], **i32))
    one = [torch.empty(k, **i32) for k in (1, 2, 2, 1, 1)]
    torch.ops.cdb.step_tables(slots[1:], seq_len, torch.ones(1, **i32), row_len, table, ring, state, row_len, state, *one,
                              rows64[:1], None)
    assert rows64[0].item() == 9 * BS + 1 and state.tolist() == [10, 47, 50, 10]
