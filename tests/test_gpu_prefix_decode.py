"""Decode attention whose groups share their prompts' blocks, against every row by itself in 64 bits.

Tolerance, with size = sum p |v| / sum p: the output's rounding, 2^-8 of the value; the weights' rounding to bf16 before
their product with V, at most 2^-8 of each, over the sum of the rounded weights, off by as much: 2^-8 (size + |o|) (over
the sum of those before, 2^-8 size); the fp32 logits (D <= 128 products whose sizes add up to some 10 here, 2^-24 each): 2^-12 size.
"""

from __future__ import annotations

import pytest
import torch

import continuous_depth_batching_b200.ops as ops
import continue_reference as ref
from continuous_depth_batching_b200 import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"
BS = 16
I32 = dict(dtype=torch.int32, device=DEV)
# How many SMs the C entry point is told to use; None: the operator, which names the device's. Sharing pays sooner
# on few, and a CTA then takes several units, so small cases go every way: shared, each row alone, both at once.
SMS = [None, 2, 3, 11]


class Case:
    """Groups of ``(rows, prefix tokens shared in the tables)``, rows' own tokens ``extra`` behind it; the cache holds NaN
    wherever no row may look."""

    def __init__(self, groups, extra, heads, kv, d, seed=0, layers=1, layer=0, spare=2):
        g = torch.Generator().manual_seed(seed)
        n = sum(r for r, _ in groups)
        self.heads, self.kv, self.d, self.layer, self.n = heads, kv, d, layer, n
        of = [i for i, (r, _) in enumerate(groups) for _ in range(r)]
        self.prefix = [p for _, p in groups]
        self.lens = [groups[of[i]][1] + extra[i] for i in range(n)]
        shared = [p // BS for _, p in groups]
        width = max((l + BS - 1) // BS for l in self.lens) + 2
        need = sum(shared) + sum((self.lens[i] + BS - 1) // BS - shared[of[i]] for i in range(n))
        self.blocks = need + spare
        ids = torch.randperm(self.blocks, generator=g).int().tolist()
        take = iter(ids)
        common = [[next(take) for _ in range(k)] for k in shared]
        self.slot = torch.randperm(n + 2, generator=g)[:n].tolist()
        table = torch.full((n + 2, width + 3), -7, dtype=torch.int32)
        self.pool = torch.full((layers, 2, self.blocks * BS + 5, kv, d), float("nan"), dtype=torch.bfloat16)
        for i in range(n):
            row = common[of[i]][:]
            while len(row) * BS < self.lens[i]:
                row.append(next(take))
            table[self.slot[i], : len(row)] = torch.tensor(row, dtype=torch.int32)
            at = torch.arange(self.lens[i])
            rows = table[self.slot[i]].long()[at // BS] * BS + at % BS
            fresh = rows[self.pool[layer, 0, rows, 0, 0].isnan()]
            self.pool[layer, :, fresh] = torch.randn(2, fresh.numel(), kv, d, generator=g).bfloat16()
        self.table = table
        self.q = torch.randn(n, heads * d, generator=g).bfloat16()
        self.start = [0]
        for r, _ in groups:
            self.start.append(self.start[-1] + r)
        self.pos = [l - 1 for l in self.lens]
        self.scale = d**-0.5

    def run(self, start=None, prefix=None, sms=None):
        start, prefix = self.start if start is None else start, self.prefix if prefix is None else prefix
        wide = torch.full((self.n, self.heads * self.d + 8), 3.0, dtype=torch.bfloat16, device=DEV)
        qw = torch.zeros(self.n, self.heads * self.d + 16, dtype=torch.bfloat16, device=DEV)
        qw[:, : self.heads * self.d] = self.q.to(DEV)
        self.dev = dict(pool=self.pool.to(DEV), table=self.table.to(DEV)[:, : self.table.shape[1] - 3])
        q, out = qw[:, : self.heads * self.d], wide[:, : self.heads * self.d]
        slot, pos = torch.tensor(self.slot, **I32), torch.tensor(self.pos, **I32)
        start, prefix = torch.tensor(start, **I32), torch.tensor(prefix, **I32)
        pool, table = self.dev["pool"], self.dev["table"]
        if sms is None:
            torch.ops.cdb.prefix_decode_attention(q, out, pool, self.layer, table, slot, pos, start, prefix, self.heads, self.scale)
        else:
            n, groups = self.n, prefix.numel()
            floats = _lib.load().cdb_prefix_decode_workspace_floats(n, groups, self.heads, self.kv, self.d, sms)
            ws = torch.full((floats + 64,), float("nan"), device=DEV)  # in any state; nothing behind it is written
            _lib.call("cdb_prefix_decode_attention", *map(_lib.ptr, (q,)), q.stride(0), _lib.ptr(out), out.stride(0), _lib.ptr(pool), pool.shape[0], pool.shape[2],
                      self.layer, _lib.ptr(table), table.stride(0), table.shape[0], table.shape[1], _lib.ptr(slot), _lib.ptr(pos), n, _lib.ptr(start),
                      _lib.ptr(prefix), groups, self.heads, self.kv, self.d, self.scale, sms, _lib.ptr(ws), floats,
                      _lib.ptr(torch.ops.cdb._status_word(q)), torch.cuda.current_stream().cuda_stream)
            assert ws[floats:].isnan().all()
        torch.cuda.synchronize()
        assert (wide[:, self.heads * self.d :] == 3).all()
        return wide[:, : self.heads * self.d].cpu()

    def check_all(self, rows=None, **how):
        for sms in SMS:
            self.check(self.run(sms=sms, **how), rows)

    def check(self, out, rows=None):
        for i in range(self.n) if rows is None else rows:
            if self.pos[i] < 0:
                assert (out[i] == 3).all()
                continue
            want, size = ref.attend(self.q[i].view(self.heads, self.d), self.pool[self.layer], self.table[self.slot[i]], self.pos[i], self.scale, self.blocks)
            tol = 2.0**-8 * want.abs() + 2.0**-8 * (size + want.abs()) + 2.0**-12 * size
            off = (out[i].double().view(self.heads, self.d) - want).abs()
            assert (off <= tol).all(), (i, float((off / tol).max()))


LAYOUTS = [(1, 1, 64), (16, 16, 128), (32, 8, 128), (8, 1, 64), (16, 1, 128), (12, 12, 64), (6, 2, 96), (55, 55, 96), (24, 2, 96), (33, 3, 128)]


@pytest.mark.parametrize("heads,kv,d", LAYOUTS)
@pytest.mark.parametrize("groups", [[(1, 0)], [(1, 5)], [(3, 16)], [(1, 100)], [(5, 47), (1, 64), (2, 0)], [(9, 130), (3, 700)], [(2, 1024)], [(70, 333)]])
def test_head_layouts_and_groups(heads, kv, d, groups):
    g = torch.Generator().manual_seed(len(groups) + heads)
    n = sum(r for r, _ in groups)
    extra = [1 + int(x) for x in torch.randint(0, 60, (n,), generator=g)]
    c = Case(groups, extra, heads, kv, d, seed=heads + n)
    c.check_all()
    assert ops.status_code() == 0


@pytest.mark.parametrize("heads,kv,d", [(16, 16, 128), (32, 8, 128), (4, 2, 96)])
@pytest.mark.parametrize("prefix", [1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 500, 1000, 4001])
@pytest.mark.parametrize("rows", [2, 33])
def test_prefix_lengths(heads, kv, d, prefix, rows):
    extra = [1 + (i * 7) % 40 for i in range(rows)]
    c = Case([(rows, prefix)], extra, heads, kv, d, seed=prefix)
    c.check_all()
    assert ops.status_code() == 0


@pytest.mark.parametrize("rows", [1, 2, 127, 128, 129, 256, 300])
def test_rows_around_a_tile(rows):
    c = Case([(rows, 200)], [1 + i % 30 for i in range(rows)], 2, 2, 64, seed=rows)
    c.check_all()
    c = Case([(rows, 96)], [1 + i % 3 for i in range(rows)], 6, 2, 64, seed=rows)
    c.check_all()
    assert ops.status_code() == 0


def test_many_groups_and_more_rows_than_threads():
    g = torch.Generator().manual_seed(9)
    groups = [(int(a), int(b)) for a, b in zip(torch.randint(1, 12, (150,), generator=g), torch.randint(0, 200, (150,), generator=g))]
    n = sum(r for r, _ in groups)
    assert n > 512
    c = Case(groups, [1 + int(x) for x in torch.randint(0, 90, (n,), generator=g)], 4, 2, 64)
    c.check_all(range(0, n, 5))
    assert ops.status_code() == 0


@pytest.mark.parametrize("own", [1, 16, 17, 3000, 20000])
def test_long_rows_of_their_own(own):
    c = Case([(3, 400), (1, 0)], [own, 5, own // 2 + 1, own], 8, 2, 128, seed=own)
    c.check_all()
    assert ops.status_code() == 0


def test_a_long_prefix():
    c = Case([(7, 40000)], [1, 2, 30, 40, 500, 3, 9], 8, 2, 128)
    c.check_all()
    assert ops.status_code() == 0


def test_groups_that_leave_rows_out_and_empty_ones():
    c = Case([(4, 160), (3, 320), (5, 80)], [3 * i + 1 for i in range(12)], 4, 4, 128)
    c.check_all()
    for start, prefix in [
        ([4, 7], [320]),  # the second group alone
        ([], []),  # every row alone
        ([0], []),
        ([0, 0, 4, 4, 7, 7, 12, 12], [50, 160, 9999, 320, 16, 80, 3]),  # empty groups between
        ([1, 3, 5, 6], [100, 0, 320]),  # parts of them
        ([0, 4, 7, 12], [-5, 0, -(2**31)]),
        ([0, 1, 1, 2], [2**31 - 1] * 3),  # more than the row: cut to what it sees
    ]:
        c.check_all(start=start, prefix=prefix)
    assert ops.status_code() == 0


def test_rows_that_see_less_than_the_prefix_and_padding_rows():
    c = Case([(6, 320), (4, 64)], [5, 9, 40, 1, 2, 3, 4, 5, 6, 7], 8, 4, 64)
    c.pos[2] = 100  # ends inside the shared blocks
    c.check_all()
    c.pos[0], c.pos[4], c.slot[0] = -1, -1, -9
    c.check_all()
    c.pos[2] = 0
    c.check_all()
    for i in range(6):
        c.pos[i] = -1
    c.check_all()
    for i in range(10):
        c.pos[i] = -1
    for sms in SMS:
        assert (c.run(sms=sms) == 3).all()
    assert ops.status_code() == 0


def test_rows_that_see_shared_blocks_only():
    """Positions that end a page, so that a row's own pages are none."""

    c = Case([(5, 256), (3, 64)], [16, 1, 32, 16, 20, 16, 16, 16], 4, 2, 128)
    for i in (0, 3):
        c.pos[i] = 255
    for i in (5, 6, 7):
        c.pos[i] = 63
    c.check_all()
    assert ops.status_code() == 0


def test_large_logits_and_a_dominant_key():
    for scale_up in (1.0, 30.0):
        c = Case([(5, 640)], [3, 30, 60, 9, 1], 4, 4, 128, seed=4)
        rows = c.table[c.slot[0]].long()
        c.pool[0, 0, rows[2] * BS + 3] *= scale_up
        own = c.table[c.slot[1]].long()[41] * BS
        c.pool[0, 0, own] *= scale_up
        for sms, i in ((sms, i) for sms in SMS for i in range(5)):
            out = c.run(sms=sms)
            want, size = ref.attend(c.q[i].view(4, 128), c.pool[0], c.table[c.slot[i]], c.pos[i], c.scale, c.blocks)
            # logits of up to 30 x 10: their fp32 sums are off by up to 128 x 2^-24 x 300 = 2^-9
            tol = 2.0**-8 * want.abs() + 2.0**-8 * (size + want.abs()) + 2.0**-8 * size
            assert ((out[i].double().view(4, 128) - want).abs() <= tol).all()


@pytest.mark.parametrize("sms", SMS)
def test_nan_and_infinity_stay_in_the_rows_that_see_them(sms):
    c = Case([(4, 128), (3, 96)], [5, 40, 3, 20, 1, 2, 3], 4, 2, 64, seed=2)
    clean = c.run(sms=sms)
    own = c.table[c.slot[1]].long()[9] * BS + 2  # position 146 of row 1
    c.pool[0, 0, own] = float("nan")
    c.pool[0, 1, c.table[c.slot[3]].long()[8] * BS] = float("inf")
    out = c.run(sms=sms)
    assert out[1].isnan().all() and (out[3] == float("inf")).all()
    keep = [0, 2, 4, 5, 6]
    assert torch.equal(out[keep], clean[keep])
    c.pool[0, 1, c.table[c.slot[4]].long()[0] * BS + 1] = float("nan")  # shared by the second group
    out = c.run(sms=sms)
    assert out[4:].isnan().all() and torch.equal(out[[0, 2]], clean[[0, 2]])
    assert ops.status_code() == 0


@pytest.mark.parametrize("sms", SMS)
@pytest.mark.parametrize("what", ["slot", "position", "own block", "own block past the cache", "shared block"])
def test_indexes_out_of_range(what, sms):
    c = Case([(3, 96), (2, 64)], [20, 3, 40, 5, 6], 4, 2, 64, seed=3)
    if what == "slot":
        c.slot[1] = 7
    elif what == "position":
        c.pos[1] = (c.table.shape[1] - 3) * BS
    elif what == "own block":
        c.table[c.slot[1], 6] = -1
    elif what == "own block past the cache":
        c.table[c.slot[1], 6] = c.blocks
    else:
        for i in range(3):
            c.table[c.slot[i], 2] = 2**31 - 1
    out = c.run(sms=sms)
    assert ops.status_code() == 6
    torch.ops.cdb._status_word(c.dev["pool"]).zero_()
    if what in ("slot", "position"):
        assert (out[1] == 3).all()
        c.check(out, [0, 2, 3, 4])
    else:
        c.check(out)  # without the keys of such blocks


@pytest.mark.parametrize("sms", SMS)
@pytest.mark.parametrize("start", [[0, 3, 2], [-1, 3, 5], [0, 3, 6], [4, 3, 5], [0, 2**31 - 1, 5]])
def test_group_bounds_out_of_range(start, sms):
    c = Case([(3, 96), (2, 64)], [20, 3, 40, 5, 6], 4, 2, 64, seed=3)
    out = c.run(start=start, sms=sms)
    assert ops.status_code() == 6
    torch.ops.cdb._status_word(c.dev["pool"]).zero_()
    c.check(out)


def test_no_rows_and_layers():
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=DEV)  # noqa: E731
    torch.ops.cdb.prefix_decode_attention(z(0, 64), z(0, 64), z(1, 2, 16, 1, 64), 0, torch.zeros(1, 1, **I32), torch.zeros(0, **I32), torch.zeros(0, **I32),
                                          torch.zeros(2, **I32), torch.zeros(1, **I32), 1, 0.125)
    c = Case([(3, 100)], [5, 6, 70], 4, 2, 96, layers=3, layer=2)
    c.check_all()
    assert ops.status_code() == 0


def test_the_same_bits_again():
    c = Case([(40, 3000), (9, 100)], [1 + (i * 37) % 300 for i in range(49)], 16, 4, 128)
    for sms in SMS:
        first = c.run(sms=sms)
        c.check(first, range(0, 49, 5))
        for _ in range(3):
            assert torch.equal(c.run(sms=sms), first)


def test_more_rows_than_the_plan_keeps():
    """More rows, and groups, than the plan's threads and shared memory hold."""

    n = 2300
    c = Case([(2, 48)] * 1100 + [(100, 600)], [1 + i % 20 for i in range(n)], 2, 1, 64, seed=8)
    assert c.n == n and len(c.prefix) == 1101
    c.check_all(list(range(0, 2200, 97)) + list(range(2200, n, 9)))
    assert ops.status_code() == 0


def test_a_cache_past_32_bits():
    kv, d, heads = 16, 128, 16
    blocks = 2**31 // (2 * BS * kv * d) // 3 + 60
    pool = torch.empty(4, 2, blocks * BS, kv, d, dtype=torch.bfloat16, device=DEV)
    assert pool.numel() > 2**31
    g = torch.Generator().manual_seed(1)
    n, prefix = 5, 400
    small = Case([(n, prefix)], [3, 30, 1, 16, 50], heads, kv, d)
    shift = blocks - small.blocks
    pool[3, :, shift * BS :] = small.pool[0, :, : small.blocks * BS].to(DEV)
    table = torch.where(small.table >= 0, small.table + shift, small.table)
    out = torch.empty(n, heads * d, dtype=torch.bfloat16, device=DEV)
    del g
    torch.ops.cdb.prefix_decode_attention(small.q.to(DEV), out, pool, 3, table.to(DEV), torch.tensor(small.slot, **I32), torch.tensor(small.pos, **I32),
                                          torch.tensor([0, n], **I32), torch.tensor([prefix], **I32), heads, small.scale)
    torch.cuda.synchronize()
    assert ops.status_code() == 0
    small.check(out.cpu())


def test_two_graphs_at_once_and_other_streams():
    """Graphs captured from one stream and replayed beside each other and beside eager calls."""

    cases = [Case([(20, 900)], [1 + i for i in range(20)], 16, 16, 128, seed=1), Case([(3, 5000), (4, 64)], [400, 5, 6, 7, 8, 9, 100], 32, 8, 128, seed=2)]
    want = [c.run() for c in cases]
    args, outs = [], []
    for c in cases:
        out = torch.zeros(c.n, c.heads * c.d, dtype=torch.bfloat16, device=DEV)
        outs.append(out)
        args.append((c.q.to(DEV), out, c.dev["pool"], 0, c.dev["table"], torch.tensor(c.slot, **I32), torch.tensor(c.pos, **I32), torch.tensor(c.start, **I32),
                     torch.tensor(c.prefix, **I32), c.heads, c.scale))
    torch.cuda.synchronize()
    graphs = []
    for a in args:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            torch.ops.cdb.prefix_decode_attention(*a)
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(6):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for out, w in zip(outs, want):
            assert torch.equal(out.cpu(), w)
        for a, s in zip(args, streams):  # eager calls of both on two streams
            a[1].zero_()
        torch.cuda.synchronize()
        for a, s in zip(args, streams):
            with torch.cuda.stream(s):
                torch.ops.cdb.prefix_decode_attention(*a)
        torch.cuda.synchronize()
        for out, w in zip(outs, want):
            assert torch.equal(out.cpu(), w)
    assert ops.status_code() == 0
