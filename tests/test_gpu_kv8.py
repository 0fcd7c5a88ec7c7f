"""The 8-bit paged KV cache on the GPU: append, read-back and decode attention against plain 64-bit
statements (kv8_reference).

Tolerances. Codes, scales and the read-back are exact (the rotation's fp32 rounding moves a value by
2^-22 of its size, an e4m3 step is 2^-3, so a code may differ only next to a rounding border: rotated
keys may be one step off in 1 of 10^4 places). q is rounded once to bf16: 2^-8 of its value, plus the
fp32 rotation. Attention: the output is rounded to bf16 (2^-8 of it); the weights are rounded to f16
(2^-11 each, so 2^-11 of A = sum p |v| / sum p), fp32 logits and ex2 add less than that again:
2^-8 |o| + 2^-10 A.
"""

from __future__ import annotations

import pytest
import torch

import continuous_depth_batching_b200.ops as ops
import kv8_reference as ref
from continuous_depth_batching_b200 import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"
BS = 16


def _rope(mode: int, d: int, positions: int):
    inv = 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    ang = torch.arange(positions, dtype=torch.float64)[:, None] * inv
    if mode == 1:
        ang = torch.cat((ang, ang), -1)
        return ang.cos().bfloat16(), ang.sin().bfloat16()
    return ang.cos().float(), ang.sin().float()


class Cache:
    """An 8-bit cache of two layers whose blocks all hold something, and shuffled block tables."""

    def __init__(self, lens, kv_heads, d, seed=0, layers=2):
        self.gen = torch.Generator().manual_seed(seed)
        pages = [-(-n // BS) for n in lens]
        self.width = max(pages + [1]) + 1
        self.blocks = sum(pages) + 3
        ids = torch.randperm(self.blocks, generator=self.gen).int()
        self.table = torch.full((len(lens), self.width), -1, dtype=torch.int32)
        at = 0
        for i, n in enumerate(pages):
            self.table[i, :n] = ids[at : at + n]
            at += n
        shape = (layers, 2, self.blocks, kv_heads, BS, d)
        self.codes = (torch.randn(shape, generator=self.gen) * 90).clamp(-448, 448).to(torch.float8_e4m3fn)
        self.scales = torch.exp2(torch.randint(-9, -5, shape[:4], generator=self.gen).float())

    def gpu(self):
        return self.codes.to(DEV), self.scales.to(DEV), self.table.to(DEV)


def _decode(c: Cache, q, pos, heads, layer=1, slots=None):
    codes, scales, table = c.gpu()
    n = len(pos)
    d = codes.shape[-1]
    out = torch.full((n, heads * d), 7.0, dtype=torch.bfloat16, device=DEV)
    slots = list(range(n)) if slots is None else slots
    torch.ops.cdb.kv8_decode_attention(
        q.to(DEV), out, codes, scales, layer, table, torch.tensor(slots, dtype=torch.int32, device=DEV),
        torch.tensor(pos, dtype=torch.int32, device=DEV), heads, d**-0.5,
    )
    torch.cuda.synchronize()
    assert ops.status_code() == 0
    return out.cpu()


def _check_rows(out, c: Cache, q, pos, heads, layer=1, slots=None):
    d = c.codes.shape[-1]
    for i, p in enumerate(pos):
        row = out[i].double().view(heads, d)
        if p < 0:
            assert torch.equal(out[i], torch.full_like(out[i], 7.0))
            continue
        s = i if slots is None else slots[i]
        o, a = ref.attend(q[i].view(1, heads, d), c.codes[layer], c.scales[layer], c.table[s], p, d**-0.5)
        assert ((row - o[0]).abs() <= 2.0**-8 * o[0].abs() + 2.0**-10 * a[0]).all(), (i, p)


@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("kv_heads,group", [(1, 1), (5, 1), (2, 2), (3, 3), (2, 8), (1, 12), (1, 20)])
def test_decode_matches_definition(d, kv_heads, group):
    pos = [0, 1, 14, 15, 16, -1, 17, 31, 32, 100, 511, -1, 600]
    heads = kv_heads * group
    c = Cache([p + 1 for p in pos], kv_heads, d, seed=d + heads)
    q = torch.randn(len(pos), heads * d, generator=c.gen).bfloat16()
    _check_rows(_decode(c, q, pos, heads), c, q, pos, heads)


@pytest.mark.parametrize("d,kv_heads,group", [(128, 2, 4), (96, 1, 1), (64, 1, 8), (128, 1, 1)])
def test_decode_one_long_row_is_split(d, kv_heads, group):
    """One row over the whole GPU: pieces meet in the workspace, call after call."""

    pos = [20001]
    c = Cache([pos[0] + 1], kv_heads, d, seed=3, layers=1)
    for _ in range(3):
        q = torch.randn(1, kv_heads * group * d, generator=c.gen).bfloat16() * 3
        _check_rows(_decode(c, q, pos, kv_heads * group, layer=0), c, q, pos, kv_heads * group, layer=0)


def test_decode_many_rows_with_shared_slots():
    """More rows than threads plan (several rows a thread), rows sharing a slot at other positions."""

    g = torch.Generator().manual_seed(4)
    pos = torch.randint(-1, 90, (700,), generator=g).tolist()
    c = Cache([90] * 40, 1, 64, seed=5)
    slots = torch.randint(0, 40, (700,), generator=g).tolist()
    q = torch.randn(700, 64, generator=c.gen).bfloat16()
    _check_rows(_decode(c, q, pos, 1, slots=slots), c, q, pos, 1, slots=slots)


def test_decode_ignores_codes_behind_the_row():
    pos = [0, 3, 20, 47]
    c = Cache([p + 1 for p in pos], 2, 128, seed=6)
    q = torch.randn(4, 4 * 128, generator=c.gen).bfloat16()
    want = _decode(c, q, pos, 4)
    raw = c.codes.view(torch.uint8)
    for i, p in enumerate(pos):
        raw[1, :, int(c.table[i, p // BS]), :, p % BS + 1 :] = 0x7F  # NaN
    assert torch.equal(_decode(c, q, pos, 4), want)


def test_decode_scales_far_apart_and_large_logits():
    """Blocks whose scales differ by 2^60, zero blocks at the smallest scale, logits of many hundreds."""

    pos = [79, 79]
    c = Cache([80, 80], 1, 128, seed=7)
    c.scales[1, 1, c.table[0, 1].long()] = 2.0**30
    c.scales[1, 1, c.table[0, 2].long()] = 2.0**-30
    c.scales[1, 1, c.table[1].long()[:5]] = 2.0**-126
    c.codes[1, 1, c.table[1].long()[:5]] = 0
    q = torch.randn(2, 128, generator=c.gen).bfloat16() * 40
    _check_rows(_decode(c, q, pos, 1), c, q, pos, 1)


def test_decode_strided_rows():
    pos = [40, 7]
    c = Cache([41, 8], 2, 64, seed=8)
    wide = torch.randn(2, 1024, generator=c.gen).bfloat16()
    q = wide[:, 512 : 512 + 128]
    codes, scales, table = c.gpu()
    out = torch.full((2, 256), 7.0, dtype=torch.bfloat16, device=DEV)
    torch.ops.cdb.kv8_decode_attention(
        wide.to(DEV)[:, 512 : 512 + 128], out[:, 64:192], codes, scales, 1, table,
        torch.arange(2, dtype=torch.int32, device=DEV), torch.tensor(pos, dtype=torch.int32, device=DEV), 2, 0.125,
    )
    out = out.cpu()
    assert (out[:, :64] == 7).all() and (out[:, 192:] == 7).all()
    _check_rows(out[:, 64:192], c, q, pos, 2)


@pytest.mark.parametrize("d,mode,biased", [(128, 0, False), (128, 1, True), (96, 2, True), (64, 1, False), (64, 2, False), (96, 1, False)])
@pytest.mark.parametrize("rows", ["prompt", "decode", "long"])
def test_append_matches_definition(d, mode, biased, rows):
    heads, hkv = 3, 2
    spans = {  # (first position, rows) of each slot in turn
        "prompt": [(0, 40), (5, 3), (16, 16), (30, 20), (0, 1)],
        "decode": [(0, 1), (15, 1), (16, 1), (31, 1), (77, 1), (3, 1)],
        "long": [(3, 1100), (0, 33)],
    }[rows]
    c = Cache([a + n for a, n in spans], hkv, d, seed=d + mode, layers=2)
    slot = [s for s, (_, n) in enumerate(spans) for _ in range(n)]
    pos = [a + i for a, n in spans for i in range(n)]
    slot.insert(1, 0)  # a padding row
    pos.insert(1, -1)
    if rows != "decode":  # the padding row must not part a run: put it first
        slot[0], slot[1], pos[0], pos[1] = slot[1], slot[0], pos[1], pos[0]
    n = len(pos)
    qkv = torch.randn(n, (heads + 2 * hkv) * d, generator=c.gen).bfloat16()
    qkv[1::3] *= 16  # some blocks have to grow
    bias = (torch.randn(heads + hkv, d, generator=c.gen) * 0.1).bfloat16() if biased else None
    cos, sin = _rope(mode, d, max(pos) + 1) if mode else (None, None)
    codes, scales, table = c.gpu()
    on = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    qkv_g = qkv.to(DEV)
    q_out = torch.full((n, heads * d), 7.0, dtype=torch.bfloat16, device=DEV)
    torch.ops.cdb.kv8_append(
        qkv_g, q_out, codes, scales, 1, table, torch.tensor(slot, dtype=torch.int32, device=DEV),
        torch.tensor(pos, dtype=torch.int32, device=DEV), on(cos), on(sin), on(bias), mode, heads,
    )
    torch.cuda.synchronize()
    assert ops.status_code() == 0
    want_codes, want_scales = c.codes[1].double(), c.scales[1].double()
    q = ref.append(qkv, want_codes, want_scales, c.table, slot, pos, cos, sin, bias, mode, heads)
    assert torch.equal(scales[1].cpu().double(), want_scales)
    got = codes[1].cpu().double()
    if mode == 0:
        assert torch.equal(got, want_codes)
    else:
        off = got != want_codes
        assert off.double().mean() <= 1e-4
        assert ((got - want_codes).abs()[off] <= 0.13 * want_codes.abs()[off] + 2.0**-9).all()
    assert torch.equal(codes[0].cpu().view(torch.uint8), c.codes[0].view(torch.uint8))
    live = torch.tensor(pos) >= 0
    assert (q_out.cpu()[~live] == 7).all()
    gotq, wantq = q_out.cpu().double()[live], q.view(n, -1)[live]
    size = qkv.double().view(n, -1, d)[:, :heads].abs().amax(-1, keepdim=True).expand(n, heads, d).reshape(n, -1)[live] + 1
    assert ((gotq - wantq).abs() <= 2.0**-8 * wantq.abs() + 2.0**-21 * size).all()
    # in place: q's own columns
    torch.ops.cdb.kv8_append(
        qkv_g, qkv_g[:, : heads * d], codes, scales, 1, table, torch.tensor(slot, dtype=torch.int32, device=DEV),
        torch.tensor(pos, dtype=torch.int32, device=DEV), on(cos), on(sin), on(bias), mode, heads,
    )
    assert torch.equal(qkv_g[:, : heads * d].cpu()[live], q_out.cpu()[live])
    assert torch.equal(qkv_g[:, heads * d :].cpu(), qkv[:, heads * d :])
    assert torch.equal(codes[1].cpu().view(torch.uint8)[..., :1, :], got.to(torch.float8_e4m3fn).view(torch.uint8)[..., :1, :])
    # read back, out of order and one block twice
    ids = torch.randperm(c.blocks, generator=c.gen)[: c.blocks - 1].int()
    ids = torch.cat((ids, ids[:1]))
    out = torch.empty(ids.numel(), 2, hkv, BS, d, dtype=torch.bfloat16, device=DEV)
    torch.ops.cdb.kv8_gather(codes, scales, 1, ids.to(DEV), out)
    vals = codes[1].cpu().double() * scales[1].cpu().double()[..., None, None]
    assert torch.equal(out.cpu().double(), vals[:, ids.long()].transpose(0, 1))


def test_append_extremes():
    """Zero rows, bf16's smallest and large values, infinities and NaN, and growth from the smallest scale."""

    d, hkv = 128, 1
    c = Cache([32] * 6, hkv, d, seed=9, layers=1)
    rows = torch.zeros(6, 3 * d)
    rows[1] = 2.0**-133
    rows[2] = 2.0**100
    rows[3, ::7] = float("inf")
    rows[3, 1::7] = float("-inf")
    rows[3, 2::7] = float("nan")
    rows[3, 3::7] = 1.5
    rows[4] = 448.0
    rows[5] = 449.0
    rows = rows.bfloat16()
    codes, scales, table = c.gpu()
    slot = torch.arange(6, dtype=torch.int32, device=DEV)
    for step in (0, 1):  # position 0, then position 1 with the rows turned round: every scale grows or stays
        src = rows if step == 0 else rows.flip(0)
        torch.ops.cdb.kv8_append(src.to(DEV), None, codes, scales, 0, table, slot, torch.full_like(slot, step), None, None, None, 0, 1)
        want_codes, want_scales = (c.codes[0].double(), c.scales[0].double()) if step == 0 else (want_codes, want_scales)
        ref.append(src, want_codes, want_scales, c.table, list(range(6)), [step] * 6, None, None, None, 0, 1)
        got = codes[0].cpu().double()
        assert torch.equal(scales[0].cpu().double(), want_scales)
        assert torch.equal(got.nan_to_num(nan=1e9), want_codes.nan_to_num(nan=1e9))
    assert ops.status_code() == 0


def test_indexes_out_of_range_are_reported_and_skipped():
    """Slots, positions and block ids that do not fit set the status word; what fits is done."""

    d = 64
    c = Cache([32] * 4, 1, d, seed=10, layers=1)
    c.table[1, 0] = c.blocks  # no such block
    codes, scales, table = c.gpu()
    before = codes.clone()
    slot = torch.tensor([0, 1, 99, 3, 2, 2], dtype=torch.int32, device=DEV)
    pos = torch.tensor([0, 0, 0, 16 * 500, 4, 4], dtype=torch.int32, device=DEV)  # and one position twice
    qkv = torch.randn(6, 3 * d, device=DEV).bfloat16()
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    sp = torch.cuda.current_stream().cuda_stream
    _lib.call("cdb_kv8_append", _lib.ptr(qkv), 3 * d, None, 0, _lib.ptr(codes), _lib.ptr(scales), 1, 0, c.blocks,
              _lib.ptr(table), table.stride(0), 4, table.shape[1], _lib.ptr(slot), _lib.ptr(pos), 0, None, None, 0, None,
              6, 1, 1, d, _lib.ptr(status), sp)
    assert int(status.item()) == 6
    changed = (codes.view(torch.uint8) != before.view(torch.uint8)).flatten(4).any(-1)[0, 0, :, 0].cpu()
    assert set(changed.nonzero().flatten().tolist()) <= {int(c.table[0, 0]), int(c.table[2, 0])}
    status.zero_()
    out = torch.full((6, d), 7.0, dtype=torch.bfloat16, device=DEV)
    ws = torch.empty(_lib.load().cdb_kv8_decode_workspace_floats(148, d), device=DEV)
    ctr = torch.zeros(_lib.load().cdb_kv8_decode_counters(148), dtype=torch.int32, device=DEV)
    _lib.call("cdb_kv8_decode_attention", _lib.ptr(qkv), 3 * d, _lib.ptr(out), d, _lib.ptr(codes), _lib.ptr(scales), 1, 0,
              c.blocks, _lib.ptr(table), table.stride(0), 4, table.shape[1], _lib.ptr(slot), _lib.ptr(pos), 6, 1, 1, d,
              0.125, 148, _lib.ptr(ws), ws.numel(), _lib.ptr(ctr), _lib.ptr(status), sp)
    assert int(status.item()) == 6
    assert (out[2] == 7).all() and (out[3] == 7).all()  # no such rows
    assert (out[1] == 0).all()  # nothing to attend to
    assert (out[0] != 7).any() and not ctr.any()
    status.zero_()
    back = torch.full((2, 2, 1, BS, d), 7.0, dtype=torch.bfloat16, device=DEV)
    ids = torch.tensor([c.blocks, 0], dtype=torch.int32, device=DEV)
    _lib.call("cdb_kv8_gather", _lib.ptr(codes), _lib.ptr(scales), 1, 0, c.blocks, 1, d, _lib.ptr(ids), 2, _lib.ptr(back), _lib.ptr(status), sp)
    assert int(status.item()) == 6 and (back[0] == 0).all() and (back[1] != 7).any()


@pytest.mark.parametrize("ctas", [1, 20, 148, 500])
def test_decode_with_any_number_of_ctas(ctas):
    """Through the C ABI: a few CTAs take everything; more CTAs than rows, with more rows than threads, too.
    One launch in place of the other gives the same values within the tolerance."""

    d, n = 64, 400
    pos = [(7 * i) % 60 - 1 for i in range(n)]
    slots = [i % 12 for i in range(n)]
    c = Cache([60] * 12, 1, d, seed=12, layers=1)
    codes, scales, table = c.gpu()
    q = torch.randn(n, d, generator=c.gen).bfloat16()
    qg, out = q.to(DEV), torch.full((n, d), 7.0, dtype=torch.bfloat16, device=DEV)
    slot, posg = (torch.tensor(v, dtype=torch.int32, device=DEV) for v in (slots, pos))
    ws = torch.empty(_lib.load().cdb_kv8_decode_workspace_floats(ctas, d), device=DEV)
    ctr = torch.zeros(_lib.load().cdb_kv8_decode_counters(ctas), dtype=torch.int32, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    _lib.call("cdb_kv8_decode_attention", _lib.ptr(qg), d, _lib.ptr(out), d, _lib.ptr(codes), _lib.ptr(scales), 1, 0, c.blocks,
              _lib.ptr(table), table.stride(0), 12, table.shape[1], _lib.ptr(slot), _lib.ptr(posg), n, 1, 1, d, d**-0.5, ctas,
              _lib.ptr(ws), ws.numel(), _lib.ptr(ctr), _lib.ptr(status), torch.cuda.current_stream().cuda_stream)
    assert int(status.item()) == 0 and not ctr.any()
    _check_rows(out.cpu(), c, q, pos, 1, layer=0, slots=slots)


def test_decode_on_two_streams_and_in_two_graphs():
    """Calls that split rows, on two streams at once and in two graphs replayed at once, keep their
    workspaces apart."""

    c = Cache([6000, 5000], 1, 128, seed=11, layers=1)
    codes, scales, table = c.gpu()
    pos = torch.tensor([5999, 4999], dtype=torch.int32, device=DEV)
    slot = torch.arange(2, dtype=torch.int32, device=DEV)
    qs = [torch.randn(2, 128, device=DEV).bfloat16() for _ in range(2)]
    outs = [torch.zeros(2, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2)]

    def call(i):
        torch.ops.cdb.kv8_decode_attention(qs[i], outs[i], codes, scales, 0, table, slot, pos, 1, 0.1)

    want = []
    for i in range(2):
        call(i)
        want.append(outs[i].clone())
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    graphs = []
    for i, s in enumerate(streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            call(i)
        graphs.append(g)
    for rep in range(20):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                if rep % 2:
                    graphs[i].replay()
                else:
                    call(i)
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want)), rep


def _prefill(c: Cache, q, spans, heads, layer=1, extra_tiles=0, table=None, codes=None):
    codes_g, scales, table_g = c.gpu()
    tiles, row = [], 0
    for s, (first, n) in enumerate(spans):
        tiles += [(row + i, min(64, n - i), s, first + i) for i in range(0, n, 64)]
        row += n
    tiles = tiles[::-1] + [(0, 0, 0, 0)] * extra_tiles
    out = torch.full((row, heads * c.codes.shape[-1]), 7.0, dtype=torch.bfloat16, device=DEV)
    torch.ops.cdb.kv8_prefill_attention(q.to(DEV), out, codes_g, scales, layer, table_g,
                                        torch.tensor(tiles, dtype=torch.int32, device=DEV), heads, c.codes.shape[-1] ** -0.5)
    torch.cuda.synchronize()
    assert ops.status_code() == 0
    return out.cpu()


def _check_prefill(out, c: Cache, q, spans, heads, layer=1):
    d, row = c.codes.shape[-1], 0
    for s, (first, n) in enumerate(spans):
        o, a = ref.attend(q[row : row + n].view(n, heads, d), c.codes[layer], c.scales[layer], c.table[s], first, d**-0.5)
        got = out[row : row + n].double().view(n, heads, d)
        assert ((got - o).abs() <= 2.0**-8 * o.abs() + 2.0**-10 * a).all(), (s, first, n)
        row += n


@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("kv_heads,group", [(1, 1), (2, 3), (1, 8)])
def test_prefill_matches_definition(d, kv_heads, group):
    spans = [(0, 1), (0, 64), (5, 65), (100, 130), (63, 2), (300, 17), (0, 200), (1000, 64)]
    heads = kv_heads * group
    c = Cache([a + n for a, n in spans], kv_heads, d, seed=d + heads)
    q = torch.randn(sum(n for _, n in spans), heads * d, generator=c.gen).bfloat16()
    _check_prefill(_prefill(c, q, spans, heads, extra_tiles=3), c, q, spans, heads)


def test_prefill_of_one_row_is_decode():
    spans = [(p, 1) for p in (0, 3, 16, 200, 511)]
    c = Cache([p + 1 for p, _ in spans], 2, 128, seed=30)
    q = torch.randn(5, 4 * 128, generator=c.gen).bfloat16()
    _check_prefill(_prefill(c, q, spans, 4), c, q, spans, 4)
    _check_prefill(_decode(c, q, [p for p, _ in spans], 4), c, q, spans, 4)


def test_prefill_scales_far_apart():
    spans = [(40, 60)]
    c = Cache([100], 1, 128, seed=31)
    c.scales[1, 1, c.table[0, 1].long()] = 2.0**40
    c.scales[1, 1, c.table[0, 3].long()] = 2.0**-40
    c.scales[1, 1, c.table[0, 6].long()] = 2.0**-126
    q = torch.randn(60, 128, generator=c.gen).bfloat16() * 30
    _check_prefill(_prefill(c, q, spans, 1), c, q, spans, 1)


def test_prefill_masked_places_hold_nan():
    """NaN in keys and values that a row may not see does not reach it; rows that see it get it, in the
    dims that hold it."""

    spans = [(10, 80), (0, 50)]
    c = Cache([90, 50], 1, 64, seed=32)
    q = torch.randn(130, 2 * 64, generator=c.gen).bfloat16()
    want = _prefill(c, q, spans, 2)
    raw = c.codes.view(torch.uint8)
    for s, (first, n) in enumerate(spans):  # behind the last token
        end = first + n
        raw[1, :, int(c.table[s, (end - 1) // BS]), :, (end - 1) % BS + 1 :] = 0xFF
    assert torch.equal(_prefill(c, q, spans, 2), want)
    raw[1, 1, int(c.table[0, 70 // BS]), 0, 70 % BS, 5] = 0x7F  # one value of position 70
    got = _prefill(c, q, spans, 2)
    sees = torch.zeros(130, dtype=torch.bool)
    sees[60:80] = True  # positions 70 .. 89
    bad = got.isnan().view(130, 2, 64)
    assert bad[sees][:, :, 5].all() and bad.sum() == 20 * 2
    assert torch.equal(got.nan_to_num(0)[~sees], want[~sees])
    raw[1, 0, int(c.table[0, 64 // BS]), 0, 0, 0] = 0x7F  # a key of position 64: rows that see it are NaN throughout
    got = _prefill(c, q, spans, 2)
    assert torch.equal(got[:54], want[:54]) and got[54:80].isnan().all() and torch.equal(got[80:], want[80:])


@pytest.mark.parametrize("order", ["shuffled", "interleaved", "twice", "short_copy", "short_followers"])
@pytest.mark.parametrize("pad", [0, 500])  # lists that are searched, and longer ones
def test_prefill_takes_tiles_in_any_order(order, pad):
    """Neighbours apart, requests in turn, every tile listed twice, a full tile also listed as a short one: each
    row comes out once, as it does in order."""

    spans = [(3, 300), (64, 200), (128, 128), (700, 65)]
    c = Cache([a + n for a, n in spans], 1, 64, seed=34)
    q = torch.randn(sum(n for _, n in spans), 2 * 64, generator=c.gen).bfloat16()
    codes, scales, table = c.gpu()
    tiles, row = [], 0
    for s, (first, n) in enumerate(spans):
        tiles += [(row + i, min(64, n - i), s, first + i) for i in range(0, n, 64)]
        row += n
    if order == "shuffled":
        tiles = [tiles[i] for i in torch.randperm(len(tiles), generator=c.gen).tolist()]
    elif order == "interleaved":
        tiles = sorted(tiles, key=lambda t: (t[3] // 64 % 3, t[2]))
    elif order == "twice":
        tiles = [t for t in tiles for _ in range(2)]
    elif order == "short_followers":
        tiles = [e for t in tiles for e in ((t, (t[0], max(1, t[1] // 2), t[2], t[3])) if (t[3] - spans[t[2]][0]) // 64 % 2 else (t,))]
    else:
        tiles = [e for t in tiles for e in (t, (t[0], max(1, t[1] // 2), t[2], t[3]))]
    tiles += [(0, 0, 0, 0)] * pad
    out = torch.full((row, 2 * 64), 7.0, dtype=torch.bfloat16, device=DEV)
    torch.ops.cdb.kv8_prefill_attention(q.to(DEV), out, codes, scales, 1, table,
                                        torch.tensor(tiles, dtype=torch.int32, device=DEV), 2, 64**-0.5)
    torch.cuda.synchronize()
    assert ops.status_code() == 0
    _check_prefill(out.cpu(), c, q, spans, 2)


def test_prefill_refuses_tiles_that_do_not_fit():
    c = Cache([64] * 2, 1, 64, seed=33, layers=1)
    c.table[1, 2] = -5
    codes, scales, table = c.gpu()
    q = torch.randn(64, 64, device=DEV).bfloat16()
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    sp = torch.cuda.current_stream().cuda_stream

    def call(*tile):
        out = torch.full((64, 64), 7.0, dtype=torch.bfloat16, device=DEV)
        status.zero_()
        t = torch.tensor([tile], dtype=torch.int32, device=DEV)
        _lib.call("cdb_kv8_prefill_attention", _lib.ptr(q), 64, _lib.ptr(out), 64, 64, _lib.ptr(codes), _lib.ptr(scales), 1, 0,
                  c.blocks, _lib.ptr(table), table.stride(0), 2, table.shape[1], _lib.ptr(t), 1, 1, 1, 64, 0.125,
                  _lib.ptr(status), sp)
        return out, int(status.item())

    for tile in [(0, 65, 0, 0), (1, 64, 0, 0), (-1, 4, 0, 0), (0, 4, 2, 0), (0, 4, -1, 0), (0, 4, 0, -1), (0, 64, 0, 5000),
                 (0, 64, 0, 2**31 - 8)]:
        out, code = call(*tile)
        assert code == 6 and (out == 7).all(), tile
    out, code = call(0, 0, 99, -4)
    assert code == 0 and (out == 7).all()
    out, code = call(0, 64, 1, 0)  # a missing block: its keys do not count
    assert code == 6 and out.isfinite().all() and (out[:, :] != 7).any()


def test_blocks_beyond_four_gigabytes():
    """Codes that lie past 2^32 bytes from the cache's start, and past it from V's: the same values, bit for bit, as
    from a small cache that holds the same blocks."""

    d, heads, n = 128, 2, 70
    far_blocks = 1 << 21  # 2 x 4 GiB of codes
    c = Cache([n], 1, d, seed=40, layers=1)
    ids = [int(b) for b in c.table[0] if b >= 0]
    far = {b: far_blocks - 1 - 7 * i for i, b in enumerate(ids)}
    far_table = c.table.clone()
    far_table[0, : len(ids)] = torch.tensor([far[b] for b in ids], dtype=torch.int32)
    qkv = torch.randn(n, (heads + 2) * d, generator=c.gen).bfloat16().to(DEV)
    slot = torch.zeros(n, dtype=torch.int32, device=DEV)
    pos = torch.arange(n, dtype=torch.int32, device=DEV)
    tiles = torch.tensor([(0, 64, 0, 0), (64, 6, 0, 64)], dtype=torch.int32, device=DEV)
    got = []
    for blocks, table in ((c.blocks, c.table), (far_blocks, far_table)):
        codes = torch.empty(1, 2, blocks, 1, BS, d, dtype=torch.float8_e4m3fn, device=DEV)
        scales = torch.empty(1, 2, blocks, 1, device=DEV)
        t = table.to(DEV)
        q = torch.empty(n, heads * d, dtype=torch.bfloat16, device=DEV)
        out, pre = torch.empty_like(q), torch.empty_like(q)
        back = torch.empty(len(ids), 2, 1, BS, d, dtype=torch.bfloat16, device=DEV)
        torch.ops.cdb.kv8_append(qkv, q, codes, scales, 0, t, slot, pos, None, None, None, 0, heads)
        torch.ops.cdb.kv8_gather(codes, scales, 0, t[0, : len(ids)].contiguous(), back)
        torch.ops.cdb.kv8_decode_attention(q, out, codes, scales, 0, t, slot, pos, heads, 0.1)
        torch.ops.cdb.kv8_prefill_attention(q, pre, codes, scales, 0, t, tiles, heads, 0.1)
        back[-1, :, :, n % BS :] = 0  # never written
        got.append((q, out, pre, back))
    torch.cuda.synchronize()
    assert ops.status_code() == 0
    assert all(torch.equal(a, b) for a, b in zip(*got))
    assert got[0][1].isfinite().all() and (got[0][1].float() - got[0][2].float()).abs().max() < 0.1


def test_no_rows():
    c = Cache([16], 1, 64, seed=41, layers=1)
    codes, scales, table = c.gpu()
    none, ints = torch.empty(0, 3 * 64, dtype=torch.bfloat16, device=DEV), torch.empty(0, dtype=torch.int32, device=DEV)
    q = torch.empty(0, 64, dtype=torch.bfloat16, device=DEV)
    torch.ops.cdb.kv8_append(none, q, codes, scales, 0, table, ints, ints, None, None, None, 0, 1)
    torch.ops.cdb.kv8_decode_attention(q, q.clone(), codes, scales, 0, table, ints, ints, 1, 0.1)
    torch.ops.cdb.kv8_prefill_attention(q, q.clone(), codes, scales, 0, table, ints.view(0, 4), 1, 0.1)
    torch.ops.cdb.kv8_gather(codes, scales, 0, ints, torch.empty(0, 2, 1, BS, 64, dtype=torch.bfloat16, device=DEV))
    torch.cuda.synchronize()
    assert ops.status_code() == 0 and torch.equal(codes.cpu().view(torch.uint8), c.codes.view(torch.uint8))
