"""The low-bit operators together, as a layer of a decoder uses them: step tables from the lengths, 4-bit QKV
projection, rotation and append to the 8-bit cache, attention, 4-bit output projection. A batch of prompts,
then decode steps, eagerly and in one captured graph that is replayed for every step.

Each stage is compared with its plain 64-bit statement on what the stage before gave, with that stage's own
tolerance (test_gpu_kv8, test_gpu_gemv_w4): a projection 2^-8 of the value and 2^-20 * 300 / 16 of max |s| sum
|x|; attention 2^-8 of the value and 2^-10 of sum p |v| / sum p; integers equal; rotated keys' codes equal but
for 1 in 10^4 next to a rounding border.
"""

from __future__ import annotations

import pytest
import torch

import continuous_depth_batching_b200.ops as ops
import kv8_reference as ref
from continuous_depth_batching_b200 import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"
BS, HEADS, KV, D, HIDDEN, GROUP = 16, 4, 2, 64, 256, 64
COLS = (HEADS + 2 * KV) * D
PROMPTS, STEPS, SLOTS, WIDTH, BLOCKS = [37, 5, 64, 1, 130], 20, 7, 12, 60


def _quantised(n, k, gen):
    w = torch.randint(0, 256, (n, k // 2), generator=gen, dtype=torch.uint8)
    s = (torch.rand(n, k // GROUP, generator=gen) * 0.02 + 0.005).bfloat16()
    z = torch.randint(6, 10, (n, k // GROUP), generator=gen, dtype=torch.uint8)
    return w, s, z


def _dense(w, s, z):
    q = torch.stack((w & 15, w >> 4), -1).view(w.shape[0], -1).double()
    return (q - z.double().repeat_interleave(GROUP, 1)) * s.double().repeat_interleave(GROUP, 1)


class Layer:
    """Weights, the cache and the allocator of one layer; ``step`` runs one batch through it."""

    def __init__(self):
        g = torch.Generator().manual_seed(5)
        self.qkv_w, self.o_w = _quantised(COLS, HIDDEN, g), _quantised(HIDDEN, HEADS * D, g)
        inv = 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
        ang = torch.arange(WIDTH * BS, dtype=torch.float64)[:, None] * inv
        ang = torch.cat((ang, ang), -1)
        self.cos, self.sin = ang.cos().bfloat16(), ang.sin().bfloat16()
        i32 = dict(dtype=torch.int32, device=DEV)
        self.dev = [tuple(t.to(DEV) for t in w) for w in (self.qkv_w, self.o_w)]
        self.dcos, self.dsin = self.cos.to(DEV), self.sin.to(DEV)
        self.ring, self.state, self.row_len = torch.empty(BLOCKS, **i32), torch.empty(4, **i32), torch.empty(SLOTS, **i32)
        self.slots = torch.tensor([3, 0, 6, 1, 4], **i32)
        self.table = torch.empty(SLOTS, WIDTH, **i32)
        self.seq_len = torch.empty(SLOTS, **i32)
        self.codes = torch.empty(1, 2, BLOCKS, KV, BS, D, dtype=torch.float8_e4m3fn, device=DEV)
        self.scales = torch.empty(1, 2, BLOCKS, KV, device=DEV)
        self.reset()

    def reset(self):
        p = _lib.ptr
        _lib.call("cdb_block_pool_init", p(self.ring), p(self.state), p(self.row_len), SLOTS, BLOCKS,
                  torch.cuda.current_stream().cuda_stream)
        self.table.fill_(-1)
        self.seq_len.zero_()
        self.codes.view(torch.uint8).fill_(0x7F)  # NaN wherever nothing is written
        self.scales.fill_(float("nan"))

    def buffers(self, n, cap):
        i32 = dict(dtype=torch.int32, device=DEV)
        bf = dict(dtype=torch.bfloat16, device=DEV)
        return dict(granted=torch.empty(n, **i32), cu_q=torch.empty(n + 1, **i32), cu_k=torch.empty(n + 1, **i32),
                    slot=torch.empty(cap, **i32), pos=torch.empty(cap, **i32),
                    map=torch.empty(cap, dtype=torch.int64, device=DEV), tiles=torch.empty(cap // 64 + n, 4, **i32),
                    x=torch.empty(cap, HIDDEN, **bf), qkv=torch.empty(cap, COLS, **bf), q=torch.empty(cap, HEADS * D, **bf),
                    o=torch.zeros(cap, HEADS * D, **bf), y=torch.empty(cap, HIDDEN, **bf), new=torch.ones(n, **i32))

    def step(self, b, prompts: bool):
        cdb = torch.ops.cdb
        cdb.step_tables(self.slots, self.seq_len, b["new"], self.row_len, self.table, self.ring, self.state, self.row_len,
                        self.state, b["granted"], b["cu_q"], b["cu_k"], b["slot"], b["pos"], b["map"], b["tiles"])
        cdb.gemv_w4(b["x"], *self.dev[0], b["qkv"])
        cdb.kv8_append(b["qkv"], b["q"], self.codes, self.scales, 0, self.table, b["slot"], b["pos"], self.dcos, self.dsin,
                       None, 1, HEADS)
        if prompts:
            cdb.kv8_prefill_attention(b["q"], b["o"], self.codes, self.scales, 0, self.table, b["tiles"], HEADS, D**-0.5)
        else:
            cdb.kv8_decode_attention(b["q"], b["o"], self.codes, self.scales, 0, self.table, b["slot"], b["pos"], HEADS, D**-0.5)
        cdb.gemv_w4(b["o"], *self.dev[1], b["y"])
        self.seq_len.index_add_(0, self.slots.long(), b["new"])


def _near_product(got, x, w):
    want = x.double() @ _dense(*w).t()
    size = x.double().abs().sum(1, keepdim=True) * w[1].double().abs().amax(1)[None, :]
    assert ((got.double() - want).abs() <= 2.0**-8 * want.abs() + 2.0**-20 * 300 / 16 * size).all()


def _inputs():
    g = torch.Generator().manual_seed(6)
    return [torch.randn(sum(PROMPTS), HIDDEN, generator=g).bfloat16()] + [torch.randn(len(PROMPTS), HIDDEN, generator=g).bfloat16()
                                                                          for _ in range(STEPS)]


def test_a_layer_over_prompts_and_decode_steps():
    layer, xs = Layer(), _inputs()
    n, cap = len(PROMPTS), sum(PROMPTS) + 9  # padding rows behind the prompts
    first, dec = layer.buffers(n, cap), layer.buffers(n, n)
    lens, slots = [0] * n, layer.slots.tolist()
    table = torch.full((SLOTS, WIDTH), -1, dtype=torch.int32)
    held, free = [0] * n, iter(range(BLOCKS))
    codes = torch.full((2, BLOCKS, KV, BS, D), float("nan"), dtype=torch.float64)
    scales = torch.full((2, BLOCKS, KV), float("nan"), dtype=torch.float64)
    eager = []
    for step, x in enumerate(xs):
        b, new = (first, PROMPTS) if step == 0 else (dec, [1] * n)
        rows = sum(new)
        b["new"].copy_(torch.tensor(new, dtype=torch.int32))
        b["x"].zero_()
        b["x"][:rows] = x.to(DEV)
        layer.step(b, step == 0)
        torch.cuda.synchronize()
        assert ops.status_code() == 0
        eager.append(b["y"][:rows].clone())
        # tables
        for j, s in enumerate(slots):
            while held[j] * BS < lens[j] + new[j]:
                table[s, held[j]] = next(free)
                held[j] += 1
        assert torch.equal(layer.table.cpu(), table)
        slot = [s for s, k in zip(slots, new) for _ in range(k)]
        pos = [lens[j] + i for j, k in enumerate(new) for i in range(k)]
        assert b["slot"][:rows].tolist() == slot and b["pos"][:rows].tolist() == pos
        assert (b["pos"][rows:] == -1).all()
        # projection, append
        qkv = b["qkv"][:rows].cpu()
        _near_product(qkv, x, layer.qkv_w)
        q = ref.append(qkv, codes, scales, table, slot, pos, layer.cos, layer.sin, None, 1, HEADS)
        assert torch.equal(layer.scales[0].cpu().double().nan_to_num(nan=-1), scales.nan_to_num(nan=-1))
        got = layer.codes[0].cpu().double()
        off = (got != codes) & ~(got.isnan() & codes.isnan())
        assert off.double().mean() <= 1e-4
        codes = got.clone()
        gotq = b["q"][:rows].cpu()
        assert ((gotq.double() - q.view(rows, -1)).abs() <= 2.0**-8 * q.view(rows, -1).abs() + 2.0**-18).all()
        # attention, projection
        o = b["o"][:rows].cpu()
        at = 0
        for j, s in enumerate(slots):
            want, size = ref.attend(gotq[at : at + new[j]].view(-1, HEADS, D), codes, scales, table[s], lens[j], D**-0.5)
            have = o[at : at + new[j]].double().view(-1, HEADS, D)
            assert ((have - want).abs() <= 2.0**-8 * want.abs() + 2.0**-10 * size).all(), (step, j)
            at += new[j]
        assert (b["o"][rows:] == 0).all()  # rows behind the last sequence
        _near_product(b["y"][:rows].cpu(), o, layer.o_w)
        lens = [a + k for a, k in zip(lens, new)]
    # the same decode steps from one graph
    layer.reset()
    first["new"].copy_(torch.tensor(PROMPTS, dtype=torch.int32))
    first["x"].zero_()
    first["x"][: sum(PROMPTS)] = xs[0].to(DEV)
    layer.step(first, True)
    torch.cuda.synchronize()
    keep = [t.clone() for t in (layer.ring, layer.state, layer.row_len, layer.table, layer.seq_len, layer.scales)]
    kept_codes = layer.codes.view(torch.uint8).clone()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        layer.step(dec, False)
    for t, k in zip((layer.ring, layer.state, layer.row_len, layer.table, layer.seq_len, layer.scales), keep):
        t.copy_(k)
    layer.codes.view(torch.uint8).copy_(kept_codes)
    for step in range(STEPS):
        dec["x"].copy_(xs[step + 1].to(DEV))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(dec["y"], eager[step + 1]), step
    assert ops.status_code() == 0
