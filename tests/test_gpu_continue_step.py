"""The operators that continue a prompt many times together, as a decode step of a one-layer model uses them: projection,
norms with rotation and append, attention over shared prompts, output projection, logits, next tokens. Two prompts are
written once, nine rows continue them eagerly and in one captured graph that is replayed for every step.

Each stage is compared with its plain 64-bit statement on what the stage before gave, with that stage's own tolerance
(test_gpu_qk_norm, test_gpu_prefix_decode, test_gpu_sample).
"""

from __future__ import annotations

import math

import pytest
import torch

import continuous_depth_batching_b200.ops as ops
import continue_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32 = dict(dtype=torch.int32, device=DEV)
BS, HEADS, KV, D, HIDDEN, VOCAB = 16, 8, 2, 64, 256, 1024
COLS = (HEADS + 2 * KV) * D
PROMPTS, COPIES, STEPS, BLOCKS, WIDTH = [53, 200], [4, 5], 12, 80, 20
N = sum(COPIES)


class Model:
    def __init__(self):
        g = torch.Generator().manual_seed(17)
        w = lambda *s: (torch.randn(*s, generator=g) * s[-1] ** -0.5).bfloat16()  # noqa: E731
        self.emb, self.qkv_w, self.o_w, self.head = torch.randn(VOCAB, HIDDEN, generator=g).bfloat16(), w(COLS, HIDDEN), w(HIDDEN, HEADS * D), w(VOCAB, HIDDEN) * 4
        self.q_w, self.k_w = (1 + 0.3 * torch.randn(D, generator=g)).bfloat16(), (1 + 0.3 * torch.randn(D, generator=g)).bfloat16()
        ang = torch.arange(WIDTH * BS, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
        ang = torch.cat((ang, ang), -1)
        self.cos, self.sin = ang.cos().bfloat16(), ang.sin().bfloat16()
        self.prompts = [torch.randint(0, VOCAB, (n,), generator=g) for n in PROMPTS]
        # the whole blocks of a prompt belong to all rows that continue it, the rest is every row's own
        free = iter(torch.randperm(BLOCKS, generator=g).tolist())
        self.table = torch.full((N + 1, WIDTH), -1, dtype=torch.int32)
        self.slot, self.start, at = list(range(N, 0, -1)), [0], 0
        for n, copies in zip(PROMPTS, COPIES):
            common = [next(free) for _ in range(n // BS)]
            for i in range(at, at + copies):
                row = common + [next(free) for _ in range((n + STEPS + BS - 1) // BS - n // BS)]
                self.table[self.slot[i], : len(row)] = torch.tensor(row, dtype=torch.int32)
            at += copies
            self.start.append(at)
        self.of = [j for j, c in enumerate(COPIES) for _ in range(c)]
        dev = lambda t: t.to(DEV)  # noqa: E731
        self.d = {k: dev(getattr(self, k)) for k in ("emb", "qkv_w", "o_w", "head", "q_w", "k_w", "cos", "sin", "table")}
        self.d_slot, self.d_start, self.d_prefix = torch.tensor(self.slot, **I32), torch.tensor(self.start, **I32), torch.tensor(PROMPTS, **I32)
        bf = dict(dtype=torch.bfloat16, device=DEV)
        self.pool = torch.empty(1, 2, BLOCKS * BS, KV, D, **bf)
        self.x, self.qkv, self.o, self.y, self.logits = (torch.empty(N, c, **bf) for c in (HIDDEN, COLS, HEADS * D, HIDDEN, VOCAB))
        self.pos, self.ids, self.logp = torch.empty(N, **I32), torch.empty(N, dtype=torch.int64, device=DEV), torch.empty(N, device=DEV)
        f = dict(dtype=torch.float32, device=DEV)
        self.u, self.t = torch.empty(N, **f), torch.linspace(0.5, 1.2, N, device=DEV)
        self.k, self.p, self.m = torch.tensor([0, 20, 40, 5, 0, 300, 1, 50, 0], **I32), torch.full((N,), 0.95, **f), torch.full((N,), 0.01, **f)

    def fill(self):
        """The prompts' keys and values: whole blocks once, the rest for every row."""

        self.pool.fill_(float("nan"))
        rows = []
        for j, n in enumerate(PROMPTS):
            mine = [i for i in range(N) if self.of[i] == j]
            rows += [(mine[0], p) for p in range(n // BS * BS)] + [(i, p) for i in mine for p in range(n // BS * BS, n)]
        tok = torch.stack([self.prompts[self.of[i]][p] for i, p in rows]).to(DEV)
        qkv = torch.empty(len(rows), COLS, dtype=torch.bfloat16, device=DEV)
        torch.ops.cdb.gemm_bf16(self.d["emb"][tok], self.d["qkv_w"], qkv)
        torch.ops.cdb.qk_norm_rope_append(qkv, None, self.pool, 0, self.d["table"], torch.tensor([self.slot[i] for i, _ in rows], **I32),
                                          torch.tensor([p for _, p in rows], **I32), self.d["q_w"], self.d["k_w"], self.d["cos"], self.d["sin"], 1, HEADS, 1e-6)
        self.pos.copy_(torch.tensor([PROMPTS[j] for j in self.of]))
        self.ids.copy_(torch.stack([self.prompts[j][-1] for j in self.of]))

    def step(self):
        cdb, d = torch.ops.cdb, self.d
        torch.index_select(d["emb"], 0, self.ids, out=self.x)
        cdb.gemm_bf16(self.x, d["qkv_w"], self.qkv)
        cdb.qk_norm_rope_append(self.qkv, self.qkv, self.pool, 0, d["table"], self.d_slot, self.pos, d["q_w"], d["k_w"], d["cos"], d["sin"], 1, HEADS, 1e-6)
        cdb.prefix_decode_attention(self.qkv, self.o, self.pool, 0, d["table"], self.d_slot, self.pos, self.d_start, self.d_prefix, HEADS, D**-0.5)
        cdb.gemm_bf16(self.o, d["o_w"], self.y)
        self.y += self.x
        cdb.gemm_bf16(self.y, d["head"], self.logits)
        cdb.sample_tokens(self.logits, self.u, self.t, self.k, self.p, self.m, self.ids, self.logp)
        self.pos += 1


def _uniform():
    g = torch.Generator().manual_seed(3)
    return [torch.rand(N, generator=g) for _ in range(STEPS)]


def test_rows_continue_two_prompts():
    model, us = Model(), _uniform()
    model.fill()
    eager = []
    for step, u in enumerate(us):
        model.u.copy_(u)
        ids_in, pos = model.ids.clone(), model.pos.tolist()
        model.step()
        torch.cuda.synchronize()
        assert ops.status_code() == 0
        eager.append((model.ids.clone(), model.logp.clone(), model.logits.clone()))
        # projection, norms and append
        qkv = torch.empty_like(model.qkv)
        torch.ops.cdb.gemm_bf16(model.d["emb"][ids_in], model.d["qkv_w"], qkv)
        q, k, v, size, at = ref.norm_append(qkv.cpu(), model.table, model.slot, pos, model.q_w, model.k_w, model.cos, model.sin, 1, HEADS, KV, 1e-6)
        got_q, pool = model.qkv.cpu()[:, : HEADS * D].view(N, HEADS, D), model.pool.cpu()[0]
        assert ((got_q.double() - q).abs() <= 2.0**-8 * q.abs() + 2.0**-17 * size[:, :HEADS]).all()
        assert ((pool[0, at].double() - k).abs() <= 2.0**-8 * k.abs() + 2.0**-17 * size[:, HEADS:]).all()
        assert torch.equal(pool[1, at].double(), v)
        # attention
        o = model.o.cpu().view(N, HEADS, D).double()
        for i in range(N):
            want, size = ref.attend(got_q[i], pool, model.table[model.slot[i]], pos[i], D**-0.5, BLOCKS)
            assert ((o[i] - want).abs() <= 2.0**-8 * want.abs() + 2.0**-8 * (size + want.abs()) + 2.0**-12 * size).all(), (step, i)
        # tokens
        logits, t, ids, logp = model.logits.cpu(), model.t.tolist(), model.ids.tolist(), model.logp.tolist()
        for i in range(N):
            want, lp = ref.sample(logits[i], u[i].item(), t[i], model.k[i].item(), model.p[i].item(), model.m[i].item())
            assert ids[i] == want and abs(logp[i] - lp) <= 2.0**-24 * abs(lp) + 2.0**-30, (step, i)
    # rows of one prompt went different ways
    first = torch.stack([e[0] for e in eager])
    assert len({tuple(first[:, i].tolist()) for i in range(N)}) > 2 and not math.isnan(float(eager[-1][1].sum()))
    # the same steps from one graph
    model.fill()
    keep = model.pos.clone(), model.ids.clone(), model.pool.clone()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        model.step()
    for to, was in zip((model.pos, model.ids, model.pool), keep):
        to.copy_(was)
    for step, u in enumerate(us):
        model.u.copy_(u)
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip((model.ids, model.logp, model.logits), eager[step]):
            assert torch.equal(got, want), step
    assert ops.status_code() == 0


def test_host_threads_at_once():
    """Two host threads, each with a stream, sizes and a model of its own, run steps at the same time."""

    import threading

    us, results = _uniform(), {}
    models = [Model(), Model()]
    want = []
    for model in models:
        model.fill()
        for u in us[:4]:
            model.u.copy_(u)
            model.step()
        torch.cuda.synchronize()
        want.append(model.ids.tolist())
        model.fill()
    torch.cuda.synchronize()

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for u in us[:4]:
                models[i].u.copy_(u)
                models[i].step()
            torch.cuda.current_stream().synchronize()
            results[i] = models[i].ids.tolist()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert results == {0: want[0], 1: want[1]}
    assert ops.status_code() == 0
