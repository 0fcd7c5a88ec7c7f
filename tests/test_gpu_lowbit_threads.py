"""Calls of one low-bit operator at once, from two host threads on two streams, with sizes that take different
amounts of shared memory: each succeeds, and gives what it gives alone."""

from __future__ import annotations

import threading

import pytest
import torch

import continuous_depth_batching_b200.ops as ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32 = dict(dtype=torch.int32, device=DEV)


def _gemv(m, k):
    g = torch.Generator().manual_seed(k)
    x = torch.randn(m, k, generator=g).bfloat16().to(DEV)
    w = torch.randint(0, 256, (64, k // 2), generator=g, dtype=torch.uint8).to(DEV)
    s = torch.randn(64, k // 128, generator=g).bfloat16().to(DEV)
    out = torch.empty(m, 64, dtype=torch.bfloat16, device=DEV)
    return (lambda: torch.ops.cdb.gemv_w4(x, w, s, None, out)), [out]


def _decode(group):
    g = torch.Generator().manual_seed(group)
    codes = (torch.randn(1, 2, 6, 1, 16, 128, generator=g) * 50).to(torch.float8_e4m3fn).to(DEV)
    scales = torch.full((1, 2, 6, 1), 2.0**-6, device=DEV)
    q = torch.randn(2, group * 128, generator=g).bfloat16().to(DEV)
    out = torch.empty_like(q)
    table, slot, pos = torch.arange(6, **I32).view(2, 3), torch.arange(2, **I32), torch.tensor([40, 17], **I32)
    return (lambda: torch.ops.cdb.kv8_decode_attention(q, out, codes, scales, 0, table, slot, pos, group, 0.1)), [out]


def _tables(n):
    slots, lens, new, held = torch.arange(n, **I32), torch.zeros(n, **I32), torch.ones(n, **I32), torch.zeros(n, **I32)
    table, ring = torch.full((n, 2), -1, **I32), torch.arange(n, **I32)
    state = torch.tensor([0, n, n, 0], **I32)
    outs = [torch.empty(k, **I32) for k in (n, 4, n, n + 1, n + 1, n, n)]
    row_len, state_out, granted, cu_q, cu_k, slot, pos = outs
    rows = torch.empty(n, dtype=torch.int64, device=DEV)
    return (lambda: torch.ops.cdb.step_tables(slots, lens, new, held, table, ring, state, row_len, state_out, granted, cu_q,
                                              cu_k, slot, pos, rows, None)), [*outs, rows]


@pytest.mark.parametrize("make,sizes", [(_gemv, [(1, 2048), (8, 5632)]), (_decode, [(2,), (8,)]), (_tables, [(3,), (8000,)])])
def test_sizes_that_differ(make, sizes):
    calls = [make(*s) for s in sizes]
    want = []
    for call, outs in calls:
        call()
        want.append([o.clone() for o in outs])
    torch.cuda.synchronize()
    errors, start = [], threading.Barrier(2)

    def work(call):
        with torch.cuda.stream(torch.cuda.Stream()):
            start.wait()
            try:
                for _ in range(3000):
                    call()
            except RuntimeError as e:
                errors.append(str(e))

    threads = [threading.Thread(target=work, args=(call,)) for call, _ in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors[0]
    assert ops.status_code() == 0
    for (_, outs), w in zip(calls, want):
        assert all(torch.equal(a, b) for a, b in zip(outs, w))
