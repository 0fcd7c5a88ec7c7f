"""Prefix decode attention from two host threads on one stream: its launches hand a plan on to one another through that
stream's workspace, so none of another call's may come between them. The calls differ in rows, groups, heads and
lengths; every one gives what it gives alone."""

from __future__ import annotations

import threading

import pytest
import torch

import continuous_depth_batching_b200.ops as ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BS = 16
I32 = dict(dtype=torch.int32, device=DEV)
CALLS = 1500


def _call(sizes, prefix, extra, heads, kv, d):
    """``sizes`` rows of each group on ``prefix`` shared tokens and up to ``extra`` of their own."""

    g = torch.Generator().manual_seed(sum(sizes) + heads)
    n = sum(sizes)
    of = [i for i, s in enumerate(sizes) for _ in range(s)]
    lens = [prefix + 1 + int(x) for x in torch.randint(0, extra, (n,), generator=g)]
    shared, width = prefix // BS, (prefix + extra) // BS + 1
    blocks = len(sizes) * shared + n * (width - shared)
    ids = torch.randperm(blocks, generator=g).int()
    table = torch.empty(n, width, dtype=torch.int32)
    for i in range(n):
        table[i, :shared] = ids[of[i] * shared : (of[i] + 1) * shared]
        table[i, shared:] = ids[len(sizes) * shared + i * (width - shared) :][: width - shared]
    pool = torch.randn(1, 2, blocks * BS, kv, d, generator=g).bfloat16().to(DEV)
    q = torch.randn(n, heads * d, generator=g).bfloat16().to(DEV)
    edges = torch.tensor([0, *sizes]).cumsum(0).int().to(DEV)
    args = (pool, 0, table.to(DEV), torch.arange(n, **I32), torch.tensor([l - 1 for l in lens], **I32), edges, torch.full((len(sizes),), prefix, **I32), heads, d**-0.5)

    def run(out):
        torch.ops.cdb.prefix_decode_attention(q, out, *args)

    return run, torch.empty_like(q)


@pytest.mark.parametrize("sizes", [
    [([3], 700, 40, 4, 4, 64), ([40, 17], 2000, 90, 16, 4, 128)],
    [([64], 4000, 200, 8, 8, 128), ([64], 4000, 200, 8, 8, 128)],  # one shape, other tables
    [([1, 1, 1], 30, 5, 2, 1, 96), ([130], 600, 20, 32, 8, 64)],
])
def test_two_host_threads_on_one_stream(sizes):
    calls = [_call(*s) for s in sizes]
    want = []
    for run, out in calls:
        run(out)
        want.append(out.clone())
    torch.cuda.synchronize()
    stream, start, errors, wrong = torch.cuda.Stream(), threading.Barrier(2), [], {}

    def work(i):
        run, out = calls[i]
        with torch.cuda.stream(stream):
            bad = torch.zeros((), dtype=torch.int64, device=DEV)
            start.wait()
            try:
                for _ in range(CALLS):
                    run(out)
                    bad += (out != want[i]).sum()
                stream.synchronize()
                wrong[i] = int(bad)
            except RuntimeError as e:
                errors.append(str(e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors[0]
    assert wrong == {0: 0, 1: 0}
    assert ops.status_code() == 0
