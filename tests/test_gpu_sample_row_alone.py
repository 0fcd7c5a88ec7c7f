"""A row's token and log-probability depend on nothing but the row: not on how many others stand beside it, by which the
kernel's width is chosen. Rows of every way through it, in calls of 148 rows and of 149."""

from __future__ import annotations

import math

import pytest
import torch

import continuous_depth_batching_b200.ops  # noqa: F401  (registers torch.ops.cdb.*)

pytestmark = pytest.mark.gpu
DEV = "cuda"
ROWS = 149


def _rows(dtype, v, g):
    x = torch.randn(ROWS, v, generator=g)
    x[:, 17] = 18.0  # all but certain, so that a log-probability shows its token's competitors to the last bit
    x[1::8, 17] = 2.0
    x[2::8, 5] = 1e-12  # more octaves below the largest than bf16 has bins
    x[3::8] *= 3
    x[4::8] = 1.5  # all equal
    x[5::8, ::9] = -math.inf
    x[6::8] = 1.5 + 1e-4 * x[6::8]
    x[7::8, 100:] = -1e30
    return x.to(dtype).to(DEV)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("v", [1000, 9001, 33003])
@pytest.mark.parametrize("filters", ["none", "k", "p", "m", "kp", "kpm", "widek"])
def test_the_same_beside_147_and_148_others(dtype, v, filters):
    g = torch.Generator().manual_seed(v)
    x = _rows(dtype, v, g)
    r = lambda: torch.rand(ROWS, generator=g).to(DEV)  # noqa: E731
    u, t = r(), 0.5 + r()
    t[9::16] = 0.0
    u[::3] = 1e-9  # the first kept tokens, the certain one among them
    k = p = m = None
    if filters == "widek":
        k = torch.randint(500, v + 10, (ROWS,), generator=g).int().to(DEV)
    elif "k" in filters:
        k = torch.randint(1, 520, (ROWS,), generator=g).int().to(DEV)
        k[2::8] = torch.randint(257, 513, (k[2::8].numel(),), generator=g).int().to(DEV)
    if "p" in filters:
        p = 0.5 + 0.5 * r()
        p[::5] = 1 - 1e-6
    if "m" in filters:
        m = 1e-6 + 1e-3 * r()
    results = []
    for n in (148, 149):
        ids, logp = torch.full((n,), -7, dtype=torch.int64, device=DEV), torch.empty(n, device=DEV)
        cut = lambda a: None if a is None else a[:n].contiguous()  # noqa: E731
        torch.ops.cdb.sample_tokens(x[:n], cut(u), cut(t), cut(k), cut(p), cut(m), ids, logp)
        results.append((ids[:148], logp[:148].view(torch.int32)))
    assert torch.equal(results[0][0], results[1][0])
    assert torch.equal(results[0][1], results[1][1]), (results[0][1] != results[1][1]).nonzero().flatten().tolist()
