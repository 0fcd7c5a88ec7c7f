"""fp32 top-p where one bin holds more tokens than 32 bits can add the lower halves of: the bin's mean then still has to show
where the border lies, or the row is searched bit by bit, some ten times slower. Against the sorted 64-bit statement, and
against the time of the same row with that bin's tokens at its least value, whose lower halves are 0."""

from __future__ import annotations

import pytest
import torch

import continuous_depth_batching_b200.ops  # noqa: F401  (registers torch.ops.cdb.*)
import continue_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _call(x, p, u):
    one = lambda v: torch.full((1,), v, device=DEV)  # noqa: E731
    args = x.to(DEV), one(u), one(1.0), None, one(p), None, torch.empty(1, dtype=torch.int64, device=DEV), torch.empty(1, device=DEV)
    times = []
    for _ in range(4):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        torch.ops.cdb.sample_tokens(*args)
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b))
    return args[-2].item(), args[-1].item(), min(times)


@pytest.mark.parametrize("seed", [1, 2])
def test_a_bin_of_many_tokens(seed):
    g = torch.Generator().manual_seed(seed)
    v, heavy, p, u = 2**20, 350_000, 0.95, 0.6
    x = torch.randn(1, v, generator=g) + 4
    x[:, :heavy] = 8 + 0.06 * torch.rand(1, heavy, generator=g)
    token, logp, ms = _call(x, p, u)
    want, lp = ref.sample(x[0], torch.tensor(u).item(), 1.0, 0, torch.tensor(p).item())
    assert token == want and abs(logp - lp) <= 2.0**-24 * abs(lp) + 2.0**-30
    x[:, :heavy] = 8.0
    assert ms < 3 * _call(x, p, u)[2]
