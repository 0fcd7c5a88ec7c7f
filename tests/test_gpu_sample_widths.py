"""Calls of more rows than SMs, which take the narrower kernel, two of them to an SM: every way through it, against the
sorted 64-bit statement (tolerance as in sampling's other tests: 2^-24 of the log-probability and 2^-30)."""

from __future__ import annotations

import math

import pytest
import torch

import continuous_depth_batching_b200.ops  # noqa: F401  (registers torch.ops.cdb.*)
import continue_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _rows(n, v, dtype, g):
    x = torch.randn(n, v, generator=g) * 2.5
    x[:, :: max(1, v // 20)] += 4
    x[3::10, ::3] = -math.inf
    x[5::10] = torch.randint(0, 4, x[5::10].shape, generator=g) * 0.5  # borders among equal logits
    x[7::30] = -0.75  # all equal
    x[8::30, 1] = 1e-15  # octaves below the others
    x[9::30] = -math.inf
    x[19::30, v // 2] = math.inf
    pitch = torch.full((n, v + 11), 1e4).to(dtype)
    pitch[:, 3 : v + 3] = x.to(dtype)
    return pitch.to(DEV)[:, 3 : v + 3]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,v", [(149, 5001), (300, 1025), (149, 9001), (151, 33), (297, 2)])
@pytest.mark.parametrize("filters", ["none", "k20", "k300", "k2000", "p", "m", "k300p", "k2000pm"])
def test_more_rows_than_sms(dtype, n, v, filters):
    g = torch.Generator().manual_seed(n + v + len(filters))
    x = _rows(n, v, dtype, g)
    r = lambda lo, hi: lo + (hi - lo) * torch.rand(n, generator=g)  # noqa: E731
    u, t = r(0, 1), r(0.4, 1.4)
    t[4::16] = 0.0
    k = p = m = None
    for size in (2000, 300, 20):
        if k is None and f"k{size}" in filters:
            k = torch.randint(size // 2, size + 1, (n,), generator=g).int()
            k[6::16] = 0
    if "p" in filters:
        p = r(0.2, 0.999)
    if "m" in filters:
        m = r(0.0, 0.1)
    ids, logp = torch.full((n + 1,), -77, dtype=torch.int64, device=DEV), torch.full((n + 1,), -77.0, device=DEV)
    d = lambda a: None if a is None else a.to(DEV)  # noqa: E731
    torch.ops.cdb.sample_tokens(x, d(u), d(t), d(k), d(p), d(m), ids[:n], logp[:n])
    ids, logp, cpu = ids.tolist(), logp.tolist(), x.cpu()
    assert ids[n] == -77 and logp[n] == -77
    off = lambda a, neutral, i: neutral if a is None else a[i].item()  # noqa: E731
    for i in range(n):
        want, lp = ref.sample(cpu[i], u[i].item(), t[i].item(), off(k, 0, i), off(p, 1.0, i), off(m, 0.0, i))
        assert ids[i] == want, (i, ids[i], want)
        assert (math.isnan(lp) and math.isnan(logp[i])) or abs(logp[i] - lp) <= 2.0**-24 * abs(lp) + 2.0**-30, (i, logp[i], lp)
