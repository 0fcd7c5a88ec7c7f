"""Rows whose weight lies in tokens of a magnitude far from the largest logit's: the difference of the two, which a weight
is computed from, then needs more than 24 bits, in bf16 too. Against the sorted 64-bit statement, with the tolerance of
sampling's other tests: one rounding of the log-probability, 2^-24 of its value, and 2^-30, which the weights' own error is
(2^-30 of each; each difference rounded would leave up to 2^-24 of the exponent: 2^-21 at 12)."""

from __future__ import annotations

import math

import pytest
import torch

import continuous_depth_batching_b200.ops  # noqa: F401  (registers torch.ops.cdb.*)
import continue_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
ROWS, VOCAB = 6, 60001
US = [0.05, 0.3, 0.61, 0.77, 0.9, 0.99]
FILTERS = {
    "none": {},
    "m": dict(m=[1e-7] * ROWS),
    "p": dict(p=[0.5, 0.8, 0.9, 0.97, 0.99, 0.999]),
    "few": dict(k=[1, 2, 50, 100, 400, 512]),
    "many": dict(k=[600, 1000, 5000, 20000, 40000, 60000]),
    "kp": dict(k=[600, 1000, 5000, 7000, 400, 60000], p=[0.9] * ROWS),
}


def _near_zero(g):
    """One token at 12, the others within 1e-5 of zero, either sign."""

    x = torch.randn(ROWS, VOCAB, generator=g) * 1e-5
    x[:, 12345] = 12.0
    x[1, 777] = 11.5
    return x


def _one_small_value(g):
    """The same, all of one value or another in a row, whose roundings do not average out."""

    x = torch.full((ROWS, VOCAB), 1.1e-5) * (1 + torch.arange(ROWS)[:, None])
    x[:, ::3] *= -2
    x[:, 12345] = 12.0
    return x


def _log_probabilities(g):
    """A token that is all but certain, at -1e-5 or so, the others about -11."""

    x = torch.randn(ROWS, VOCAB, generator=g) * 0.3 - 11
    x[:, 54321] = -torch.logspace(-7, -4, ROWS)
    return x


def _both(g):
    """Tokens about zero and far from it around a largest one of middling size."""

    x = torch.randn(ROWS, VOCAB, generator=g) * 1e-4
    x[:, ::2] = -3 + torch.randn(ROWS, (VOCAB + 1) // 2, generator=g)
    x[:, ::7] *= 1e-3
    x[:, 4321] = 0.02 * torch.arange(1, ROWS + 1)
    x[:, 5::100] = -math.inf  # banned
    return x.clamp(max=0.12)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("make", [_near_zero, _one_small_value, _log_probabilities, _both])
@pytest.mark.parametrize("filters", FILTERS)
def test_weights_of_far_logits(dtype, make, filters):
    g = torch.Generator().manual_seed(21)
    x = make(g).to(dtype)
    f = lambda v: None if v is None else torch.tensor(v, dtype=torch.float32)  # noqa: E731
    how = FILTERS[filters]
    k = torch.tensor(how["k"], dtype=torch.int32) if "k" in how else None
    p, m, u = f(how.get("p")), f(how.get("m")), f(US)
    t = f([1.0, 0.9, 1.0, 1.1, 1.0, 0.95])
    ids, logp = torch.empty(ROWS, dtype=torch.int64, device=DEV), torch.empty(ROWS, device=DEV)
    d = lambda v: None if v is None else v.to(DEV)  # noqa: E731
    torch.ops.cdb.sample_tokens(x.to(DEV), d(u), d(t), d(k), d(p), d(m), ids, logp)
    off = lambda v, neutral, i: neutral if v is None else v[i].item()  # noqa: E731
    for i in range(ROWS):
        want, lp = ref.sample(x[i], u[i].item(), t[i].item(), off(k, 0, i), off(p, 1.0, i), off(m, 0.0, i))
        got = logp[i].item()
        assert ids[i].item() == want, (i, ids[i].item(), want)
        assert abs(got - lp) <= 2.0**-24 * abs(lp) + 2.0**-30, (i, got, lp, abs(got - lp) / 2.0**-30)
