"""The next token from logits and one random number, against a sorted 64-bit statement: tokens equal, log-probabilities
to one rounding (2^-24 of the value) and what the 64-bit sums leave (2^-30, far above them).
"""

from __future__ import annotations

import math

import pytest
import torch

import continuous_depth_batching_b200.ops  # noqa: F401  (registers torch.ops.cdb.*)
import continue_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
INF, NAN = math.inf, math.nan


def _call(logits, u, t, k=None, p=None, m=None, logp=True):
    n = logits.shape[0]
    f32 = dict(dtype=torch.float32, device=DEV)
    ids = torch.full((n + 1,), -77, dtype=torch.int64, device=DEV)
    out = torch.full((n + 1,), -77.0, **f32) if logp else None
    give = lambda x, **kw: None if x is None else torch.tensor(x, **kw)  # noqa: E731
    torch.ops.cdb.sample_tokens(logits, give(u, **f32), give(t, **f32), give(k, dtype=torch.int32, device=DEV), give(p, **f32), give(m, **f32), ids[:n],
                                out[:n] if logp else None)
    torch.cuda.synchronize()
    assert ids[n] == -77 and (not logp or out[n] == -77)
    return ids[:n].tolist(), out[:n].tolist() if logp else None


def _check(logits, u, t, k=None, p=None, m=None):
    n = logits.shape[0]
    f = lambda x: torch.tensor(x, dtype=torch.float32).tolist()  # noqa: E731  (as the kernel is given them)
    ids, logp = _call(logits, u, t, k, p, m)
    cpu = logits.cpu()
    for i in range(n):
        want, lp = ref.sample(cpu[i], f(u)[i], f(t)[i], 0 if k is None else k[i], 1.0 if p is None else f(p)[i], 0.0 if m is None else f(m)[i])
        assert ids[i] == want, (i, ids[i], want)
        assert (math.isnan(lp) and math.isnan(logp[i])) or abs(logp[i] - lp) <= 2.0**-24 * abs(lp) + 2.0**-30, (i, logp[i], lp)


def _rows(n, v, dtype, g, spread=2.5):
    x = torch.randn(n, v, generator=g) * spread
    x[:, :: max(1, v // 20)] += 4
    return x.to(dtype).to(DEV)


def _mixed(n, g):
    r = lambda: torch.rand(n, generator=g).tolist()  # noqa: E731
    return r(), [0.4 + x for x in r()]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("v", [1, 2, 3, 31, 33, 100, 257, 1000, 1025, 4097, 50257, 49152, 65536, 131071])
@pytest.mark.parametrize("filters", ["none", "k", "p", "m", "kp", "kpm"])
def test_against_sorting(dtype, v, filters):
    g = torch.Generator().manual_seed(v + len(filters))
    n = 9 if v < 40000 else 4
    u, t = _mixed(n, g)
    k = [1 + int(x * min(v, 300)) for x in torch.rand(n, generator=g).tolist()] if "k" in filters else None
    p = (0.3 + 0.69 * torch.rand(n, generator=g)).tolist() if "p" in filters else None
    m = (0.001 + 0.2 * torch.rand(n, generator=g)).tolist() if "m" in filters else None
    _check(_rows(n, v, dtype, g), u, t, k, p, m)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("v", [5, 700, 20000])
def test_equal_logits(dtype, v):
    """Rows of a few distinct values, so that every border falls among equal logits."""

    g = torch.Generator().manual_seed(v)
    n = 12
    x = torch.randint(0, 4, (n, v), generator=g).float() * 0.5
    x[0] = 3.0
    x[1] = -1e-3
    x[2, 1:] = x[2, 0] - 1e-30
    u, t = _mixed(n, g)
    k = [1 + i * v // 13 for i in range(n)]
    p = (0.05 + 0.9 * torch.rand(n, generator=g)).tolist()
    x = x.to(dtype).to(DEV)
    _check(x, u, t, k)
    _check(x, u, t, None, p)
    _check(x, u, t, k, p, [0.3] * n)


def test_borders_that_numbers_meet_exactly():
    x = torch.zeros(5, 4, device=DEV)
    # running sums 1, 2, 3, 4: the first that passes u * 4
    assert _call(x, [0.0, 0.25, 0.5, 0.75, 0.999], [1.0] * 5)[0] == [0, 1, 2, 3, 3]
    # three of four hold exactly 0.75 of the weight
    ids, logp = _call(x, [0.0, 0.34, 0.67, 0.99, 0.3], [1.0] * 5, None, [0.75] * 5)
    assert ids == [0, 1, 2, 2, 0] and all(abs(a + math.log(3)) < 1e-6 for a in logp)
    # w = min_p exactly: kept
    y = torch.tensor([[0.0, 0.0, -INF, 0.0]], device=DEV).repeat(2, 1)
    assert _call(y, [0.99, 0.5], [1.0, 1.0], None, None, [1.0, 1.0])[0] == [3, 1]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_temperatures_and_numbers_at_their_ends(dtype):
    g = torch.Generator().manual_seed(1)
    t = [0.0, -0.0, -1.0, NAN, 1e-30, 1e-3, 1e3, 1e30, INF, 1e-45]
    n = len(t)
    x = _rows(n, 999, dtype, g)
    x[:, 500] = x.amax(1) - 0.0  # two largest
    _check(x, torch.rand(n, generator=g).tolist(), t, None, None, None)
    _check(x, torch.rand(n, generator=g).tolist(), t, [40] * n, [0.7] * n, [0.01] * n)
    u = [0.0, -0.0, -3.0, NAN, 1.0, 7.0, INF, 1 - 2.0**-24, 2.0**-30, -INF]
    _check(x, u, [0.9] * n)
    _check(x, u, [0.9] * n, [7] * n, [0.8] * n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_filters_at_their_ends(dtype):
    g = torch.Generator().manual_seed(2)
    v = 777
    k = [0, -5, 1, 2, v - 1, v, v + 1, 2**31 - 1, -(2**31)]
    n = len(k)
    x = _rows(n, v, dtype, g)
    u, t = _mixed(n, g)
    _check(x, u, t, k)
    p = [0.0, -1.0, 1e-9, 1.0, 2.0, NAN, INF, 1 - 2.0**-24, 2.0**-149]
    _check(x, u, t, None, p)
    m = [0.0, -1.0, 1e-9, 1.0, 2.0, NAN, INF, 1 - 2.0**-24, 2.0**-149]
    _check(x, u, t, None, None, m)
    _check(x, u, t, k, p, m)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_infinities_and_nan(dtype):
    g = torch.Generator().manual_seed(4)
    x = torch.randn(9, 300, generator=g) * 2
    x[0] = -INF
    x[1] = NAN
    x[2, ::2] = -INF
    x[3, 5::7] = NAN
    x[4, [10, 20, 30]] = INF
    x[5, 17] = INF
    x[5, 18:] = NAN
    x[6] = torch.finfo(torch.bfloat16).min  # masks of the type's lowest value
    x[7, 1:] = torch.finfo(torch.bfloat16).min
    x[8, :] = -INF
    x[8, 299] = -1e30
    x = x.to(dtype).to(DEV)
    n = 9
    for u in (0.0, 0.37, 0.99999):
        _check(x, [u] * n, [0.8] * n)
        _check(x, [u] * n, [0.8] * n, [200] * n)
        _check(x, [u] * n, [0.8] * n, [2] * n, [0.9] * n, [0.1] * n)
        _check(x, [u] * n, [0.0] * n)
        _check(x, [u] * n, [INF] * n, [250] * n, [0.9] * n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("v,pitch,offset", [(1000, 1003, 1), (1000, 1000, 3), (4096, 4099, 0), (65, 71, 5), (30011, 30017, 7)])
def test_strides_and_alignments(dtype, v, pitch, offset):
    g = torch.Generator().manual_seed(v)
    n = 6
    whole = torch.full((n * pitch + offset + 16,), 1e4, dtype=dtype, device=DEV)  # large logits between the rows
    x = whole[offset : offset + n * pitch].view(n, pitch)[:, :v]
    x.copy_(_rows(n, v, dtype, g))
    u, t = _mixed(n, g)
    _check(x, u, t)
    _check(x, u, t, [50] * n, [0.9] * n)
    _check(x, u, t, None, [0.95] * n, [0.02] * n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("spread", [0.0, 1e-6, 1e-3, 0.05, 30.0, 3000.0])
def test_flat_and_steep_rows(dtype, spread):
    """From rows whose logits hardly differ (a border bin holds the whole row) to rows of one likely token."""

    g = torch.Generator().manual_seed(11)
    n, v = 5, 33000
    x = (torch.randn(n, v, generator=g) * spread + 1.25).to(dtype).to(DEV)
    u, t = _mixed(n, g)
    _check(x, u, t)
    _check(x, u, t, None, [0.2, 0.5, 0.9, 0.99, 0.999])
    _check(x, u, t, [1, 50, 1000, 20000, 32999])
    _check(x, u, t, [32999, 20000, 1000, 50, 1], [0.9] * n, [0.5] * n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_wide_vocabularies(dtype):
    g = torch.Generator().manual_seed(12)
    for v in (300_001, 2**20 + 5):
        x = _rows(2, v, dtype, g)
        _check(x, [0.3, 0.8], [1.0, 0.7], [0, 4000], [0.97, 0.9])
        _check(x, [0.6, 0.1], [1.0, 0.7])


@pytest.mark.parametrize("rows", [1, 2, 7, 80, 149, 300, 700])
def test_many_rows(rows):
    g = torch.Generator().manual_seed(rows)
    v = 5000
    x = _rows(rows, v, torch.bfloat16, g)
    u, t = _mixed(rows, g)
    ids, _ = _call(x, u, t, [20] * rows, [0.9] * rows, logp=False)
    cpu = x.cpu()
    f = lambda a: torch.tensor(a, dtype=torch.float32).tolist()  # noqa: E731
    assert ids == [ref.sample(cpu[i], f(u)[i], f(t)[i], 20, f([0.9])[0])[0] for i in range(rows)]


def test_no_rows():
    assert _call(torch.zeros(0, 5, device=DEV), [], [])[0] == []


def test_in_a_graph_and_on_another_stream():
    g = torch.Generator().manual_seed(5)
    n, v = 33, 49152
    xs = [_rows(n, v, torch.bfloat16, g) for _ in range(3)]
    us = [torch.rand(n, generator=g).to(DEV) for _ in range(3)]
    t, p, k = torch.full((n,), 0.8, device=DEV), torch.full((n,), 0.9, device=DEV), torch.full((n,), 100, dtype=torch.int32, device=DEV)
    want = []
    for x, u in zip(xs, us):
        ids, logp = torch.empty(n, dtype=torch.int64, device=DEV), torch.empty(n, device=DEV)
        torch.ops.cdb.sample_tokens(x, u, t, k, p, None, ids, logp)
        want.append((ids, logp))
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    x, u = xs[0].clone(), us[0].clone()
    ids, logp = torch.empty(n, dtype=torch.int64, device=DEV), torch.empty(n, device=DEV)
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        torch.ops.cdb.sample_tokens(x, u, t, k, p, None, ids, logp)
    for i in (2, 0, 1):
        x.copy_(xs[i])
        u.copy_(us[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(ids, want[i][0]) and torch.equal(logp, want[i][1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shift", [-40.0, -9.0, -0.75, 0.0, 0.75])
@pytest.mark.parametrize("filters", ["p", "kp", "kpm"])
def test_borders_below_and_about_zero(dtype, shift, filters):
    """Borders among negative logits, among ones next to zero (both signs, zeros too), and at the ends of the steps of 2^-7
    that the upper 16 bits take: a number, and its 32-bit neighbours on either side."""

    g = torch.Generator().manual_seed(int(shift * 4) + 1000)
    n, v = 10, 9001
    x = torch.randn(n, v, generator=g) * 1.5 + shift
    x[:, 5::11] = x[:, 5::11].bfloat16().float()
    x[:, 6::11] = torch.nextafter(x[:, 5::11][:, : x[:, 6::11].shape[1]], torch.tensor(INF))
    x[:, 7::11] = torch.nextafter(x[:, 5::11][:, : x[:, 7::11].shape[1]], torch.tensor(-INF))
    x[::2, ::13] *= 1e-5  # next to zero
    x[::3, ::17] = torch.tensor([0.0, -0.0]).repeat(v)[: x[::3, ::17].shape[1]]
    u, t = _mixed(n, g)
    p = (0.2 + 0.79 * torch.rand(n, generator=g)).tolist()
    k = torch.randint(600, 8000, (n,), generator=g).tolist() if "k" in filters else None
    m = [0.001] * n if "m" in filters else None
    _check(x.to(dtype).to(DEV), u, t, k, p, m)
