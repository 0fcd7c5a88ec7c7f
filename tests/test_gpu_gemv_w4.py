"""gemv_w4 against the product in 64 bits.

Tolerance. Weights and products are exact; sums are fp32: each of the K additions rounds to 2^-24 of a
partial sum that stays below s * (136 + 128 + z) * sum |x| of its group (the offset of 128 that is taken off
again), so 2^-20 * max |s| * 300 * sum |x| / 16 is far above what they add up to; the result is rounded to
bf16 once: 2^-8 of it.
"""

from __future__ import annotations

import pytest
import torch

import continuous_depth_batching_b200.ops as ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _weights(n, k, group, zeros, seed):
    g = torch.Generator().manual_seed(seed)
    w = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
    s = (torch.randn(n, k // group, generator=g) * 0.02).bfloat16()
    z = torch.randint(0, 256 if zeros == "any" else 16, (n, k // group), generator=g, dtype=torch.uint8) if zeros else None
    return w, s, z, g


def _dense(w, s, z, group):
    q = torch.stack((w & 15, w >> 4), -1).view(w.shape[0], -1).double()
    off = 8.0 if z is None else z.double().repeat_interleave(group, 1)
    return (q - off) * s.double().repeat_interleave(group, 1)


def _check(out, x, w, s, z, group):
    d = _dense(w, s, z, group)
    want = x.double() @ d.t()
    size = x.double().abs().sum(1, keepdim=True) * s.double().abs().amax(1)[None, :]
    assert ((out.double() - want).abs() <= 2.0**-8 * want.abs() + 2.0**-20 * 300 / 16 * size).all()


@pytest.mark.parametrize("m", [1, 2, 7, 8, 9, 16, 17, 24, 31, 32, 33, 70])
@pytest.mark.parametrize("n,k,group,zeros", [(64, 256, 64, False), (100, 1024, 128, True), (2048, 2048, 32, True)])
def test_tokens(m, n, k, group, zeros):
    w, s, z, g = _weights(n, k, group, zeros, m + n)
    x = torch.randn(m, k, generator=g).bfloat16()
    out = torch.full((m, n), 7.0, dtype=torch.bfloat16, device=DEV)
    torch.ops.cdb.gemv_w4(x.to(DEV), w.to(DEV), s.to(DEV), None if z is None else z.to(DEV), out)
    torch.cuda.synchronize()
    assert ops.status_code() == 0
    _check(out.cpu(), x, w, s, z, group)


@pytest.mark.parametrize("n,k,group,zeros", [
    (1, 32, 32, False), (1, 128, 128, True), (15, 96, 32, True), (17, 64, 64, False), (129, 5632, 128, True),
    (5280, 5280, 32, False), (33, 17920, 128, "any"), (700, 2112, 64, "any"), (65, 2304, 2304, True), (257, 768, 384, False),
    (130, 40960, 256, True),
])
@pytest.mark.parametrize("m", [1, 5, 20, 32])
def test_sizes(n, k, group, zeros, m):
    w, s, z, g = _weights(n, k, group, zeros, n + k)
    x = (torch.randn(m, k, generator=g) * 4 + 1).bfloat16()  # a mean, so that the offsets matter
    out = torch.empty(m, n, dtype=torch.bfloat16, device=DEV)
    torch.ops.cdb.gemv_w4(x.to(DEV), w.to(DEV), s.to(DEV), None if z is None else z.to(DEV), out)
    torch.cuda.synchronize()
    assert ops.status_code() == 0
    _check(out.cpu(), x, w, s, z, group)


@pytest.mark.parametrize("m", [6, 8, 9, 11, 16])
@pytest.mark.parametrize("n,k,group", [(50, 7424, 32), (50, 7936, 128), (20, 38656, 32)])
def test_token_rows_that_nearly_fill_shared_memory(n, k, group, m):
    """K where the rings that one tile of tokens would like do not fit beside its rows."""

    w, s, z, g = _weights(n, k, group, True, k + m)
    x = (torch.randn(m, k, generator=g) + 0.5).bfloat16()
    out = torch.empty(m, n, dtype=torch.bfloat16, device=DEV)
    torch.ops.cdb.gemv_w4(x.to(DEV), w.to(DEV), s.to(DEV), z.to(DEV), out)
    torch.cuda.synchronize()
    assert ops.status_code() == 0
    _check(out.cpu(), x, w, s, z, group)


def test_refuses_token_rows_that_do_not_fit():
    w, s, z, g = _weights(4, 65536, 128, False, 9)
    x = torch.zeros(1, 65536, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError, match="cdb_gemv_w4"):
        torch.ops.cdb.gemv_w4(x, w.to(DEV), s.to(DEV), None, torch.empty(1, 4, dtype=torch.bfloat16, device=DEV))


def test_strided_and_repeatable():
    """Rows of wider tensors; places between the rows stay; the same call gives the same bits."""

    w, s, z, g = _weights(300, 512, 64, True, 1)
    wide_w = torch.zeros(300, 400, dtype=torch.uint8, device=DEV)
    wide_w[:, 16:272] = w.to(DEV)
    wide_x = torch.randn(3, 1040, generator=g).bfloat16().to(DEV)
    wide_o = torch.full((3, 500), 7.0, dtype=torch.bfloat16, device=DEV)
    for rep in range(3):
        torch.ops.cdb.gemv_w4(wide_x[:, 8:520], wide_w[:, 16:272], s.to(DEV), z.to(DEV), wide_o[:, 101:401])
        first = wide_o.clone() if rep == 0 else first
        assert torch.equal(first, wide_o)
    assert (wide_o[:, :101] == 7).all() and (wide_o[:, 401:] == 7).all()
    _check(wide_o[:, 101:401].cpu(), wide_x[:, 8:520].cpu(), w, s, z, 64)


def test_infinities_and_nan_stay_in_their_rows():
    w, s, z, g = _weights(40, 256, 64, True, 2)
    x = torch.randn(3, 256, generator=g).bfloat16()
    out = torch.empty(3, 40, dtype=torch.bfloat16, device=DEV)
    args = w.to(DEV), s.to(DEV), z.to(DEV), out
    torch.ops.cdb.gemv_w4(x.to(DEV), *args)
    want = out.clone()
    x[1, 77] = float("nan")
    torch.ops.cdb.gemv_w4(x.to(DEV), *args)
    assert torch.equal(out[0], want[0]) and torch.equal(out[2], want[2]) and out[1].isnan().all()


def test_captured_and_on_another_stream():
    w, s, z, g = _weights(500, 1024, 128, False, 3)
    x = torch.randn(4, 1024, generator=g).bfloat16().to(DEV)
    w, s = w.to(DEV), s.to(DEV)
    want, out = (torch.zeros(4, 500, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    torch.ops.cdb.gemv_w4(x, w, s, None, want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    stream = torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        torch.ops.cdb.gemv_w4(x, w, s, None, out)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    x.neg_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, -want)
