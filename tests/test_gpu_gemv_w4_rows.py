"""gemv_w4 with more token rows than one pass over the weights takes (29 at K = 2048, 12 at 5632). Tolerance as in
test_gpu_gemv_w4: 2^-8 of the value and 2^-20 * 300 / 16 of max |s| sum |x|."""

from __future__ import annotations

import pytest
import torch

import continuous_depth_batching_b200.ops as ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("m", [13, 30, 32, 33, 48, 64, 80, 100, 257])
@pytest.mark.parametrize("n,k,group", [(300, 2048, 128), (300, 5632, 128), (100, 5632, 32), (100, 14336, 64)])
def test_passes(m, n, k, group):
    g = torch.Generator().manual_seed(m + k)
    w = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
    s = (torch.randn(n, k // group, generator=g) * 0.02).bfloat16()
    z = torch.randint(0, 16, (n, k // group), generator=g, dtype=torch.uint8)
    x = (torch.randn(m, k, generator=g) + 0.5).bfloat16()
    out = torch.full((m + 1, n), 7.0, dtype=torch.bfloat16, device=DEV)
    torch.ops.cdb.gemv_w4(x.to(DEV), w.to(DEV), s.to(DEV), z.to(DEV), out[:m])
    torch.cuda.synchronize()
    assert ops.status_code() == 0
    q = torch.stack((w & 15, w >> 4), -1).view(n, k).double()
    dense = (q - z.double().repeat_interleave(group, 1)) * s.double().repeat_interleave(group, 1)
    want = x.double() @ dense.t()
    size = x.double().abs().sum(1, keepdim=True) * s.double().abs().amax(1)[None, :]
    got = out.cpu()
    assert ((got[:m].double() - want).abs() <= 2.0**-8 * want.abs() + 2.0**-20 * 300 / 16 * size).all()
    assert (got[m] == 7).all()
