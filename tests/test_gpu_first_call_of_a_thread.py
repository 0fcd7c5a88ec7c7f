"""An operator as the first CUDA call of a host thread, which has no current context until then."""

from __future__ import annotations

import threading

import pytest
import torch

import continuous_depth_batching_b200.ops as ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32 = dict(dtype=torch.int32, device=DEV)


def _bf(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).bfloat16().to(DEV)


def _gemm():
    out = torch.zeros(16, 256, dtype=torch.bfloat16, device=DEV)
    x, w = _bf(16, 256), _bf(256, 256, seed=1)
    return lambda: torch.ops.cdb.gemm_bf16(x, w, out), out


def _gemv():
    out = torch.zeros(2, 64, dtype=torch.bfloat16, device=DEV)
    x, w, s = _bf(2, 256), torch.full((64, 128), 0x5A, dtype=torch.uint8, device=DEV), _bf(64, 2, seed=1)
    return lambda: torch.ops.cdb.gemv_w4(x, w, s, None, out), out


def _cache():
    codes = (torch.randn(1, 2, 6, 1, 16, 128, generator=torch.Generator().manual_seed(2)) * 50).to(torch.float8_e4m3fn).to(DEV)
    return codes, torch.full((1, 2, 6, 1), 2.0**-6, device=DEV), torch.arange(6, **I32).view(2, 3)


def _decode():
    q, out = _bf(2, 128), torch.zeros(2, 128, dtype=torch.bfloat16, device=DEV)
    (codes, scales, table), slot, pos = _cache(), torch.arange(2, **I32), torch.tensor([40, 17], **I32)
    return lambda: torch.ops.cdb.kv8_decode_attention(q, out, codes, scales, 0, table, slot, pos, 1, 0.1), out


def _prefill():
    q, out = _bf(20, 128), torch.zeros(20, 128, dtype=torch.bfloat16, device=DEV)
    (codes, scales, table), tiles = _cache(), torch.tensor([(0, 20, 1, 5)], **I32)
    return lambda: torch.ops.cdb.kv8_prefill_attention(q, out, codes, scales, 0, table, tiles, 1, 0.1), out


@pytest.mark.parametrize("make", [_gemm, _gemv, _decode, _prefill])
def test_first_call(make):
    make()[0]()  # workspaces and the status word are there
    call, out = make()  # tensors that no call has seen
    torch.cuda.synchronize()
    errors = []

    def work():
        try:
            call()
        except RuntimeError as e:
            errors.append(str(e))

    thread = threading.Thread(target=work)
    thread.start()
    thread.join()
    torch.cuda.synchronize()
    assert not errors, errors[0]
    assert ops.status_code() == 0
    first = out.clone()
    call()
    assert first.any() and torch.equal(first, out)
