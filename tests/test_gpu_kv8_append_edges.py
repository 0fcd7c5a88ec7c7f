"""Append to the 8-bit cache at the ends of its ranges."""

from __future__ import annotations

import pytest
import torch

from continuous_depth_batching_b200 import _lib

pytestmark = pytest.mark.gpu
I32 = dict(dtype=torch.int32, device="cuda")


def test_last_position_that_32_bits_hold():
    """Position 2^31 - 1 lies behind the tables of angles: reported, and nothing written."""

    d, rope_rows = 64, 4
    codes = torch.full((1, 2, 2, 1, 16, d), 1.0, device="cuda").to(torch.float8_e4m3fn)
    scales = torch.ones(1, 2, 2, 1, device="cuda")
    table = torch.zeros(1, 1 << 27, **I32)
    qkv = torch.full((1, 3 * d), 2.0, dtype=torch.bfloat16, device="cuda")
    cos = torch.ones(rope_rows, d, dtype=torch.bfloat16, device="cuda")
    q_out = torch.full((1, d), 7.0, dtype=torch.bfloat16, device="cuda")
    slot, pos, status = torch.zeros(1, **I32), torch.full((1,), 2**31 - 1, **I32), torch.zeros(1, **I32)
    p = _lib.ptr
    _lib.call("cdb_kv8_append", p(qkv), 3 * d, p(q_out), d, p(codes), p(scales), 1, 0, 2, p(table), table.stride(0), 1,
              table.shape[1], p(slot), p(pos), 1, p(cos), p(cos), rope_rows, None, 1, 1, 1, d, p(status),
              torch.cuda.current_stream().cuda_stream)
    assert int(status.item()) == 6
    assert (codes.float() == 1).all() and (scales == 1).all() and (q_out == 7).all()
