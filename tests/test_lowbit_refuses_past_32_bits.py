"""Numbers that do not fit the 32 bits that the low-bit operators count in are refused (on the host, no GPU), rather
than cut to another number."""

from __future__ import annotations

import pytest
import torch

from test_lowbit_refusals import BF, _append_args, _cache, _decode_args, _gemv_args, _prefill_args, _tables_args

MANY = 2**32 + 3
WRAPS = (2**60 + 2) // 3  # heads of 96: 64 columns modulo 2^64


def test_the_number_wraps_as_stated():
    assert WRAPS * 96 % 2**64 == 64 and WRAPS % 2 == 0 and WRAPS % 2**32 < 2**31


@pytest.mark.parametrize("op,args", [
    ("kv8_append", _append_args(heads=2**58 + 4)),
    ("kv8_append", _append_args(table=torch.empty(0, MANY, dtype=torch.int32))),
    ("kv8_append", _append_args(table=torch.empty(MANY, 0, dtype=torch.int32))),
    ("kv8_decode_attention", _decode_args(heads=2**58 + 4)),
    ("kv8_decode_attention", _decode_args(heads=WRAPS, **dict(zip(("codes", "scales"), _cache(dim=96))))),
    ("kv8_decode_attention", _decode_args(table=torch.empty(MANY, 0, dtype=torch.int32))),
    ("kv8_prefill_attention", _prefill_args(heads=2**58 + 4)),
    ("kv8_prefill_attention", _prefill_args(table=torch.empty(0, MANY, dtype=torch.int32))),
    ("step_tables", _tables_args(table=torch.empty(MANY, 0, dtype=torch.int32))),
])
def test_refused(op, args):
    with pytest.raises(ValueError, match=r"must be below 2\^31"):
        getattr(torch.ops.cdb, op)(*args)


def test_gemv_refuses_more_rows_than_it_takes():
    x = torch.empty(65536, 256, dtype=BF)
    with pytest.raises(ValueError, match="65535 token rows"):
        torch.ops.cdb.gemv_w4(*_gemv_args(x=x, out=torch.empty(65536, 5, dtype=BF)))
