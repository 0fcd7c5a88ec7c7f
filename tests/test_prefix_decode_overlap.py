"""Prefix decode attention's out beside q, on the host: q's own columns and other columns of one buffer are taken, rows that
overlap q's in part are refused before anything is launched (CPU tensors that pass every check are told that there is
no CPU path)."""

from __future__ import annotations

import pytest
import torch

import continuous_depth_batching_b200.ops  # noqa: F401  (registers torch.ops.cdb.*)

COLS = 256


def _call(q, out):
    n = 3
    i32 = dict(dtype=torch.int32)
    pool = torch.zeros(1, 2, 64, 2, 64, dtype=torch.bfloat16)
    torch.ops.cdb.prefix_decode_attention(q, out, pool, 0, torch.zeros(n, 5, **i32), torch.zeros(n, **i32), torch.zeros(n, **i32), torch.zeros(2, **i32),
                                          torch.zeros(1, **i32), 4, 0.125)


def _rows(pitch, rows=3):
    return torch.zeros(rows * pitch + 4 * COLS, dtype=torch.bfloat16)


def _view(whole, at, pitch, rows=3):
    return whole[at:].as_strided((rows, COLS), (pitch, 1))


@pytest.mark.parametrize("pitch,q_at,out_at,out_pitch", [
    (256, 0, 8, 256),  # shifted by 16 bytes
    (256, 8, 0, 256),
    (256, 0, 256, 256),  # by a row
    (768, 0, 248, 768),  # the last columns
    (768, 512, 264, 768),
    (768, 0, 520, 768),  # round the corner: the next row's first columns
    (256, 0, 0, 264),  # one beginning, other rows
    (512, 0, 256, 768),
])
def test_partial_overlaps_are_refused(pitch, q_at, out_at, out_pitch):
    whole = _rows(1024)
    with pytest.raises(ValueError, match="may not overlap"):
        _call(_view(whole, q_at, pitch), _view(whole, out_at, out_pitch))


@pytest.mark.parametrize("pitch,q_at,out_at,out_pitch", [
    (256, 0, 0, 256),  # in place
    (768, 256, 256, 768),
    (512, 0, 256, 512),  # columns of one buffer
    (768, 512, 0, 768),
    (768, 0, 512, 768),
    (512, 256, 512, 512),  # the next row's first columns, q being the last
    (256, 0, 768, 256),  # behind one another
    (256, 1024, 0, 264),
])
def test_the_same_rows_and_rows_apart_are_taken(pitch, q_at, out_at, out_pitch):
    whole = _rows(1024)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        _call(_view(whole, q_at, pitch), _view(whole, out_at, out_pitch))
