"""Blocks of the 8-bit cache to the host and back: codes and scales are two calls of cdb_kv_blocks_host_copy."""

from __future__ import annotations

import pytest
import torch

import continuous_depth_batching_b200.ops as ops
from continuous_depth_batching_b200 import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"
LAYERS, BLOCKS, HEADS, BS, D = 3, 9, 2, 16, 96


def _copy(pool, rows, row_bytes, block_size, device_blocks, host, host_blocks, to_host):
    ids = [torch.tensor(v, dtype=torch.int32) for v in (device_blocks, host_blocks)]
    _lib.call("cdb_kv_blocks_host_copy", _lib.ptr(pool), LAYERS, rows, row_bytes, block_size, BLOCKS, ids[0].data_ptr(),
              host.data_ptr(), host.shape[0], ids[1].data_ptr(), len(device_blocks), to_host,
              torch.cuda.current_stream().cuda_stream)


def _swap(codes, scales, device_blocks, host, host_blocks, to_host):
    _copy(codes, BLOCKS * BS, HEADS * D, BS, device_blocks, host[0], host_blocks, to_host)
    _copy(scales, BLOCKS, HEADS * 4, 1, device_blocks, host[1], host_blocks, to_host)


def test_round_trip_into_other_blocks():
    g = torch.Generator().manual_seed(0)
    codes = (torch.randn(LAYERS, 2, BLOCKS, HEADS, BS, D, generator=g) * 90).clamp(-448, 448).to(torch.float8_e4m3fn).to(DEV)
    scales = torch.exp2(torch.randint(-9, 9, (LAYERS, 2, BLOCKS, HEADS), generator=g).float()).to(DEV)
    host = (torch.zeros(4, 2 * LAYERS, HEADS * BS * D, dtype=torch.uint8).pin_memory(),
            torch.zeros(4, 2 * LAYERS, HEADS, dtype=torch.float32).pin_memory())

    def read(layer, blocks):
        out = torch.empty(len(blocks), 2, HEADS, BS, D, dtype=torch.bfloat16, device=DEV)
        torch.ops.cdb.kv8_gather(codes, scales, layer, torch.tensor(blocks, dtype=torch.int32, device=DEV), out)
        return out

    want = [read(layer, [7, 0, 4]) for layer in range(LAYERS)]
    others = [read(layer, [1, 3, 5]) for layer in range(LAYERS)]
    _swap(codes, scales, [7, 0, 4], host, [2, 3, 0], 1)
    torch.cuda.synchronize()
    _swap(codes, scales, [2, 8, 6], host, [2, 3, 0], 0)
    for layer in range(LAYERS):
        assert torch.equal(read(layer, [2, 8, 6]), want[layer])
        assert torch.equal(read(layer, [1, 3, 5]), others[layer])
    assert ops.status_code() == 0
