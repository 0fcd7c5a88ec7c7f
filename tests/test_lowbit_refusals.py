"""What the low-bit decode step's entry points refuse, on the host (no GPU): torch.ops.cdb.* raise with a
reason before anything is launched, and the C ABI returns its code."""

from __future__ import annotations

import pytest
import torch

import continuous_depth_batching_b200.ops  # noqa: F401  (registers torch.ops.cdb.*)
from continuous_depth_batching_b200 import _lib

OPS = ["step_tables", "kv8_append", "kv8_gather", "kv8_decode_attention", "kv8_prefill_attention", "gemv_w4"]
BF, F8, I32 = torch.bfloat16, torch.float8_e4m3fn, torch.int32


def _cache(layers=1, blocks=4, heads=2, dim=64, bs=16):
    return torch.zeros(layers, 2, blocks, heads, bs, dim, dtype=F8), torch.zeros(layers, 2, blocks, heads)


def _ints(*shape, dtype=I32):
    return torch.zeros(*shape, dtype=dtype)


def _append_args(**over):
    codes, scales = _cache()
    a = dict(qkv=torch.zeros(3, 8 * 64, dtype=BF), q_out=torch.zeros(3, 4 * 64, dtype=BF), codes=codes, scales=scales,
             layer=0, table=_ints(3, 5), slot=_ints(3), pos=_ints(3), cos=torch.zeros(9, 64, dtype=BF),
             sin=torch.zeros(9, 64, dtype=BF), bias=None, mode=1, heads=4)
    a.update(over)
    return tuple(a.values())


def _decode_args(**over):
    codes, scales = _cache()
    a = dict(q=torch.zeros(3, 256, dtype=BF), out=torch.zeros(3, 256, dtype=BF), codes=codes, scales=scales, layer=0,
             table=_ints(3, 5), slot=_ints(3), pos=_ints(3), heads=4, scale=0.125)
    a.update(over)
    return tuple(a.values())


def _prefill_args(**over):
    codes, scales = _cache()
    a = dict(q=torch.zeros(3, 256, dtype=BF), out=torch.zeros(3, 256, dtype=BF), codes=codes, scales=scales, layer=0,
             table=_ints(3, 5), tiles=_ints(2, 4), heads=4, scale=0.125)
    a.update(over)
    return tuple(a.values())


def _gemv_args(**over):
    a = dict(x=torch.zeros(2, 256, dtype=BF), w=torch.zeros(5, 128, dtype=torch.uint8), scales=torch.zeros(5, 4, dtype=BF),
             zeros=None, out=torch.zeros(2, 5, dtype=BF))
    a.update(over)
    return tuple(a.values())


def _tables_args(**over):
    a = dict(slots=_ints(2), seq_len=_ints(6), new_len=_ints(2), row_len=_ints(6), table=_ints(6, 8), ring=_ints(20),
             state=_ints(4), row_len_out=_ints(6), state_out=_ints(4), granted=_ints(2), cu_q=_ints(3), cu_k=_ints(3),
             slot=_ints(10), pos=_ints(10), map=_ints(10, dtype=torch.int64), tiles=_ints(3, 4))
    a.update(over)
    return tuple(a.values())


@pytest.mark.parametrize("name", OPS)
def test_registered_and_cpu_refused(name):
    assert str(getattr(torch.ops.cdb, name).default._schema).startswith(f"cdb::{name}(")
    args = {"step_tables": _tables_args, "kv8_append": _append_args, "kv8_decode_attention": _decode_args,
            "kv8_prefill_attention": _prefill_args, "gemv_w4": _gemv_args}.get(name)
    codes, scales = _cache()
    args = args() if args else (codes, scales, 0, _ints(1), torch.zeros(1, 2, 2, 16, 64, dtype=BF))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        getattr(torch.ops.cdb, name)(*args)


def _odd(rows, cols, pitch):
    return torch.zeros(rows, pitch, dtype=BF)[:, :cols]


@pytest.mark.parametrize("what,args", [
    ("codes must be", _append_args(codes=_cache(bs=32)[0])),
    ("codes must be", _append_args(codes=_cache()[0].view(torch.uint8))),
    ("scales must be", _append_args(scales=torch.zeros(1, 2, 4, 3))),
    ("head dims 64, 96 and 128", _append_args(codes=_cache(dim=32)[0])),
    ("cache_layer", _append_args(layer=1)),
    ("cache_layer", _append_args(layer=-1)),
    ("num_heads must be positive", _append_args(heads=0)),
    ("qkv must be", _append_args(heads=5)),
    ("qkv must be", _append_args(qkv=torch.zeros(2, 512, dtype=BF))),
    ("qkv must be", _append_args(qkv=torch.zeros(3, 512))),
    ("multiple of 8", _append_args(qkv=_odd(3, 512, 516))),
    ("multiple of 8", _append_args(q_out=torch.zeros(3, 260, dtype=BF)[:, 4:])),
    ("item_slot must be", _append_args(slot=_ints(2))),
    ("item_pos must be", _append_args(pos=_ints(3, dtype=torch.int64))),
    ("block_table must be", _append_args(table=_ints(5, 3).t())),
    ("rope_mode must be", _append_args(mode=3)),
    ("rope_cos and rope_sin must be given", _append_args(sin=None)),
    ("rope_cos and rope_sin must be contiguous", _append_args(mode=2)),
    ("qk_bias must be", _append_args(bias=torch.zeros(4, 64, dtype=BF))),
])
def test_append_refuses(what, args):
    with pytest.raises(ValueError, match=what):
        torch.ops.cdb.kv8_append(*args)


@pytest.mark.parametrize("what,args", [
    ("multiple of the cache's 2 kv heads", _decode_args(heads=3)),
    ("multiple of the cache's 2 kv heads", _decode_args(heads=0)),
    ("q must be", _decode_args(heads=6)),
    ("out must be", _decode_args(out=torch.zeros(2, 256, dtype=BF))),
    ("item_pos must be", _decode_args(pos=_ints(6)[::2])),
    ("scale must be positive", _decode_args(scale=0.0)),
    ("scale must be positive", _decode_args(scale=float("nan"))),
    ("scales must be", _decode_args(scales=torch.zeros(1, 2, 4, 2, dtype=torch.float64))),
])
def test_decode_refuses(what, args):
    with pytest.raises(ValueError, match=what):
        torch.ops.cdb.kv8_decode_attention(*args)


@pytest.mark.parametrize("what,args", [
    ("tiles must be", _prefill_args(tiles=_ints(2, 3))),
    ("tiles must be", _prefill_args(tiles=_ints(2, 4, dtype=torch.int64))),
    ("scale must be positive", _prefill_args(scale=-0.125)),
    ("65535 tiles", _prefill_args(tiles=_ints(65536, 4))),
    ("out must be", _prefill_args(out=torch.zeros(2, 256, dtype=BF))),
    ("multiple of the cache's 2 kv heads", _prefill_args(heads=5)),
])
def test_prefill_refuses(what, args):
    with pytest.raises(ValueError, match=what):
        torch.ops.cdb.kv8_prefill_attention(*args)


def test_gather_refuses():
    codes, scales = _cache()
    with pytest.raises(ValueError, match="out must be"):
        torch.ops.cdb.kv8_gather(codes, scales, 0, _ints(2), torch.zeros(1, 2, 2, 16, 64, dtype=BF))
    with pytest.raises(ValueError, match="blocks must be"):
        torch.ops.cdb.kv8_gather(codes, scales, 0, _ints(1, dtype=torch.int64), torch.zeros(1, 2, 2, 16, 64, dtype=BF))


@pytest.mark.parametrize("what,args", [
    ("w must be", _gemv_args(w=torch.zeros(5, 128, dtype=torch.int8))),
    ("K a multiple of 32", _gemv_args(w=torch.zeros(5, 136, dtype=torch.uint8))),
    ("row stride", _gemv_args(w=torch.zeros(5, 136, dtype=torch.uint8)[:, :128])),
    ("16-byte alignment", _gemv_args(w=torch.zeros(5, 144, dtype=torch.uint8)[:, 8:136])),
    ("scales must be", _gemv_args(scales=torch.zeros(4, 4, dtype=BF))),
    ("scales must be", _gemv_args(scales=torch.zeros(5, 3, dtype=BF))),
    ("scales must be", _gemv_args(scales=torch.zeros(5, 4))),
    ("groups of 32, 64", _gemv_args(scales=torch.zeros(5, 16, dtype=BF))),
    ("zeros must be", _gemv_args(zeros=torch.zeros(5, 4))),
    ("columns, the weights", _gemv_args(x=torch.zeros(2, 264, dtype=BF))),
    ("x must be", _gemv_args(x=torch.zeros(2, 128, dtype=BF))),
    ("out must be", _gemv_args(out=torch.zeros(2, 6, dtype=BF))),
])
def test_gemv_refuses(what, args):
    with pytest.raises(ValueError, match=what):
        torch.ops.cdb.gemv_w4(*args)


@pytest.mark.parametrize("what,args", [
    ("new_len must be", _tables_args(new_len=_ints(1))),
    ("cu_seq_lens_q must be", _tables_args(cu_q=_ints(2))),
    ("seq_len must be", _tables_args(seq_len=_ints(5))),
    ("block_table needs a row", _tables_args(table=_ints(5, 8))),
    ("slot_map must be", _tables_args(map=_ints(10))),
    ("item_slot must be", _tables_args(slot=_ints(9))),
    ("state must be", _tables_args(state=_ints(3))),
    ("tiles must be", _tables_args(tiles=_ints(3, 3))),
    ("8192 requests", _tables_args(slots=_ints(8193), new_len=_ints(8193), granted=_ints(8193), cu_q=_ints(8194), cu_k=_ints(8194))),
])
def test_tables_refuse(what, args):
    with pytest.raises(ValueError, match=what):
        torch.ops.cdb.step_tables(*args)


def test_c_abi_refuses_on_the_host():
    lib = _lib.load()
    some = 1 << 20  # a 16-byte aligned address that no call gets to use
    inval, unsupported = 1, 2
    append = lambda layers=1, layer=0, mode=0, heads=2, kv=2, dim=64, qkv=some, stride=512, n=1: lib.cdb_kv8_append(  # noqa: E731
        qkv, stride, None, 0, some, some, layers, layer, 4, some, 5, 3, 5, some, some, mode, None, None, 0, None, n, heads,
        kv, dim, None, None)
    assert append(layer=1) == inval and append(mode=1) == inval and append(mode=5) == inval
    assert append(qkv=some + 2) == inval and append(stride=513) == inval and append(n=-1) == inval
    assert append(dim=80) == unsupported and append(n=0) == 0
    decode = lambda heads=4, dim=64, ws=1 << 30, n=1, q=some: lib.cdb_kv8_decode_attention(  # noqa: E731
        q, 256, some, 256, some, some, 1, 0, 4, some, 5, 3, 5, some, some, n, heads, 2, dim, 0.1, 296, some, ws, some, None, None)
    assert decode(heads=3) == inval and decode(ws=100) == inval and decode(q=some + 8) == inval
    assert decode(dim=256) == unsupported and decode(n=0) == 0
    prefill = lambda tiles=1, dim=64: lib.cdb_kv8_prefill_attention(  # noqa: E731
        some, 256, some, 256, 8, some, some, 1, 0, 4, some, 5, 3, 5, some, tiles, 4, 2, dim, 0.1, None, None)
    assert prefill(tiles=70000) == inval and prefill(dim=32) == unsupported and prefill(tiles=0) == 0
    gemv = lambda k=256, group=64, ldw=128, m=1: lib.cdb_gemv_w4(  # noqa: E731
        some, 256, some, ldw, some, None, some, 64, m, 64, k, group, 148, None, None)
    assert gemv(k=240) == inval and gemv(group=96) == inval and gemv(ldw=120) == inval and gemv(m=0) == 0
    assert lib.cdb_kv8_gather(some, some, 1, 0, 4, 2, 64, some, -1, some, None, None) == inval
    assert lib.cdb_step_tables(some, some, some, some, 9000, some, 5, 3, 5, some, 9, some, some, some, some, some, some,
                               some, some, some, 1, None, 0, None, None) == unsupported
    assert lib.cdb_step_tables(some, some, some, some, 1, some, 5, 3, 5, None, 9, some, some, some, some, some, some,
                               some, some, some, 1, None, 0, None, None) == inval
    assert lib.cdb_kv8_decode_workspace_floats(148, 128) >= 148 * 2 * 8 * 130
