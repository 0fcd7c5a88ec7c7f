"""What the operators that continue a prompt many times refuse, on the host (no GPU): torch.ops.cdb.* raise with a reason
before anything is launched, and the C ABI returns its code."""

from __future__ import annotations

import pytest
import torch

import continuous_depth_batching_b200.ops  # noqa: F401  (registers torch.ops.cdb.*)
from continuous_depth_batching_b200 import _lib

BF, I32, F32 = torch.bfloat16, torch.int32, torch.float32


def _b(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


def _i(*shape, dtype=I32):
    return torch.zeros(*shape, dtype=dtype)


def _norm(**over):
    a = dict(qkv=_b(3, 8 * 64), q_out=_b(3, 4 * 64), pool=_b(2, 2, 64, 2, 64), layer=1, table=_i(3, 5), slot=_i(3), pos=_i(3), q_w=_b(64), k_w=_b(64),
             cos=_b(9, 64), sin=_b(9, 64), mode=1, heads=4, eps=1e-6)
    a.update(over)
    return "qk_norm_rope_append", tuple(a.values())


def _prefix(**over):
    a = dict(q=_b(3, 256), out=_b(3, 256), pool=_b(2, 2, 64, 2, 64), layer=1, table=_i(3, 5), slot=_i(3), pos=_i(3), start=_i(3), prefix=_i(2), heads=4, scale=0.125)
    a.update(over)
    return "prefix_decode_attention", tuple(a.values())


def _sample(**over):
    a = dict(logits=_b(3, 100), u=_b(3, dtype=F32), t=_b(3, dtype=F32), k=_i(3), p=_b(3, dtype=F32), m=_b(3, dtype=F32), ids=_i(3, dtype=torch.int64),
             logp=_b(3, dtype=F32))
    a.update(over)
    return "sample_tokens", tuple(a.values())


@pytest.mark.parametrize("make", [_norm, _prefix, _sample])
def test_registered_and_cpu_refused(make):
    name, args = make()
    assert str(getattr(torch.ops.cdb, name).default._schema).startswith(f"cdb::{name}(")
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        getattr(torch.ops.cdb, name)(*args)


def test_optional_arguments_are_optional():
    for name, args in (_norm(q_out=None, cos=None, sin=None, mode=0), _prefix(start=_i(0), prefix=_i(0)), _sample(k=None, p=None, m=None, logp=None),
                       _sample(logits=_b(3, 100, dtype=F32)), _sample(logits=_b(3, 120)[:, 7:107])):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            getattr(torch.ops.cdb, name)(*args)


def _over(rows, cols, at):
    """qkv, and q_out at column `at` of it."""

    qkv = _b(rows, cols)
    return dict(qkv=qkv, q_out=qkv[:, at : at + 256])


@pytest.mark.parametrize("what,call", [
    ("kv_pool must be", _norm(pool=_b(2, 2, 64, 2, 64, dtype=F32))),
    ("kv_pool must be", _norm(pool=_b(2, 2, 64, 64))),
    ("kv_pool must be", _norm(pool=_b(2, 2, 15, 2, 64))),
    ("kv_pool must be", _norm(pool=_b(2, 2, 64, 2, 128)[..., :64])),
    ("head dims", _norm(pool=_b(2, 2, 64, 2, 80))),
    ("cache_layer", _norm(layer=2)),
    ("cache_layer", _norm(layer=-1)),
    ("qkv must be", _norm(qkv=_b(3, 8 * 64 - 8))),
    ("qkv must be", _norm(qkv=_b(2, 8 * 64))),
    ("qkv must be", _norm(qkv=_b(3, 8 * 64, dtype=F32))),
    ("qkv needs", _norm(qkv=_b(3, 8 * 64 + 3)[:, : 8 * 64])),
    ("q_out must be", _norm(q_out=_b(3, 3 * 64))),
    ("q_out needs", _norm(q_out=_b(3, 4 * 64 + 1)[:, 1:])),
    ("may not overlap", _norm(**_over(3, 8 * 64, 64))),
    ("may not overlap", _norm(**_over(3, 8 * 64, 256))),
    ("q_weight must be", _norm(q_w=_b(65))),
    ("k_weight must be", _norm(k_w=_b(64, dtype=F32))),
    ("k_weight must be", _norm(k_w=_b(65)[1:])),
    ("item_pos must be", _norm(pos=_i(3, dtype=torch.int64))),
    ("item_slot must be", _norm(slot=_i(2))),
    ("block_table must be", _norm(table=_i(3))),
    ("rope_mode must be", _norm(mode=3)),
    ("must be given", _norm(cos=None)),
    ("rope_cos and rope_sin must be", _norm(mode=2)),
    ("num_heads must be positive", _norm(heads=0)),
    ("eps must be", _norm(eps=-1.0)),
    ("eps must be", _norm(eps=float("nan"))),
    ("at most 2\\^20 heads", _norm(heads=2**20)),
    ("num_heads must be below 2", _norm(heads=2**31)),
    ("kv_pool must be", _prefix(pool=_b(2, 2, 64, 2, 64, dtype=torch.float16))),
    ("head dims", _prefix(pool=_b(2, 2, 64, 2, 32))),
    ("num_heads must be a positive multiple", _prefix(heads=3)),
    ("scale must be", _prefix(scale=0.0)),
    ("scale must be", _prefix(scale=float("nan"))),
    ("q must be", _prefix(q=_b(3, 255))),
    ("out must be", _prefix(out=_b(2, 256))),
    ("out needs", _prefix(out=_b(3, 260)[:, :256])),
    ("group_start must be", _prefix(start=_i(2))),
    ("group_start must be", _prefix(start=_i(3, dtype=torch.int64))),
    ("prefix_len must be", _prefix(prefix=_i(2, dtype=torch.int64))),
    ("item_slot must be", _prefix(slot=_i(2))),
    ("logits must be", _sample(logits=_b(3, 100, dtype=torch.float16))),
    ("logits must be", _sample(logits=_b(300))),
    ("logits must be", _sample(logits=_b(3, 0))),
    ("unit column stride", _sample(logits=_b(3, 200)[:, ::2])),
    ("unit column stride", _sample(logits=_b(1, 100).expand(3, 100))),
    ("vocabularies of up to", _sample(logits=_b(1, 2**24 + 1), u=_b(1, dtype=F32))),
    ("uniform must be", _sample(u=_b(2, dtype=F32))),
    ("uniform must be", _sample(u=_b(3, dtype=torch.float64))),
    ("temperature must be", _sample(t=_b(3))),
    ("top_k must be", _sample(k=_i(3, dtype=torch.int64))),
    ("top_p must be", _sample(p=_b(3, dtype=torch.float64))),
    ("min_p must be", _sample(m=_b(6, dtype=F32)[::2])),
    ("out_ids must be", _sample(ids=_i(3))),
    ("out_logprobs must be", _sample(logp=_b(3))),
])
def test_refused(what, call):
    with pytest.raises(ValueError, match=what):
        getattr(torch.ops.cdb, call[0])(*call[1])


def test_c_abi_refuses_without_launching():
    lib = _lib.load()
    p = 1 << 20  # never followed: these calls end on the host
    norm = lambda **o: lib.cdb_qk_norm_rope_append(*{**dict(  # noqa: E731
        qkv=p, qs=512, qo=p, qos=256, kv=p, layers=2, rows=64, layer=1, bt=p, bts=5, btr=3, btw=5, slot=p, pos=p, qw=p, kw=p, mode=1, cos=p, sin=p, rr=9, eps=1e-6, n=3,
        h=4, kvh=2, d=64, status=None, stream=None), **o}.values())
    assert norm(layer=2) == 1 and norm(rows=15) == 1 and norm(mode=3) == 1 and norm(eps=-1.0) == 1 and norm(n=-1) == 1 and norm(kvh=0) == 1
    assert norm(qkv=p + 8) == 1 and norm(qs=511) == 1 and norm(qw=p + 2) == 1 and norm(cos=None) == 1 and norm(pos=None) == 1
    assert norm(d=80) == 2 and norm(h=2**20) == 2 and norm(n=0) == 0
    att = lambda **o: lib.cdb_prefix_decode_attention(*{**dict(  # noqa: E731
        q=p, qs=256, out=p, os=256, kv=p, layers=2, rows=64, layer=1, bt=p, bts=5, btr=3, btw=5, slot=p, pos=p, n=3, start=p, prefix=p, groups=2, h=4, kvh=2, d=64,
        scale=0.125, sms=148, ws=p, floats=1 << 40, status=None, stream=None), **o}.values())
    assert att(h=5) == 1 and att(scale=0.0) == 1 and att(sms=1) == 1 and att(sms=1024) == 1 and att(layer=-1) == 1 and att(groups=-1) == 1
    assert att(ws=p + 4) == 1 and att(ws=None) == 1 and att(start=None) == 1 and att(floats=10) == 1 and att(out=p + 2) == 1
    assert att(d=72) == 2 and att(rows=2**30) == 2 and att(n=2**28) == 2 and att(n=0) == 0
    size = lib.cdb_prefix_decode_workspace_floats
    assert size(3, 2, 5, 2, 64, 148) == 0 and size(-1, 2, 4, 2, 64, 148) == 0 and 0 < size(3, 0, 4, 2, 64, 148) < size(3, 2, 4, 2, 64, 148)
    sample = lambda **o: lib.cdb_sample_tokens(*{**dict(  # noqa: E731
        logits=p, wide=0, stride=100, n=3, v=100, u=p, t=p, k=None, p=None, m=None, ids=p, logp=None, stream=None), **o}.values())
    assert sample(v=0) == 1 and sample(n=-1) == 1 and sample(u=None) == 1 and sample(ids=None) == 1 and sample(logits=p + 1) == 1 and sample(wide=1, logits=p + 2) == 1
    assert sample(v=2**24 + 1) == 2 and sample(n=0) == 0
