"""``torch.ops.cdb.*``: the library's hot-path entry points as PyTorch custom operators.

A model adapter written against PyTorch (the reference's ``CDBModelAdapter`` seam,
``model_adapter.py:14-102``) can call these instead of ``ctypes``: they take tensors, run on the
current CUDA stream, and raise on CPU tensors (there is no CPU path). Persistent scratch (the
shared status word, the attention plan, the GEMM split workspace) is allocated on an op's first
call on a device, and that call raises instead if the stream is being captured; returned tensors
come from PyTorch's caching allocator. Each wraps one ``include/cdb_b200.h`` entry point:

* ``cdb::gemm_bf16(x, w, out)``: ``out = x @ w.T`` (``cdb_gemm_bf16``);
* ``cdb::mlp_gateup_silu(x, w_gate_up, act)``: SwiGLU of interleaved gate/up rows
  (``cdb_mlp_gateup_silu_gemm``);
* ``cdb::lm_head_argmax(x, w) -> ids``: greedy next tokens without logits (``cdb_lm_head_argmax``);
* ``cdb::add_rmsnorm(x, a, w_a, w_next, y)``: ``x += norm_a(a)``, ``y = norm_next(x)``
  (``cdb_add_rmsnorm``);
* ``cdb::paged_decode_attention(...)``: RoPE, KV append and paged decode attention in one
  launch (``cdb_attn_plan`` + ``cdb_paged_decode_attn_append``). Its work plan and split-combine
  scratch are allocated once per device, on the first call; that first call allocates and so must
  not run while a stream is being captured (the op raises if it does); later calls allocate
  nothing. The scratch is shared by the op's calls on one device, so those calls must be ordered
  (one stream);
* ``cdb::exit_gate_route(...)``: exit decision, routing and compaction of one recurrent launch
  (``cdb_exit_gate_route``).
"""

from __future__ import annotations

import torch

from . import _lib

__all__ = ["gemm_bf16", "mlp_gateup_silu", "lm_head_argmax", "add_rmsnorm", "paged_decode_attention", "exit_gate_route"]


def _cuda(*tensors: torch.Tensor | None) -> None:
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise RuntimeError("torch.ops.cdb kernels run on CUDA tensors only (sm_100a); there is no CPU path")


def _stream(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def _sms(t: torch.Tensor) -> int:
    return torch.cuda.get_device_properties(t.device).multi_processor_count


_STATUS: dict[int, torch.Tensor] = {}
_LM_SCRATCH: dict[int, tuple[torch.Tensor, torch.Tensor]] = {}


def _capturing(t: torch.Tensor) -> bool:
    return torch.cuda.is_current_stream_capturing()


def _status(t: torch.Tensor) -> torch.Tensor:
    idx = t.device.index
    if idx not in _STATUS:
        if _capturing(t):
            raise RuntimeError(
                "torch.ops.cdb: the first call on a device allocates the shared status word; make one call "
                "before capturing a CUDA graph"
            )
        _STATUS[idx] = torch.zeros(1, dtype=torch.int32, device=t.device)
    return _STATUS[idx]


# Decode-attention work plan and split-combine scratch, per device: rows x heads the split
# scratch covers, and the plan's unit capacity, grown (outside capture) when a call needs more.
_ATTN_SCRATCH_ROWHEADS = 4096
_ATTN: dict[int, dict[str, torch.Tensor | int]] = {}


def _attn_scratch(t: torch.Tensor, n_items: int, num_heads: int, head_dim: int) -> dict:
    idx = t.device.index
    hg = 5 if head_dim == 96 else 4
    scratch_items = max(1, _ATTN_SCRATCH_ROWHEADS // num_heads)
    cap = max(scratch_items * (num_heads // hg) * 64, n_items * (num_heads // hg)) + _lib.ATTN_PLAN_MAX_CHUNKS
    cur = _ATTN.get(idx)
    if cur is None or cur["cap"] < cap or cur["head_dim"] < head_dim or cur["scratch_items"] != scratch_items:
        if _capturing(t):
            raise RuntimeError(
                "torch.ops.cdb.paged_decode_attention: the scratch for this shape is not allocated yet; make one "
                "call with the largest batch before capturing a CUDA graph"
            )
        dev = t.device
        cur = {
            "cap": cap,
            "head_dim": head_dim,
            "scratch_items": scratch_items,
            "hdr": torch.zeros(_lib.ATTN_PLAN_HEADER_INTS, dtype=torch.int32, device=dev),
            "units": torch.zeros(cap, 4, dtype=torch.int32, device=dev),
            "part_o": torch.zeros(scratch_items * num_heads * 64 * head_dim, dtype=torch.float32, device=dev),
            "part_ml": torch.zeros(scratch_items * num_heads * 64 * 2, dtype=torch.float32, device=dev),
            "counters": torch.zeros(scratch_items * num_heads, dtype=torch.int32, device=dev),
        }
        _ATTN[idx] = cur
    return cur


# Stream-K GEMM split workspace and tile counters, per device, grown (outside capture) on demand.
_GEMM: dict[int, tuple[int, int, _lib.GemmWorkspace]] = {}


def _gemm_ws(t: torch.Tensor, m: int, n: int) -> tuple:
    idx = t.device.index
    cur = _GEMM.get(idx)
    if cur is None or cur[0] < m or cur[1] < n:
        if _capturing(t):
            raise RuntimeError(
                "torch.ops.cdb: the GEMM workspace for this shape is not allocated yet; make one call with the "
                "largest shape before capturing a CUDA graph"
            )
        m2, n2 = max(m, 256, cur[0] if cur else 0), max(n, 65536, cur[1] if cur else 0)
        cur = (m2, n2, _lib.GemmWorkspace(t.device, m2, n2, _sms(t)))
        _GEMM[idx] = cur
    return cur[2].args()


def _check_index(name: str, t: torch.Tensor | None) -> None:
    if t is not None and (t.dtype != torch.int32 or not t.is_contiguous()):
        raise ValueError(f"{name} must be a contiguous int32 tensor, got {t.dtype} (contiguous={t.is_contiguous()})")


def _check_rows(name: str, t: torch.Tensor) -> None:
    if t.dtype != torch.bfloat16 or t.dim() != 2 or t.stride(1) != 1:
        raise ValueError(f"{name} must be a 2-D bf16 tensor with unit column stride, got {t.dtype} {tuple(t.shape)}")


def status_code(device: torch.device | str | int | None = None) -> int:
    """The device-side status word the ops share on ``device`` (0 = ok); reading it synchronises."""

    dev = torch.device("cuda") if device is None else torch.device(device)
    idx = dev.index if dev.index is not None else torch.cuda.current_device()
    s = _STATUS.get(idx)
    return 0 if s is None else int(s.item())


@torch.library.custom_op("cdb::gemm_bf16", mutates_args=("out",))
def gemm_bf16(x: torch.Tensor, w: torch.Tensor, out: torch.Tensor) -> None:
    """``out[M, N] = x[M, K] @ w[N, K].T`` in bf16 with fp32 accumulation (tcgen05)."""

    _cuda(x, w, out)
    m, k = x.shape
    status = _status(x)
    ws = _gemm_ws(x, m, w.shape[0])
    _lib.call(
        "cdb_gemm_bf16", _lib.ptr(x), x.stride(0), _lib.ptr(w), w.stride(0), _lib.ptr(out), out.stride(0), m,
        w.shape[0], k, 0, *ws, _sms(x), _lib.ptr(status), _stream(x),
    )


@torch.library.custom_op("cdb::mlp_gateup_silu", mutates_args=("act",))
def mlp_gateup_silu(x: torch.Tensor, w_gate_up: torch.Tensor, act: torch.Tensor) -> None:
    """``act = silu(x @ Wg.T) * (x @ Wu.T)`` with ``w_gate_up`` rows interleaved (gate j, up j)."""

    _cuda(x, w_gate_up, act)
    m, k = x.shape
    status = _status(x)
    ws = _gemm_ws(x, m, w_gate_up.shape[0])
    _lib.call(
        "cdb_mlp_gateup_silu_gemm", _lib.ptr(x), x.stride(0), _lib.ptr(w_gate_up), w_gate_up.stride(0),
        _lib.ptr(act), act.stride(0), m, w_gate_up.shape[0] // 2, k, 0, *ws, _sms(x), _lib.ptr(status), _stream(x),
    )


@torch.library.custom_op("cdb::lm_head_argmax", mutates_args=())
def lm_head_argmax(x: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    """Greedy next token of every row of ``x`` under the LM head ``w [vocab, K]`` (int64 [M])."""

    _cuda(x, w)
    m, k = x.shape
    idx = x.device.index
    if idx not in _LM_SCRATCH or _LM_SCRATCH[idx][0].numel() < m:
        if _capturing(x):
            raise RuntimeError("torch.ops.cdb.lm_head_argmax: make one call with the largest batch before capture")
        _LM_SCRATCH[idx] = (
            torch.zeros(max(m, 256), dtype=torch.int64, device=x.device),
            torch.zeros(1, dtype=torch.int32, device=x.device),
        )
    keys, done = _LM_SCRATCH[idx]
    status = _status(x)
    ws = _gemm_ws(x, m, w.shape[0])
    ids = torch.empty(m, dtype=torch.int64, device=x.device)
    _lib.call(
        "cdb_lm_head_argmax", _lib.ptr(x), x.stride(0), _lib.ptr(w), w.stride(0), m, w.shape[0], k, _lib.ptr(ids),
        None, None, None, _lib.ptr(keys), _lib.ptr(done), *ws, _sms(x), _lib.ptr(status), _stream(x),
    )
    return ids


@lm_head_argmax.register_fake
def _(x, w):
    return x.new_empty(x.shape[0], dtype=torch.int64)


@torch.library.custom_op("cdb::add_rmsnorm", mutates_args=("x", "y"))
def add_rmsnorm(x: torch.Tensor, a: torch.Tensor, w_a: torch.Tensor, w_next: torch.Tensor, y: torch.Tensor,
                eps: float) -> None:
    """Ouro's sandwich step: ``x = bf16(x + norm_a(a))``, ``y = norm_next(x)`` (bf16 rounding as
    OuroRMSNorm rounds)."""

    _cuda(x, a, w_a, w_next, y)
    _lib.call(
        "cdb_add_rmsnorm", _lib.ptr(x), x.stride(0), _lib.ptr(a), a.stride(0), _lib.ptr(w_a), _lib.ptr(w_next),
        _lib.ptr(y), y.stride(0), None, None, None, None, x.shape[0], x.shape[1], eps, _stream(x),
    )


@torch.library.custom_op("cdb::paged_decode_attention", mutates_args=("out", "kv_pool"))
def paged_decode_attention(
    qkv: torch.Tensor, out: torch.Tensor, kv_pool: torch.Tensor, cache_layer: int, block_table: torch.Tensor,
    item_slot: torch.Tensor, item_pos: torch.Tensor, rope_cos: torch.Tensor | None, rope_sin: torch.Tensor | None,
    qk_bias: torch.Tensor | None, rope_mode: int, num_heads: int, head_dim: int, scale: float,
) -> None:
    """Decode attention of rows at ``item_pos`` over the paged pool ``kv_pool [layers, 2, rows, H, D]``
    with RoPE and the KV append fused (``qkv`` rows hold q | k | v; q is not modified)."""

    _cuda(qkv, out, kv_pool, block_table, item_slot, item_pos, rope_cos, rope_sin, qk_bias)
    if kv_pool.dtype != torch.bfloat16 or kv_pool.dim() != 5 or not kv_pool.is_contiguous():
        raise ValueError("kv_pool must be a contiguous bf16 tensor [layers, 2, rows, heads, head_dim]")
    if kv_pool.shape[1] != 2 or kv_pool.shape[3] != num_heads or kv_pool.shape[4] != head_dim:
        raise ValueError(f"kv_pool shape {tuple(kv_pool.shape)} does not match {num_heads} heads of {head_dim}")
    _check_rows("qkv", qkv)
    _check_rows("out", out)
    for name, t in (("item_slot", item_slot), ("item_pos", item_pos)):
        _check_index(name, t)
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.stride(1) != 1:
        raise ValueError("block_table must be a 2-D int32 tensor with unit column stride")
    n = item_pos.numel()
    if item_slot.numel() < n or qkv.shape[0] < n or out.shape[0] < n:
        raise ValueError("item_slot, qkv and out need a row per item_pos entry")
    hd = num_heads * head_dim
    if qkv.shape[1] < 3 * hd or out.shape[1] < hd:
        raise ValueError("qkv rows must hold q | k | v and out rows num_heads * head_dim values")
    status = _status(qkv)
    sc = _attn_scratch(qkv, n, num_heads, head_dim)
    stream = _stream(qkv)
    _lib.call(
        "cdb_attn_plan", _lib.ptr(item_pos), n, 2, num_heads, head_dim, 16, sc["cap"], sc["scratch_items"],
        _sms(qkv), _lib.ptr(sc["hdr"]), _lib.ptr(sc["units"]), stream,
    )
    _lib.call(
        "cdb_paged_decode_attn_append", _lib.ptr(qkv), qkv.stride(0), hd, 2 * hd, _lib.ptr(out), out.stride(0),
        _lib.ptr(kv_pool), kv_pool.shape[0], kv_pool.shape[2], cache_layer, _lib.ptr(block_table),
        block_table.stride(0), _lib.ptr(item_slot), _lib.ptr(item_pos), rope_mode, _lib.ptr(rope_cos),
        _lib.ptr(rope_sin), _lib.ptr(qk_bias), 2, _lib.ptr(sc["hdr"]), _lib.ptr(sc["units"]),
        _lib.ptr(sc["part_o"]), _lib.ptr(sc["part_ml"]), _lib.ptr(sc["counters"]), sc["scratch_items"], n,
        num_heads, head_dim, 16, scale, 2 * _sms(qkv), _lib.ptr(status), stream,
    )


@torch.library.custom_op("cdb::exit_gate_route", mutates_args=("cdf", "surv", "pending"))
def exit_gate_route(
    signal: torch.Tensor, hidden: torch.Tensor, step: torch.Tensor, depth: torch.Tensor | None,
    reset: torch.Tensor | None, cdf: torch.Tensor, surv: torch.Tensor, pending: torch.Tensor | None, policy: int,
    delayed: bool, min_steps: int, max_steps: int, threshold: float,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Exit flags, survivor rows, exit rows and ``{num_survivors, num_exits}`` of one launch."""

    _cuda(signal, hidden, step, depth, reset, cdf, surv, pending)
    n = hidden.numel()
    flags = torch.empty(n, dtype=torch.int8, device=hidden.device)
    surv_rows = torch.empty(n, dtype=torch.int32, device=hidden.device)
    exit_rows = torch.empty(n, dtype=torch.int32, device=hidden.device)
    counts = torch.empty(2, dtype=torch.int32, device=hidden.device)
    _lib.call(
        "cdb_exit_gate_route", _lib.ptr(signal), signal.stride(0) if signal.dim() else 1, _lib.ptr(hidden),
        _lib.ptr(step), _lib.ptr(depth), _lib.ptr(reset), _lib.ptr(cdf), _lib.ptr(surv), _lib.ptr(pending), n, policy,
        int(delayed), min_steps, max_steps, threshold, _lib.ptr(flags), _lib.ptr(surv_rows), _lib.ptr(exit_rows),
        _lib.ptr(counts), _stream(hidden),
    )
    return flags, surv_rows, exit_rows, counts


@exit_gate_route.register_fake
def _(signal, hidden, step, depth, reset, cdf, surv, pending, policy, delayed, min_steps, max_steps, threshold):
    n = hidden.numel()
    i32 = torch.int32
    return hidden.new_empty(n, dtype=torch.int8), hidden.new_empty(n, dtype=i32), hidden.new_empty(n, dtype=i32), \
        hidden.new_empty(2, dtype=i32)


# ---------------------------------------------------------------- low-bit decode step
# Defined on a Library rather than with custom_op: a decode step makes hundreds of these calls, and a
# call costs 3 us of host time here against 15 us through custom_op's wrapper.
_LIBRARY = torch.library.Library("cdb", "FRAGMENT")

KV8_BLOCK = 16  # tokens of one block of the 8-bit cache
_SM_COUNT: dict[int, int] = {}
_KV8_WS: dict[tuple[int, int], tuple[torch.Tensor, torch.Tensor]] = {}


def _define(schema: str):
    """Register the decorated function as ``cdb::<schema>``, under its Python signature. The ops write
    into tensors that they are given, so tracing needs no shapes from them."""

    name = schema[: schema.index("(")]

    def register(fn):
        _LIBRARY.define(schema)
        _LIBRARY.impl(name, fn, "CompositeExplicitAutograd")
        torch.library.register_fake(f"cdb::{name}", lambda *args, **kwargs: None, lib=_LIBRARY)
        __all__.append(name)
        return fn

    return register


def _one_device(*tensors: torch.Tensor | None) -> torch.device:
    """The CUDA device that all the tensors share; raises otherwise."""

    dev = None
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError("torch.ops.cdb kernels run on CUDA tensors only (sm_100a); there is no CPU path")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError(f"all tensors must be on one device, got {dev} and {t.device}")
    return dev


def _launch(dev: torch.device, name: str, *args) -> None:
    """Call an entry point on ``dev``'s current stream, with ``dev`` current for the launch."""

    stream = torch.cuda.current_stream(dev).cuda_stream
    if torch.cuda.current_device() == dev.index:
        _lib.call(name, *args, stream)
    else:
        with torch.cuda.device(dev):
            _lib.call(name, *args, stream)


def _sm_count(dev: torch.device) -> int:
    n = _SM_COUNT.get(dev.index)
    if n is None:
        n = _SM_COUNT[dev.index] = torch.cuda.get_device_properties(dev).multi_processor_count
    return n


def _dtype(name: str, t: torch.Tensor, dtype: torch.dtype, dim: int) -> None:
    if t.dtype != dtype or t.dim() != dim:
        raise ValueError(f"{name} must be a {dim}-D {dtype} tensor, got {t.dtype} {tuple(t.shape)}")


def _rows_of(name: str, t: torch.Tensor, rows: int, cols: int) -> None:
    """A 2-D bf16 tensor of at least that size whose rows the kernels may read 16 bytes at a time."""

    if t.dtype != torch.bfloat16 or t.dim() != 2 or t.shape[0] < rows or t.shape[1] < cols:
        raise ValueError(f"{name} must be a 2-D bf16 tensor of at least {rows} x {cols}, got {t.dtype} {tuple(t.shape)}")
    if t.stride(1) != 1 or (t.shape[0] > 1 and t.stride(0) < cols) or t.stride(0) % 8 or t.data_ptr() % 16:
        raise ValueError(f"{name} needs unit column stride, a row stride that is a multiple of 8 and 16-byte alignment")


def _int_row(name: str, t: torch.Tensor, n: int, dtype: torch.dtype = torch.int32) -> None:
    if t.dtype != dtype or t.dim() != 1 or t.shape[0] < n or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous 1-D {dtype} tensor of at least {n} entries, got {t.dtype} {tuple(t.shape)}")


def _table_of(name: str, t: torch.Tensor) -> None:
    if t.dtype != torch.int32 or t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        raise ValueError(f"{name} must be a 2-D int32 tensor with unit column stride, got {t.dtype} {tuple(t.shape)}")


def _kv8_cache(codes: torch.Tensor, scales: torch.Tensor, cache_layer: int) -> tuple[int, int, int, int]:
    """(layers, blocks, kv heads, head dim) of an 8-bit cache, checked."""

    if codes.dtype != torch.float8_e4m3fn or codes.dim() != 6 or not codes.is_contiguous() or codes.shape[1] != 2 or codes.shape[4] != KV8_BLOCK:
        raise ValueError(f"codes must be a contiguous float8_e4m3fn tensor [layers, 2, blocks, kv heads, {KV8_BLOCK}, head dim], got {codes.dtype} {tuple(codes.shape)}")
    if scales.dtype != torch.float32 or scales.shape != codes.shape[:4] or not scales.is_contiguous():
        raise ValueError(f"scales must be a contiguous fp32 tensor {tuple(codes.shape[:4])}, got {scales.dtype} {tuple(scales.shape)}")
    layers, _, blocks, heads, _, dim = codes.shape
    if dim not in (64, 96, 128):
        raise ValueError(f"the 8-bit cache takes head dims 64, 96 and 128, got {dim}")
    if not 0 <= cache_layer < layers:
        raise ValueError(f"cache_layer must be in [0, {layers}), got {cache_layer}")
    if codes.data_ptr() % 16:
        raise ValueError("codes must be 16-byte aligned")
    return layers, blocks, heads, dim


@_define(
    "kv8_append(Tensor qkv, Tensor(a!)? q_out, Tensor(b!) codes, Tensor(c!) scales, int cache_layer, Tensor block_table, "
    "Tensor item_slot, Tensor item_pos, Tensor? rope_cos, Tensor? rope_sin, Tensor? qk_bias, int rope_mode, int num_heads) -> ()"
)
def kv8_append(qkv, q_out, codes, scales, cache_layer, block_table, item_slot, item_pos, rope_cos, rope_sin, qk_bias,
               rope_mode, num_heads):
    """Rotate the rows' queries and keys and write keys and values into the 8-bit cache
    (``cdb_kv8_append``). ``qkv`` rows hold q | k | v; the rotated q goes to ``q_out`` (which may be
    q's columns of ``qkv``; None leaves q alone). Rows of one request are consecutive, at ascending
    positions; a row at a negative position is skipped."""

    dev = _one_device(qkv, q_out, codes, scales, block_table, item_slot, item_pos, rope_cos, rope_sin, qk_bias)
    layers, blocks, kv_heads, dim = _kv8_cache(codes, scales, cache_layer)
    n = item_pos.numel()
    if num_heads <= 0:
        raise ValueError(f"num_heads must be positive, got {num_heads}")
    _rows_of("qkv", qkv, n, (num_heads + 2 * kv_heads) * dim)
    if q_out is not None:
        _rows_of("q_out", q_out, n, num_heads * dim)
    _int_row("item_pos", item_pos, n)
    _int_row("item_slot", item_slot, n)
    _table_of("block_table", block_table)
    if rope_mode not in (0, 1, 2):
        raise ValueError(f"rope_mode must be 0 (none), 1 (split halves) or 2 (interleaved pairs), got {rope_mode}")
    rope_rows = 0
    if rope_mode:
        if rope_cos is None or rope_sin is None or rope_cos.shape != rope_sin.shape:
            raise ValueError("rope_cos and rope_sin must be given, with one shape, when rope_mode is not 0")
        want, cols = (torch.bfloat16, dim) if rope_mode == 1 else (torch.float32, dim // 2)
        for name, t in (("rope_cos", rope_cos), ("rope_sin", rope_sin)):
            if t.dtype != want or t.dim() != 2 or t.shape[1] != cols or not t.is_contiguous() or t.data_ptr() % 16:
                raise ValueError(f"{name} must be a contiguous 16-byte aligned {want} tensor [positions, {cols}] in rope_mode {rope_mode}")
        rope_rows = rope_cos.shape[0]
    if qk_bias is not None and (qk_bias.dtype != torch.bfloat16 or qk_bias.numel() != (num_heads + kv_heads) * dim or not qk_bias.is_contiguous() or qk_bias.data_ptr() % 16):
        raise ValueError(f"qk_bias must be a contiguous 16-byte aligned bf16 tensor of {num_heads} + {kv_heads} heads of {dim}")
    _launch(
        dev, "cdb_kv8_append", qkv.data_ptr(), qkv.stride(0), _lib.ptr(q_out), 0 if q_out is None else q_out.stride(0),
        codes.data_ptr(), scales.data_ptr(), layers, cache_layer, blocks, block_table.data_ptr(), block_table.stride(0),
        block_table.shape[0], block_table.shape[1], item_slot.data_ptr(), item_pos.data_ptr(), rope_mode,
        _lib.ptr(rope_cos) if rope_mode else None, _lib.ptr(rope_sin) if rope_mode else None, rope_rows,
        _lib.ptr(qk_bias), n, num_heads, kv_heads, dim, _status(qkv).data_ptr(),
    )


@_define("kv8_gather(Tensor codes, Tensor scales, int cache_layer, Tensor blocks, Tensor(a!) out) -> ()")
def kv8_gather(codes, scales, cache_layer, blocks, out):
    """Read blocks of the 8-bit cache back: ``out [n, 2, kv heads, 16, head dim]`` (bf16, exact) from
    block ids ``blocks [n]`` (``cdb_kv8_gather``)."""

    dev = _one_device(codes, scales, blocks, out)
    layers, nblocks, kv_heads, dim = _kv8_cache(codes, scales, cache_layer)
    n = blocks.numel()
    _int_row("blocks", blocks, n)
    if out.dtype != torch.bfloat16 or out.shape != (n, 2, kv_heads, KV8_BLOCK, dim) or not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError(f"out must be a contiguous 16-byte aligned bf16 tensor {(n, 2, kv_heads, KV8_BLOCK, dim)}, got {out.dtype} {tuple(out.shape)}")
    _launch(dev, "cdb_kv8_gather", codes.data_ptr(), scales.data_ptr(), layers, cache_layer, nblocks, kv_heads, dim,
            blocks.data_ptr(), n, out.data_ptr(), _status(codes).data_ptr())


def _kv8_workspace(dev: torch.device, ctas: int, dim: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Piece buffer and arrival counters of the decode attention. Eager calls keep one per stream, so
    that calls on two streams never share one. A captured call takes its own from the graph's memory
    and zeroes the counters inside the graph, so that two graphs may be replayed at once."""

    floats = _lib.load().cdb_kv8_decode_workspace_floats(ctas, dim)
    if torch.cuda.is_current_stream_capturing():
        return (torch.empty(floats, dtype=torch.float32, device=dev), torch.zeros(ctas, dtype=torch.int32, device=dev))
    key = (dev.index, torch.cuda.current_stream(dev).cuda_stream)
    ws = _KV8_WS.get(key)
    if ws is None or ws[0].numel() < floats:
        ws = _KV8_WS[key] = (torch.empty(floats, dtype=torch.float32, device=dev),
                             torch.zeros(ctas, dtype=torch.int32, device=dev))
    return ws


def _kv8_heads(num_heads: int, kv_heads: int) -> None:
    if num_heads <= 0 or num_heads % kv_heads:
        raise ValueError(f"num_heads must be a positive multiple of the cache's {kv_heads} kv heads, got {num_heads}")


@_define(
    "kv8_decode_attention(Tensor q, Tensor(a!) out, Tensor codes, Tensor scales, int cache_layer, Tensor block_table, "
    "Tensor item_slot, Tensor item_pos, int num_heads, float scale) -> ()"
)
def kv8_decode_attention(q, out, codes, scales, cache_layer, block_table, item_slot, item_pos, num_heads, scale):
    """Decode attention over the 8-bit cache: row i attends to positions ``0 .. item_pos[i]`` of slot
    ``item_slot[i]`` (``cdb_kv8_decode_attention``). ``q`` is rotated; a row at a negative position
    is skipped and its ``out`` left as it was. Any multiple of the cache's kv heads."""

    dev = _one_device(q, out, codes, scales, block_table, item_slot, item_pos)
    layers, blocks, kv_heads, dim = _kv8_cache(codes, scales, cache_layer)
    _kv8_heads(num_heads, kv_heads)
    n = item_pos.numel()
    _rows_of("q", q, n, num_heads * dim)
    _rows_of("out", out, n, num_heads * dim)
    _int_row("item_pos", item_pos, n)
    _int_row("item_slot", item_slot, n)
    _table_of("block_table", block_table)
    ctas = 2 * _sm_count(dev)
    ws, counters = _kv8_workspace(dev, ctas, dim)
    _launch(
        dev, "cdb_kv8_decode_attention", q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0), codes.data_ptr(),
        scales.data_ptr(), layers, cache_layer, blocks, block_table.data_ptr(), block_table.stride(0),
        block_table.shape[0], block_table.shape[1], item_slot.data_ptr(), item_pos.data_ptr(), n, num_heads, kv_heads,
        dim, scale, ctas, ws.data_ptr(), ws.numel(), counters.data_ptr(), _status(q).data_ptr(),
    )


@_define(
    "kv8_prefill_attention(Tensor q, Tensor(a!) out, Tensor codes, Tensor scales, int cache_layer, Tensor block_table, "
    "Tensor tiles, int num_heads, float scale) -> ()"
)
def kv8_prefill_attention(q, out, codes, scales, cache_layer, block_table, tiles, num_heads, scale):
    """Causal attention of prompt chunks over the 8-bit cache (``cdb_kv8_prefill_attention``).
    ``tiles [n, 4]`` int32 as ``OuroRunner.prefill_tiles`` or ``step_tables`` make them: first row, rows
    (at most 64; 0 for an unused entry), slot, position of the first row. The chunk's own keys and
    values are in the cache already, ``q`` is rotated."""

    dev = _one_device(q, out, codes, scales, block_table, tiles)
    layers, blocks, kv_heads, dim = _kv8_cache(codes, scales, cache_layer)
    _kv8_heads(num_heads, kv_heads)
    if tiles.dtype != torch.int32 or tiles.dim() != 2 or tiles.shape[1] != 4 or not tiles.is_contiguous() or tiles.data_ptr() % 16:
        raise ValueError(f"tiles must be a contiguous 16-byte aligned int32 tensor [n, 4], got {tiles.dtype} {tuple(tiles.shape)}")
    if tiles.shape[0] > 65535:
        raise ValueError(f"one call takes at most 65535 tiles, got {tiles.shape[0]}")
    rows = q.shape[0]
    _rows_of("q", q, 0, num_heads * dim)
    _rows_of("out", out, rows, num_heads * dim)
    _table_of("block_table", block_table)
    _launch(
        dev, "cdb_kv8_prefill_attention", q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0), rows,
        codes.data_ptr(), scales.data_ptr(), layers, cache_layer, blocks, block_table.data_ptr(), block_table.stride(0),
        block_table.shape[0], block_table.shape[1], tiles.data_ptr(), tiles.shape[0], num_heads, kv_heads, dim, scale,
        _status(q).data_ptr(),
    )


@_define(
    "step_tables(Tensor slots, Tensor seq_len, Tensor new_len, Tensor row_len, Tensor(a!) block_table, Tensor ring, "
    "Tensor state, Tensor(b!) row_len_out, Tensor(c!) state_out, Tensor(d!) granted, Tensor(e!) cu_seq_lens_q, "
    "Tensor(f!) cu_seq_lens_k, Tensor(g!) item_slot, Tensor(h!) item_pos, Tensor(i!) slot_map, Tensor(j!)? tiles) -> ()"
)
def step_tables(slots, seq_len, new_len, row_len, block_table, ring, state, row_len_out, state_out, granted,
                cu_seq_lens_q, cu_seq_lens_k, item_slot, item_pos, slot_map, tiles):
    """One step's metadata from its requests' lengths (``cdb_step_tables``): blocks for the new tokens
    taken from the FIFO ring into ``block_table``, cumulative lengths, every token's slot, position and
    cache row (-1 behind the last), and the prefill tiles. ``row_len_out`` / ``state_out`` may be
    ``row_len`` / ``state`` themselves."""

    dev = _one_device(slots, seq_len, new_len, row_len, block_table, ring, state, row_len_out, state_out, granted,
                      cu_seq_lens_q, cu_seq_lens_k, item_slot, item_pos, slot_map, tiles)
    n, rows = slots.numel(), row_len.numel()
    _int_row("slots", slots, n)
    _int_row("new_len", new_len, n)
    _int_row("granted", granted, n)
    _int_row("cu_seq_lens_q", cu_seq_lens_q, n + 1)
    _int_row("cu_seq_lens_k", cu_seq_lens_k, n + 1)
    _int_row("row_len", row_len, rows)
    _int_row("row_len_out", row_len_out, rows)
    _int_row("seq_len", seq_len, rows)
    _int_row("ring", ring, 0)
    _int_row("state", state, 4)
    _int_row("state_out", state_out, 4)
    _table_of("block_table", block_table)
    if block_table.shape[0] < rows:
        raise ValueError(f"block_table needs a row for each of the {rows} slots, got {block_table.shape[0]}")
    cap = item_pos.numel()
    _int_row("item_pos", item_pos, cap)
    _int_row("item_slot", item_slot, cap)
    _int_row("slot_map", slot_map, cap, torch.int64)
    if n > 8192:
        raise ValueError(f"one call takes at most 8192 requests, got {n}")
    if tiles is not None and (tiles.dtype != torch.int32 or tiles.dim() != 2 or tiles.shape[1] != 4 or not tiles.is_contiguous() or tiles.data_ptr() % 16):
        raise ValueError(f"tiles must be a contiguous 16-byte aligned int32 tensor [n, 4], got {tiles.dtype} {tuple(tiles.shape)}")
    _launch(
        dev, "cdb_step_tables", slots.data_ptr(), seq_len.data_ptr(), new_len.data_ptr(), row_len.data_ptr(), n,
        block_table.data_ptr(), block_table.stride(0), rows, block_table.shape[1], ring.data_ptr(), ring.numel(),
        state.data_ptr(), row_len_out.data_ptr(), state_out.data_ptr(), granted.data_ptr(), cu_seq_lens_q.data_ptr(),
        cu_seq_lens_k.data_ptr(), item_slot.data_ptr(), item_pos.data_ptr(), slot_map.data_ptr(), cap,
        _lib.ptr(tiles), 0 if tiles is None else tiles.shape[0], _status(slots).data_ptr(),
    )


@_define("gemv_w4(Tensor x, Tensor w, Tensor scales, Tensor? zeros, Tensor(a!) out) -> ()")
def gemv_w4(x, w, scales, zeros, out):
    """``out [M, N] = x [M, K] @ W.T`` for a few token rows, ``W = scales * (q - zeros)`` from 4-bit
    ``w [N, K / 2]`` uint8 (low nibble first), bf16 ``scales [N, K / group]`` and uint8 ``zeros`` of the
    same shape (None: 8) (``cdb_gemv_w4``). Groups of 32, 64 or a multiple of 128. The weights are
    read once per 32 rows: above some hundred rows ``gemm_bf16`` is the better call."""

    dev = _one_device(x, w, scales, zeros, out)
    if w.dtype != torch.uint8 or w.dim() != 2 or w.shape[0] == 0 or w.shape[1] == 0 or w.stride(1) != 1:
        raise ValueError(f"w must be a 2-D uint8 tensor [N, K / 2] with unit column stride, got {w.dtype} {tuple(w.shape)}")
    n, k = w.shape[0], 2 * w.shape[1]
    ldw = w.stride(0) if n > 1 else -(-w.shape[1] // 16) * 16
    if k % 32 or ldw % 16 or ldw < w.shape[1] or w.data_ptr() % 16:
        raise ValueError(f"w needs K a multiple of 32, a row stride that is a multiple of 16 bytes and 16-byte alignment, got K {k}")
    _dtype("scales", scales, torch.bfloat16, 2)
    groups = scales.shape[1]
    if scales.shape[0] != n or groups == 0 or k % groups or not scales.is_contiguous():
        raise ValueError(f"scales must be contiguous [{n}, K / group], got {tuple(scales.shape)} for K {k}")
    group = k // groups
    if group not in (32, 64) and group % 128:
        raise ValueError(f"groups of 32, 64 or a multiple of 128 are taken, got {group}")
    if zeros is not None and (zeros.dtype != torch.uint8 or zeros.shape != scales.shape or not zeros.is_contiguous()):
        raise ValueError(f"zeros must be a contiguous uint8 tensor {tuple(scales.shape)}, got {zeros.dtype} {tuple(zeros.shape)}")
    m = x.shape[0]
    _rows_of("x", x, m, k)
    if x.shape[1] != k:
        raise ValueError(f"x has {x.shape[1]} columns, the weights {k}")
    if out.dtype != torch.bfloat16 or out.shape != (m, n) or (n > 1 and out.stride(1) != 1) or (m > 1 and out.stride(0) < n):
        raise ValueError(f"out must be a bf16 tensor [{m}, {n}] with unit column stride, got {out.dtype} {tuple(out.shape)}")
    _launch(
        dev, "cdb_gemv_w4", x.data_ptr(), max(x.stride(0), k), w.data_ptr(), ldw, scales.data_ptr(), _lib.ptr(zeros),
        out.data_ptr(), max(out.stride(0), n), m, n, k, group, _sm_count(dev), _status(x).data_ptr(),
    )
