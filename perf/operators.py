"""The low-bit decode step's operators, as cases that can be timed and compared.

* ``tables``: block tables, slot maps and prefill tiles of one step from the requests' lengths;
* ``append``: rotated keys and values quantised into the 8-bit paged cache (one scale per block of
  16 tokens and head), and the touched blocks read back;
* ``decode`` / ``prefill``: attention over that cache for single tokens and for prompt chunks;
* ``gemv``: a few token rows times 4-bit weights with group scales.

``run`` computes each in elementary torch operations where ``own`` is false and calls
``torch.ops.cdb`` where it is true; ``exact`` restates the definitions in 64 bits.

The cache holds e4m3 codes ``[layers, 2, blocks, kv heads, 16, head dim]`` and fp32 scales
``[layers, 2, blocks, kv heads]``. A scale is the smallest power of two that brings its block's
largest finite magnitude to at most 448; appending to a part-filled block can only raise it, and
the codes that were there are then rescaled.
"""

from __future__ import annotations

import math

import torch

own = False

BS = 16  # tokens of one cache block
TILE = 64  # query rows of one prefill tile
DEV = "cuda"
E4M3_MAX = 448.0


def listed():
    return [
        # One decode step of the engine's whole batch (256 requests): one token each.
        dict(name="tables decode step", op="tables", requests=256, max_ctx=2048, max_new=1, pad=0),
        # Prompt admission: 64 requests of up to 512 new tokens, some with earlier chunks cached.
        dict(name="tables prefill step", op="tables", requests=64, max_ctx=1024, max_new=512, pad=100),
        # One layer of a recurrent launch at the engine's mean width, 16 heads of 128, split-half RoPE.
        dict(name="append 80 tokens", op="append", requests=80, max_ctx=1024, max_new=1, heads=16, kv_heads=16, dim=128, rope=1, bias=False),
        # Prompt rows of the 55 x 96 model: interleaved RoPE with the learned bias.
        dict(name="append prompts 55x96", op="append", requests=16, max_ctx=64, max_new=512, heads=55, kv_heads=55, dim=96, rope=2, bias=True),
        # One interactive request: only latency counts.
        dict(name="decode one request", op="decode", requests=1, min_ctx=700, max_ctx=700, heads=16, kv_heads=16, dim=128),
        # The engine's mean recurrent launch: 80 rows at ragged positions.
        dict(name="decode 80 requests", op="decode", requests=80, min_ctx=64, max_ctx=1300, heads=16, kv_heads=16, dim=128),
        # Long documents under grouped heads: the cache is what is read.
        dict(name="decode long grouped", op="decode", requests=8, min_ctx=30000, max_ctx=65536, heads=32, kv_heads=8, dim=128),
        # Ragged prompt chunks, some after cached tokens.
        dict(name="prefill ragged chunks", op="prefill", requests=12, max_ctx=700, max_new=400, heads=16, kv_heads=16, dim=128),
        # A long prompt's second half.
        dict(name="prefill long chunk", op="prefill", requests=1, max_ctx=4096, max_new=4096, heads=16, kv_heads=16, dim=128),
        # Down projection (2048 x 5632) of one token.
        dict(name="gemv down 1 token", op="gemv", tokens=1, n=2048, k=5632, group=128, zeros=False),
        # Gate and up projections (2 x 5632 x 2048) of a small batch.
        dict(name="gemv gate-up 24 tokens", op="gemv", tokens=24, n=11264, k=2048, group=128, zeros=True),
        # LM head (vocabulary 49152) of 8 tokens, small groups with zero points.
        dict(name="gemv lm head 8 tokens", op="gemv", tokens=8, n=49152, k=2048, group=64, zeros=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tables", "append", "decode", "prefill", "gemv"])
    if op == "tables":
        r = _log(rng, 1, 512)
        return dict(op=op, requests=r, max_ctx=_log(rng, 16, 4096), max_new=_log(rng, 1, max(1, min(2048, 32768 // r))), pad=rng.randint(0, 300))
    if op == "gemv":
        group = rng.choice([32, 64, 128])
        k = group * max(1, _log(rng, 256, 8192) // group)
        n = _log(rng, 64, min(49152, 49152 * 2048 // k))
        return dict(op=op, tokens=_log(rng, 1, 32), n=n, k=k, group=group, zeros=rng.random() < 0.5)
    dim = rng.choice([64, 96, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 16, 55 if dim == 96 else 12])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 8] if kv_heads <= 8 else [1])
    if op == "append":
        r = _log(rng, 1, 256)
        return dict(op=op, requests=r, max_ctx=_log(rng, 16, 2048), max_new=_log(rng, 1, max(1, min(1024, 4096 // r))), heads=heads, kv_heads=kv_heads, dim=dim, rope=rng.randint(0, 2), bias=rng.random() < 0.5)
    if op == "decode":
        r = _log(rng, 1, 256)
        top = _log(rng, 1, max(1, min(65536, 500_000_000 // (r * kv_heads * dim))))
        return dict(op=op, requests=r, min_ctx=max(1, top // rng.randint(1, 8)), max_ctx=top, heads=heads, kv_heads=kv_heads, dim=dim)
    if heads > 55:
        heads = kv_heads
    r = _log(rng, 1, 16)
    return dict(op=op, requests=r, max_ctx=_log(rng, 1, max(1, 4096 // r)), max_new=_log(rng, 1, max(1, 1536 // r)), heads=heads, kv_heads=kv_heads, dim=dim)


# ---------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _ints(g, lo, hi, n):
    return torch.randint(lo, hi + 1, (n,), generator=g, device=DEV, dtype=torch.int32)


def _lengths(case, g):
    """Cached and new tokens of each request: the same lengths for every seed, so that outputs keep
    their shapes, in another order."""

    r = case["requests"]
    fixed = _gen(r)
    if case["op"] == "decode":
        total = _ints(fixed, case["min_ctx"], case["max_ctx"], r)
        ctx, new = total - 1, torch.ones_like(total)
    else:
        ctx, new = _ints(fixed, 0, case["max_ctx"], r), _ints(fixed, 1, case["max_new"], r)
        if case["max_new"] > 1:
            ctx[::3] = 0  # fresh prompts among later chunks
    if r == 1:
        ctx[:], new[:] = case["max_ctx"] - (case["op"] == "decode"), 1 if case["op"] == "decode" else case["max_new"]
    order = torch.randperm(r, generator=g, device=DEV)
    return ctx[order], new[order]


def _rows(ctx, new):
    """Request and position of every token row, requests in order."""

    total = int(new.sum())
    req = torch.repeat_interleave(torch.arange(new.numel(), device=DEV), new.long(), output_size=total)
    first = (new.cumsum(0) - new).long()
    pos = ctx.long()[req] + torch.arange(total, device=DEV) - first[req]
    return req, pos


def _prefill_tiles(ctx, new):
    """{first row, rows, slot, position} of every run of at most 64 rows, longest attention first."""

    tiles, row = [], 0
    for slot, (c, n) in enumerate(zip(ctx.tolist(), new.tolist())):
        tiles += [(row + i, min(TILE, n - i), slot, c + i) for i in range(0, n, TILE)]
        row += n
    tiles.sort(key=lambda t: -(t[3] + t[1]))
    return torch.tensor(tiles, dtype=torch.int32).to(DEV)


def _cache(case, g, blocks, layers=1):
    """A cache with every block written: values of unit size, block scales that differ a little."""

    shape = (layers, 2, blocks, case["kv_heads"], BS, case["dim"])
    codes = torch.empty(shape, dtype=torch.float8_e4m3fn, device=DEV)
    for layer in range(layers):
        for kv in range(2):
            v = torch.randn(shape[2:], generator=g, device=DEV, dtype=torch.bfloat16)
            codes[layer, kv] = (v * 90).clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    e = torch.randint(-8, -5, shape[:4], generator=g, device=DEV)
    return codes, torch.ldexp(torch.ones(shape[:4], device=DEV), e)


def _block_table(g, pages, width, spare=0):
    """Pages of every request at shuffled block ids; -1 past a request's pages."""

    total = int(pages.sum())
    ids = torch.randperm(total + spare, generator=g, device=DEV).int()
    first = (pages.cumsum(0) - pages).long()
    col = torch.arange(width, device=DEV)
    at = (first[:, None] + col[None, :]).clamp_(max=max(0, total - 1))
    return torch.where(col[None, :] < pages[:, None], ids[at], torch.full_like(ids[at], -1)), ids[total:]


def _rope_tables(case, positions):
    dim = case["dim"]
    inv = 10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=DEV) / dim)
    ang = torch.arange(positions, dtype=torch.float64, device=DEV)[:, None] * inv
    if case["rope"] == 1:  # bf16 [positions, dim], the two halves alike
        ang = torch.cat((ang, ang), -1)
        return ang.cos().bfloat16(), ang.sin().bfloat16()
    return ang.cos().float(), ang.sin().float()  # fp32 [positions, dim / 2]


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case)
    if case["op"] == "gemv":
        m, n, k, grp = case["tokens"], case["n"], case["k"], case["group"]
        s["x"] = torch.randn(m, k, generator=g, device=DEV, dtype=torch.bfloat16)
        s["w"] = torch.randint(0, 256, (n, k // 2), generator=g, device=DEV, dtype=torch.uint8)
        s["scales"] = (torch.rand(n, k // grp, generator=g, device=DEV) * 0.01 + 0.002).bfloat16()
        s["zeros"] = torch.randint(4, 12, (n, k // grp), generator=g, device=DEV, dtype=torch.uint8) if case["zeros"] else None
        s["out"] = torch.empty(m, n, device=DEV, dtype=torch.bfloat16)
        return s
    ctx, new = _lengths(case, g)
    if case["op"] == "tables":
        return _prepare_tables(s, g, ctx, new)
    r = ctx.numel()
    pages = (ctx + new + BS - 1) // BS
    width = int(pages.max()) + 3
    s["table"], _ = _block_table(g, pages, width)
    s["codes"], s["scales"] = _cache(case, g, int(pages.sum()) + 2)
    hq, hkv, d = case["heads"], case["kv_heads"], case["dim"]
    req, pos = _rows(ctx, new)
    s["slot"], s["pos"] = req.int(), pos.int()
    s["scale"] = d**-0.5
    s["ctx"], s["new"] = ctx, new
    if case["op"] == "append":
        s["qkv"] = torch.randn(req.numel(), (hq + 2 * hkv) * d, generator=g, device=DEV, dtype=torch.bfloat16)
        # some requests' newest tokens are larger than what their block holds: its scale has to grow
        s["qkv"][::3] *= 4
        s["bias_t"] = torch.randn(hq + hkv, d, generator=g, device=DEV).mul_(0.1).bfloat16() if case["bias"] else None
        s["cos"], s["sin"] = _rope_tables(case, int((ctx + new).max())) if case["rope"] else (None, None)
        s["q_out"] = torch.empty(req.numel(), hq * d, device=DEV, dtype=torch.bfloat16)
        first = ctx // BS
        col = torch.arange(width, device=DEV)
        hit = (col[None, :] >= first[:, None]) & (col[None, :] < pages[:, None])
        s["blocks"] = s["table"][hit].contiguous()
        s["read"] = torch.empty(s["blocks"].numel(), 2, hkv, BS, d, device=DEV, dtype=torch.bfloat16)
        return s
    s["q"] = torch.randn(req.numel(), hq * d, generator=g, device=DEV, dtype=torch.bfloat16)
    s["out"] = torch.empty_like(s["q"])
    if case["op"] == "prefill":
        s["tiles"] = _prefill_tiles(ctx, new)
        # sizes that a server knows on the host
        s["n_max"], s["l_max"] = int(new.max()), int((ctx + new).max())
        s["first"] = new.cumsum(0) - new
    else:
        s["l_max"] = int((ctx + new).max())
    return s


def _prepare_tables(s, g, ctx, new):
    r = ctx.numel()
    slots_n = r + 8
    slots = torch.randperm(slots_n, generator=g, device=DEV)[:r].int()
    held = (ctx + BS - 1) // BS
    total = (ctx + new + BS - 1) // BS
    width = int(total.max()) + 2
    rows, free = _block_table(g, held, width, spare=int((total - held).sum()) + 9)
    s["table"] = torch.full((slots_n, width), -1, dtype=torch.int32, device=DEV)
    s["table"][slots.long()] = rows
    # the free ids lie in the ring from `head` on, around its end
    nb = int(held.sum()) + free.numel()
    head = int(torch.randint(0, nb, (1,), generator=g, device=DEV))
    s["ring"] = torch.full((nb,), -1, dtype=torch.int32, device=DEV)
    s["ring"][(head + torch.arange(free.numel(), device=DEV)) % nb] = free
    s["state"] = torch.tensor([head, free.numel(), nb, int(held.sum())], dtype=torch.int32, device=DEV)
    s["row_len"] = torch.zeros(slots_n, dtype=torch.int32, device=DEV)
    s["row_len"][slots.long()] = held
    s["seq_len"] = torch.zeros(slots_n, dtype=torch.int32, device=DEV)
    s["seq_len"][slots.long()] = ctx
    s["slots"], s["new"] = slots, new
    cap = int(new.sum()) + s["pad"]  # the launch bucket that the host has chosen
    s["cap"], s["tile_cap"] = cap, cap // TILE + r
    s["need_max"] = int((total - held).max())
    i32 = dict(dtype=torch.int32, device=DEV)
    s["o_row_len"], s["o_state"], s["granted"] = s["row_len"].clone(), torch.empty(4, **i32), torch.empty(r, **i32)
    s["cu_q"], s["cu_k"] = torch.empty(r + 1, **i32), torch.empty(r + 1, **i32)
    s["slot"], s["pos"], s["tiles"] = torch.empty(cap, **i32), torch.empty(cap, **i32), torch.empty(s["tile_cap"], 4, **i32)
    s["map"] = torch.empty(cap, dtype=torch.int64, device=DEV)
    return s


# ---------------------------------------------------------------- passes


def run(state):
    return {"tables": _tables, "append": _append, "decode": _decode, "prefill": _prefill, "gemv": _gemv}[state["op"]](state)


def _ops():
    import continuous_depth_batching_b200.ops  # noqa: F401  (registers torch.ops.cdb)

    return torch.ops.cdb


def _tables(s):
    if own:
        _ops().step_tables(s["slots"], s["seq_len"], s["new"], s["row_len"], s["table"], s["ring"], s["state"], s["o_row_len"], s["o_state"], s["granted"],
                           s["cu_q"], s["cu_k"], s["slot"], s["pos"], s["map"], s["tiles"])
        return {k: s[k] for k in ("table", "o_row_len", "o_state", "granted", "cu_q", "cu_k", "slot", "pos", "map", "tiles")}
    sl, new = s["slots"].long(), s["new"].long()
    ctx, held = s["seq_len"][sl].long(), s["row_len"][sl].long()
    total = (ctx + new + BS - 1) // BS
    need = (total - held).clamp(min=0)
    off = need.cumsum(0) - need
    nb = s["ring"].numel()
    # new block ids, request by request, from the ring's head; places past a request's need go to a spare column
    i = torch.arange(s["need_max"], device=DEV)
    ids = s["ring"][(s["state"][0] + off[:, None] + i) % nb]
    width = s["table"].shape[1]
    rows = torch.nn.functional.pad(s["table"][sl], (0, 1))
    rows.scatter_(1, torch.where(i < need[:, None], held[:, None] + i, width), ids)
    table = s["table"].clone()
    table[sl] = rows[:, :width]
    row_len = s["o_row_len"].clone()
    row_len[sl] = (held + need).int()
    taken = need.sum()
    st = s["state"].long()
    state = torch.stack(((st[0] + taken) % nb, st[1] - taken, st[2], torch.maximum(st[3], st[2] - st[1] + taken))).int()
    zero = torch.zeros(1, dtype=torch.int64, device=DEV)
    cu_q, cu_k = torch.cat((zero, new.cumsum(0))), torch.cat((zero, (ctx + new).cumsum(0)))
    t = torch.arange(s["cap"], device=DEV)
    req = torch.searchsorted(cu_q[1:], t, right=True)
    live = req < sl.numel()
    req = req.clamp(max=sl.numel() - 1)
    pos = ctx[req] + t - cu_q[req]
    page = (pos // BS).clamp(max=table.shape[1] - 1)
    rows = table[sl[req], page].long() * BS + pos % BS
    pad = lambda v: torch.where(live, v, torch.full_like(v, -1))  # noqa: E731
    cu_t = ((new + TILE - 1) // TILE).cumsum(0)
    u = torch.arange(s["tile_cap"], device=DEV)
    tr = torch.searchsorted(cu_t, u, right=True)
    tl = (tr < sl.numel())[:, None]
    tr = tr.clamp(max=sl.numel() - 1)
    at = (u - cu_t[tr] + (new[tr] + TILE - 1) // TILE) * TILE
    tiles = torch.stack((cu_q[tr] + at, (new[tr] - at).clamp(max=TILE), sl[tr], ctx[tr] + at), 1)
    return {"table": table, "o_row_len": row_len, "o_state": state, "granted": torch.ones_like(s["slots"]), "cu_q": cu_q.int(), "cu_k": cu_k.int(),
            "slot": pad(sl[req]).int(), "pos": pad(pos).int(), "map": pad(rows), "tiles": torch.where(tl, tiles, torch.zeros_like(tiles)).int()}


def _scale_of(amax):
    """2^e with the smallest e for which amax <= 448 * 2^e (e >= -126)."""

    m, e = torch.frexp(amax)
    e = e.long() - 9 + (m > 0.875).long()
    return torch.ldexp(torch.ones_like(amax), torch.where(amax > 0, e, torch.full_like(e, -126)).clamp(min=-126))


def _rotate(x, case, cos, sin, pos):
    if case["rope"] == 1:
        c, sn = cos[pos][:, None].to(x.dtype), sin[pos][:, None].to(x.dtype)
        h = x.shape[-1] // 2
        return x * c + torch.cat((-x[..., h:], x[..., :h]), -1) * sn
    if case["rope"] == 2:
        c, sn = cos[pos][:, None].to(x.dtype), sin[pos][:, None].to(x.dtype)
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * c - b * sn, b * c + a * sn), -1).flatten(-2)
    return x


def _append(s):
    if own:
        ops = _ops()
        ops.kv8_append(s["qkv"], s["q_out"], s["codes"], s["scales"], 0, s["table"], s["slot"], s["pos"], s["cos"], s["sin"], s["bias_t"], s["rope"], s["heads"])
        ops.kv8_gather(s["codes"], s["scales"], 0, s["blocks"], s["read"])
        return {"q": s["q_out"], "blocks": s["read"]}
    hq, hkv, d, t = s["heads"], s["kv_heads"], s["dim"], s["qkv"].shape[0]
    x = s["qkv"].float().view(t, hq + 2 * hkv, d)
    qk = x[:, : hq + hkv]
    if s["bias_t"] is not None:
        qk = qk + s["bias_t"].float()
    pos = s["pos"].long()
    qk = _rotate(qk, s, s["cos"], s["sin"], pos)
    s["q_out"].copy_(qk[:, :hq].reshape(t, -1))
    new = torch.stack((qk[:, hq:], x[:, hq + hkv :]), 1)  # [t, 2, hkv, d]
    codes, scales = s["codes"][0].view(torch.uint8), s["scales"][0]
    blk = s["table"][s["slot"].long(), pos // BS].long()
    off = pos % BS
    nb = codes.shape[1]
    amax = torch.zeros(nb, 2, hkv, device=DEV).index_reduce_(0, blk, new.abs().amax(-1), "amax")
    start = torch.full((nb,), BS, device=DEV).index_reduce_(0, blk, off, "amin")  # first token written now
    fresh = _scale_of(amax)
    b = s["blocks"].long()
    was = scales[:, b].transpose(0, 1)  # [blocks, 2, hkv]
    grown = torch.where((start[b] == 0)[:, None, None], fresh[b], torch.maximum(was, fresh[b]))
    held = codes[:, b].view(torch.float8_e4m3fn).transpose(0, 1).float()  # [blocks, 2, hkv, 16, d]
    keep = torch.arange(BS, device=DEV)[None, :] < start[b][:, None]
    moved = held * torch.where(keep[:, None, None, :], (was / grown)[..., None], torch.ones((), device=DEV))[..., None]
    codes[:, b] = moved.to(torch.float8_e4m3fn).view(torch.uint8).transpose(0, 1)
    scales[:, b] = grown.transpose(0, 1)
    q = (new / scales[:, blk].transpose(0, 1)[..., None]).clamp(-E4M3_MAX, E4M3_MAX)
    q = q.to(torch.float8_e4m3fn).view(torch.uint8)
    codes[0, blk, :, off] = q[:, 0]
    codes[1, blk, :, off] = q[:, 1]
    read = (codes[:, b].view(torch.float8_e4m3fn).float() * scales[:, b][..., None, None]).transpose(0, 1)
    return {"q": s["q_out"], "blocks": read.bfloat16()}


def _keys_values(s, dtype):
    """Cached keys and values of every request, [requests, kv heads, tokens, dim], padded with zeros."""

    l = s["l_max"]
    blk = s["table"][:, : (l + BS - 1) // BS].long().clamp(min=0)
    r, w = blk.shape
    live = torch.arange(w * BS, device=DEV)[None, :] < (s["ctx"] + s["new"])[:, None]

    def get(kv):
        x = s["codes"][0, kv].view(torch.uint8)[blk].view(torch.float8_e4m3fn).to(dtype) * s["scales"][0, kv][blk].to(dtype)[..., None, None]
        x = x.transpose(1, 2).reshape(r, s["kv_heads"], w * BS, s["dim"])
        return x.masked_fill_(~live[:, None, :, None], 0)

    return get(0), get(1), live


def _decode(s):
    if own:
        _ops().kv8_decode_attention(s["q"], s["out"], s["codes"], s["scales"], 0, s["table"], s["slot"], s["pos"], s["heads"], s["scale"])
        return s["out"]
    k, v, live = _keys_values(s, torch.float32)
    r, hkv, d = s["requests"], s["kv_heads"], s["dim"]
    q = s["q"].float().view(r, hkv, -1, d)
    x = torch.matmul(q, k.transpose(-1, -2)) * s["scale"]
    x = x.masked_fill(~live[:, None, None, :], -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    return (torch.matmul(p, v) / p.sum(-1, keepdim=True)).reshape(r, -1).bfloat16()


def _prefill(s):
    if own:
        _ops().kv8_prefill_attention(s["q"], s["out"], s["codes"], s["scales"], 0, s["table"], s["tiles"], s["heads"], s["scale"])
        return s["out"]
    k, v, live = _keys_values(s, torch.float32)
    r, hkv, d, n = s["requests"], s["kv_heads"], s["dim"], s["n_max"]
    g = s["heads"] // hkv
    i = torch.arange(n, device=DEV)
    rows = (s["first"][:, None] + i).clamp(max=s["q"].shape[0] - 1).long()
    q = s["q"].float()[rows].view(r, n, hkv, g, d).permute(0, 2, 3, 1, 4)
    x = torch.matmul(q, k[:, :, None].transpose(-1, -2)).mul_(s["scale"])
    at = s["ctx"][:, None] + i
    seen = torch.arange(k.shape[2], device=DEV)[None, None, :] <= at[:, :, None]
    x.masked_fill_(~seen[:, None, None], -math.inf)
    p = x.sub_(x.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(p, v[:, :, None]) / p.sum(-1, keepdim=True)
    o = o.permute(0, 3, 1, 2, 4).reshape(r, n, -1).bfloat16()
    req = s["slot"].long()
    return o[req, s["pos"].long() - s["ctx"].long()[req]]


def _gemv(s):
    if own:
        _ops().gemv_w4(s["x"], s["w"], s["scales"], s["zeros"], s["out"])
        return s["out"]
    n, k, g = s["n"], s["k"], s["group"]
    q = torch.stack((s["w"] & 15, s["w"] >> 4), -1).view(n, k // g, g).float()
    z = s["zeros"].float()[..., None] if s["zeros"] is not None else 8.0
    w = ((q - z) * s["scales"].float()[..., None]).view(n, k)
    return torch.matmul(s["x"].float(), w.t()).bfloat16()


# ---------------------------------------------------------------- work and definition


def _spans(case):
    """Mean cached and new tokens per request, as prepare() spreads them."""

    if case["op"] == "decode":
        return (case["min_ctx"] + case["max_ctx"]) / 2 - 1, 1.0
    if case["requests"] == 1:
        return float(case["max_ctx"]), float(case["max_new"])
    ctx = case["max_ctx"] / 2 * (2 / 3 if case["max_new"] > 1 else 1)
    return ctx, (1 + case["max_new"]) / 2


def work(case):
    if case["op"] == "gemv":
        m, n, k, g = case["tokens"], case["n"], case["k"], case["group"]
        return {"bytes": n * k / 2 + n * (k // g) * (3 if case["zeros"] else 2) + 2 * m * (n + k), "flops": 2 * m * n * k}
    r = case["requests"]
    ctx, new = _spans(case)
    if case["op"] == "tables":
        # lengths in; request offsets, row slots, positions and cache rows out, new blocks in and out
        return {"bytes": r * (4 * 4 + 3 * 4) + r * new * (4 + 4 + 8 + 8 / BS + 16 / TILE), "flops": 0}
    hq, hkv, d = case["heads"], case["kv_heads"], case["dim"]
    rows = r * new
    if case["op"] == "append":
        # q, k, v in, q out; the touched blocks' codes in (held rows), out, and read back as bf16
        blocks = r * (new / BS + (1 if new < BS else 0.5))
        return {"bytes": rows * d * (2 * (hq + 2 * hkv) + 2 * hq + 2 * hkv) + blocks * 2 * hkv * BS * d * 3, "flops": 0}
    if case["op"] == "decode":
        keys = r * (ctx + 1)
    else:
        keys = rows * (ctx + new / 2)  # causal: the average row of a chunk sees half of it
    cache = r * (ctx + new) * 2 * hkv * (d + 4 / BS)
    return {"bytes": cache + rows * hq * d * 4, "flops": 4 * keys * hq * d}


def exact(case, seed):
    s = prepare(case, seed)
    return {"tables": _exact_tables, "append": _exact_append, "decode": _exact_attention, "prefill": _exact_attention, "gemv": _exact_gemv}[case["op"]](s)


def _exact_tables(s):
    return None  # whole numbers only: they have to be equal


def _exact_gemv(s):
    w = s["w"].to(torch.int64)
    n, k, grp = s["n"], s["k"], s["group"]
    col = torch.arange(k, device=DEV)
    q = torch.bitwise_and(torch.bitwise_right_shift(w[:, col // 2], 4 * (col % 2)), 15)
    z = s["zeros"].to(torch.int64)[:, col // grp] if s["zeros"] is not None else 8
    w64 = (q - z).double() * s["scales"].double()[:, col // grp]
    return torch.einsum("mk,nk->mn", s["x"].double(), w64)


def _exact_append(s):
    hq, hkv, d, t = s["heads"], s["kv_heads"], s["dim"], s["qkv"].shape[0]
    x = s["qkv"].double().reshape(t, hq + 2 * hkv, d).clone()
    pos = s["pos"].long()
    if s["bias_t"] is not None:
        x[:, : hq + hkv] += s["bias_t"].double()
    y = x.clone()
    if s["rope"]:
        c, sn = s["cos"].double()[pos], s["sin"].double()[pos]
        half = d // 2
        lo, hi = (torch.arange(half), torch.arange(half) + half) if s["rope"] == 1 else (torch.arange(0, d, 2), torch.arange(1, d, 2))
        lo, hi = lo.to(DEV), hi.to(DEV)
        c, sn = c[:, None, :half], sn[:, None, :half]
        a, b = x[:, : hq + hkv, lo], x[:, : hq + hkv, hi]
        y[:, : hq + hkv, lo], y[:, : hq + hkv, hi] = a * c - b * sn, b * c + a * sn
    # block by block: where its scale ends, and what every one of its places stands for
    table, slot = s["table"], s["slot"].long()
    blk = table[slot, pos // BS].long()
    b = s["blocks"].long()
    index = torch.full((s["codes"].shape[2],), -1, dtype=torch.int64, device=DEV)
    index[b] = torch.arange(b.numel(), device=DEV)
    home, off = index[blk], pos % BS
    kv = torch.stack((y[:, hq : hq + hkv], y[:, hq + hkv :]), 1)
    full = torch.zeros(b.numel(), BS, 2, hkv, d, dtype=torch.float64, device=DEV)
    here = torch.zeros(b.numel(), BS, dtype=torch.bool, device=DEV)
    full[home, off] = kv
    here[home, off] = True
    first = torch.where(here.any(1), here.int().argmax(1), BS)
    amax = full.abs().amax(-1).amax(1)
    e = torch.ceil(torch.log2(amax / 448)).clamp(min=-126)
    e = torch.where(torch.exp2(e) * 448 < amax, e + 1, torch.where(torch.exp2(e - 1) * 448 >= amax, e - 1, e))
    was = s["scales"][0].double()[:, b].permute(1, 0, 2)
    scale = torch.where((first > 0)[:, None, None], torch.maximum(was, torch.exp2(e)), torch.exp2(e))

    def to_codes(v):  # nearest e4m3 value, ties to the even mantissa
        p = torch.floor(torch.log2(v.abs().clamp(min=2.0**-9))).clamp(min=-6)
        step = torch.exp2(p - 3)
        return (torch.round(v / step) * step).clamp(-448, 448)

    old = s["codes"][0].view(torch.uint8)[:, b].view(torch.float8_e4m3fn).double().permute(1, 3, 0, 2, 4)  # [blocks, 16, 2, hkv, d]
    place = torch.arange(BS, device=DEV)[None, :]
    ratio = torch.where((place < first[:, None])[:, :, None, None], (was / scale)[:, None], 1.0)
    codes = torch.where(here[:, :, None, None, None], to_codes(full / scale[:, None, ..., None]), to_codes(old * ratio[..., None]))
    return {"q": y[:, :hq].reshape(t, -1), "blocks": (codes * scale[:, None, ..., None]).permute(0, 2, 3, 1, 4)}


def _exact_attention(s):
    ctx, new = s["ctx"].tolist(), s["new"].tolist()
    hq, hkv, d = s["heads"], s["kv_heads"], s["dim"]
    if sum(n * (c + n) for c, n in zip(ctx, new)) * hq * d > 2e12:
        return None
    out, row = [], 0
    for j, (c, n) in enumerate(zip(ctx, new)):
        l = c + n
        blk = s["table"][j, : (l + BS - 1) // BS].long()
        kv = s["codes"][0].view(torch.uint8)[:, blk].view(torch.float8_e4m3fn).double() * s["scales"][0][:, blk].double()[..., None, None]
        k, v = kv.permute(0, 2, 1, 3, 4).reshape(2, hkv, -1, d)[:, :, :l]
        q = s["q"][row : row + n].double().view(n, hkv, hq // hkv, d)
        x = torch.einsum("nhgd,hld->hgnl", q, k) * s["scale"]
        x = x + torch.triu(torch.full((n, l), -math.inf, dtype=torch.float64, device=DEV), diagonal=c + 1)
        out.append(torch.einsum("hgnl,hld->nhgd", torch.softmax(x, -1), v).reshape(n, -1))
        row += n
    return torch.cat(out)
