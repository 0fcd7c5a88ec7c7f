"""Operators of a decode step that continues prompts many times, as cases that can be timed and compared.

* ``norm``: RMS norms of each head's query and key, the position rotation and the append to the bf16 paged
  cache, in one pass;
* ``prefix``: decode attention over that cache for requests that share a prompt, whose keys and values are
  read once for all of them;
* ``sample``: the next token of every row from its logits, by temperature, top-k, top-p and min-p and one
  given random number, with its log-probability.

``run`` computes each in elementary torch operations where ``own`` is false and calls ``torch.ops.cdb``
where it is true; ``exact`` restates the definitions in 64 bits.

The cache is ``[layers, 2, rows, kv heads, head dim]`` in bf16; position p of a request lies in row
``table[slot, p // 16] * 16 + p % 16``.

A row of ``sample``: tokens weigh w = exp((logit - largest) / temperature) and are ordered by falling logit,
equal ones by index. Of them top-k keeps the first k, top-p of those the shortest beginning that holds a share
p of their weight, min-p of those the ones with w >= min_p. The token is the first by index at which the kept
weights' running sum passes u times their total. Temperature 0 takes the largest logit.
"""

from __future__ import annotations

import math

import torch

own = False

BS = 16  # tokens of one cache block
DEV = "cuda"
EPS = 1e-6


def listed():
    return [
        # One layer of a recurrent launch at the engine's mean width: 80 rows, 16 heads of 128, split-half RoPE.
        dict(name="norm 80 tokens", op="norm", requests=80, max_ctx=200, max_new=1, heads=16, kv_heads=16, dim=128, rope=1),
        # A batch of prompts under grouped heads.
        dict(name="norm prompts grouped", op="norm", requests=24, max_ctx=100, max_new=400, heads=32, kv_heads=8, dim=128, rope=1),
        # Prompt rows of the 55 x 96 model, interleaved pairs.
        dict(name="norm prompts 55x96", op="norm", requests=5, max_ctx=40, max_new=300, heads=55, kv_heads=55, dim=96, rope=2),
        # Four continuations of a short prompt: only latency counts.
        dict(name="prefix 4 of a short prompt", op="prefix", groups=1, requests=4, prefix=700, own=40, heads=16, kv_heads=16, dim=128),
        # Sixty-four continuations of one prompt, part way through.
        dict(name="prefix 64 of one prompt", op="prefix", groups=1, requests=64, prefix=4100, own=512, heads=16, kv_heads=16, dim=128),
        # Several system prompts of different popularity, grouped heads.
        dict(name="prefix 5 prompts grouped", op="prefix", groups=5, requests=80, prefix=12000, own=700, heads=32, kv_heads=8, dim=128),
        # A long document asked about by the engine's whole batch.
        dict(name="prefix 256 of a document", op="prefix", groups=1, requests=256, prefix=32768, own=100, heads=32, kv_heads=8, dim=128),
        # One interactive request: top-k then top-p, vocabulary 49152.
        dict(name="sample one row", op="sample", rows=1, vocab=49152, dtype="bf16", top_k=50, top_p=True, min_p=False),
        # The engine's mean width, top-k and top-p.
        dict(name="sample 80 rows top-k top-p", op="sample", rows=80, vocab=49152, dtype="bf16", top_k=200, top_p=True, min_p=False),
        # Rollouts at plain temperature, the larger vocabulary.
        dict(name="sample 256 rows plain", op="sample", rows=256, vocab=65536, dtype="bf16", top_k=0, top_p=False, min_p=False),
        # Logits that a program has worked on in 32 bits (penalties, bans): top-p alone over a wide row.
        dict(name="sample 256 rows fp32 top-p", op="sample", rows=256, vocab=49152, dtype="fp32", top_k=0, top_p=True, min_p=False),
        # An odd vocabulary with min-p, 32 bits.
        dict(name="sample 37 rows fp32 min-p", op="sample", rows=37, vocab=50257, dtype="fp32", top_k=0, top_p=False, min_p=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "prefix", "sample"])
    if op == "sample":
        rows = _log(rng, 1, 256)
        vocab = _log(rng, 100, min(131072, 256 * 49152 // rows))
        return dict(op=op, rows=rows, vocab=vocab, dtype=rng.choice(["bf16", "fp32"]), top_k=rng.choice([0, 0, 1, _log(rng, 2, 2000)]),
                    top_p=rng.random() < 0.5, min_p=rng.random() < 0.3)
    dim = rng.choice([64, 96, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 16, 55 if dim == 96 else 12])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 8] if kv_heads <= 8 else [1])
    if op == "norm":
        r = _log(rng, 1, 256)
        return dict(op=op, requests=r, max_ctx=_log(rng, 16, 256), max_new=_log(rng, 1, max(1, min(1024, 4096 // r))), heads=heads, kv_heads=kv_heads, dim=dim,
                    rope=rng.randint(0, 2))
    r = _log(rng, 1, 256)
    # at most what the largest listed case computes and what some of the others read
    prefix = _log(rng, 1, max(1, min(32768, 256 * 32768 * 32 * 128 // (r * heads * dim))))
    most = max(1, min(2000, 300_000_000 // (r * kv_heads * dim)))
    return dict(op=op, groups=rng.randint(1, min(r, 8)), requests=r, prefix=prefix, own=_log(rng, 1, most), heads=heads, kv_heads=kv_heads, dim=dim)


# ---------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _ints(g, lo, hi, n):
    return torch.randint(lo, hi + 1, (n,), generator=g, device=DEV, dtype=torch.int32)


def _pool(g, case, blocks):
    """Every row written, values of unit size."""

    return torch.randn(1, 2, blocks * BS, case["kv_heads"], case["dim"], generator=g, device=DEV, dtype=torch.bfloat16)


def prepare(case, seed):
    return {"norm": _prepare_norm, "prefix": _prepare_prefix, "sample": _prepare_sample}[case["op"]](case, _gen(seed))


def _norm_lengths(case):
    """Cached and new tokens of each request: the same for every seed, so that outputs keep their shapes."""

    r = case["requests"]
    fixed = _gen(r)
    ctx, new = _ints(fixed, 0, case["max_ctx"], r), _ints(fixed, 1, case["max_new"], r)
    if case["max_new"] > 1:
        ctx[::3] = 0  # fresh prompts among later chunks
        new[0] = case["max_new"]
    return ctx, new


def _prepare_norm(case, g):
    s = dict(case)
    hq, hkv, d = case["heads"], case["kv_heads"], case["dim"]
    ctx, new = _norm_lengths(case)
    order = torch.randperm(ctx.numel(), generator=g, device=DEV)
    ctx, new = ctx[order], new[order]
    pages = (ctx + new + BS - 1) // BS
    total, width = int(pages.sum()), int(pages.max()) + 1
    ids = torch.randperm(total, generator=g, device=DEV).int()
    first = (pages.cumsum(0) - pages).long()
    col = torch.arange(width, device=DEV)
    at = (first[:, None] + col).clamp(max=total - 1)
    s["table"] = torch.where(col < pages[:, None], ids[at], torch.full_like(ids[at], -1))
    req = torch.repeat_interleave(torch.arange(ctx.numel(), device=DEV), new.long())
    start = (new.cumsum(0) - new).long()
    s["slot"] = req.int()
    s["pos"] = (ctx.long()[req] + torch.arange(req.numel(), device=DEV) - start[req]).int()
    s["pool"] = _pool(g, case, total)
    s["qkv"] = torch.randn(req.numel(), (hq + 2 * hkv) * d, generator=g, device=DEV, dtype=torch.bfloat16)
    s["qkv"][::5] *= 6  # rows differ in size, which the norm takes out
    s["q_w"] = (1 + 0.2 * torch.randn(d, generator=g, device=DEV)).bfloat16()
    s["k_w"] = (1 + 0.2 * torch.randn(d, generator=g, device=DEV)).bfloat16()
    s["cos"], s["sin"] = None, None
    if case["rope"]:
        inv = 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device=DEV) / d)
        ang = torch.arange(width * BS, dtype=torch.float64, device=DEV)[:, None] * inv
        if case["rope"] == 1:  # bf16 [positions, dim], the two halves alike
            ang = torch.cat((ang, ang), -1)
            s["cos"], s["sin"] = ang.cos().bfloat16(), ang.sin().bfloat16()
        else:  # fp32 [positions, dim / 2]
            s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
    s["q_out"] = torch.empty(req.numel(), hq * d, device=DEV, dtype=torch.bfloat16)
    return s


def _groups(case):
    """Requests and shared tokens of each group and own tokens of each request, the same for every seed: the
    first prompt is the most popular one."""

    n, k = case["requests"], case["groups"]
    share = [1.0 / (i + 1) for i in range(k)]
    sizes = [max(1, int(n * x / sum(share))) for x in share]
    sizes[0] += n - sum(sizes)
    while sizes[0] < 1:
        j = max(range(k), key=lambda i: sizes[i])
        sizes[j] -= 1
        sizes[0] += 1
    prefix = [max(1, int(case["prefix"] * (1.0 if i == 0 else 0.3 + 0.7 * ((i * 37) % 11) / 11))) for i in range(k)]
    return sizes, prefix, _ints(_gen(n), 1, case["own"], n)


def _prepare_prefix(case, g):
    s = dict(case)
    hq, d, n = case["heads"], case["dim"], case["requests"]
    sizes, prefix, extra = _groups(case)
    s["sizes"], s["prefix_host"] = sizes, prefix  # a server's own book-keeping
    group = torch.repeat_interleave(torch.arange(len(sizes), device=DEV), torch.tensor(sizes, device=DEV))
    lens = torch.tensor(prefix, device=DEV)[group] + extra[torch.randperm(n, generator=g, device=DEV)]
    shared = torch.tensor([p // BS for p in prefix], device=DEV)  # whole pages are shared, a part-filled one is copied
    pages = (lens + BS - 1) // BS
    mine = pages - shared[group]
    total = int(shared.sum() + mine.sum())
    width = int(pages.max()) + 1
    ids = torch.randperm(total, generator=g, device=DEV).int()
    first_shared = (shared.cumsum(0) - shared)[group]
    first_own = int(shared.sum()) + mine.cumsum(0) - mine
    col = torch.arange(width, device=DEV)
    at = torch.where(col < shared[group][:, None], first_shared[:, None] + col, first_own[:, None] + col - shared[group][:, None])
    rows = torch.where(col < pages[:, None], ids[at.clamp(max=total - 1)], -1).int()
    slots = torch.randperm(n + 3, generator=g, device=DEV)[:n]  # resident slots, some of them idle
    s["table"] = torch.full((n + 3, width), -1, dtype=torch.int32, device=DEV)
    s["table"][slots] = rows
    s["slot"], s["pos"] = slots.int(), (lens - 1).int()
    s["pool"] = _pool(g, case, total)
    s["q"] = torch.randn(n, hq * d, generator=g, device=DEV, dtype=torch.bfloat16)
    s["out"] = torch.empty_like(s["q"])
    edges = [0]
    for k in sizes:
        edges.append(edges[-1] + k)
    s["group_start"] = torch.tensor(edges, dtype=torch.int32, device=DEV)
    s["prefix_len"] = torch.tensor(prefix, dtype=torch.int32, device=DEV)
    s["scale"] = d**-0.5
    s["own_max"] = case["own"] + BS  # own tokens and the copied part of a shared page, at most
    return s


def _prepare_sample(case, g):
    s = dict(case)
    n, v = case["rows"], case["vocab"]
    # a language model's rows: a wide body, a few dozen likely tokens, some rows surer than others
    x = torch.randn(n, v, generator=g, device=DEV) * 2.2
    top = torch.randint(0, v, (n, 40), generator=g, device=DEV)
    sure = 3 + 6 * torch.rand(n, 1, generator=g, device=DEV)
    x.scatter_add_(1, top, sure * torch.rand(n, 40, generator=g, device=DEV))
    x[::4].masked_fill_(torch.rand(x[::4].shape, generator=g, device=DEV) < 0.01, -math.inf)  # banned tokens
    s["logits"] = x.bfloat16() if case["dtype"] == "bf16" else x
    s["u"] = torch.rand(n, generator=g, device=DEV)
    s["temperature"] = 0.6 + 0.8 * torch.rand(n, generator=g, device=DEV)
    if n > 8:
        s["temperature"][3::16] = 0.0  # some requests ask for the likeliest token
    k = case["top_k"]
    s["k"] = _ints(g, max(1, k // 2), k, n) if k else None
    if k and n > 8:
        s["k"][5::16] = 0  # off in some rows
    s["p"] = 0.7 + 0.29 * torch.rand(n, generator=g, device=DEV) if case["top_p"] else None
    s["m"] = 0.01 + 0.1 * torch.rand(n, generator=g, device=DEV) if case["min_p"] else None
    s["ids"] = torch.empty(n, dtype=torch.int64, device=DEV)
    s["logp"] = torch.empty(n, device=DEV)
    return s


# ---------------------------------------------------------------- passes


def run(state):
    return {"norm": _norm, "prefix": _prefix, "sample": _sample}[state["op"]](state)


def _ops():
    import continuous_depth_batching_b200.ops  # noqa: F401  (registers torch.ops.cdb)

    return torch.ops.cdb


def _norm(s):
    if own:
        _ops().qk_norm_rope_append(s["qkv"], s["q_out"], s["pool"], 0, s["table"], s["slot"], s["pos"], s["q_w"], s["k_w"], s["cos"], s["sin"], s["rope"],
                                   s["heads"], EPS)
        return {"q": s["q_out"], "pool": s["pool"]}
    hq, hkv, d, t = s["heads"], s["kv_heads"], s["dim"], s["qkv"].shape[0]
    x = s["qkv"].float().view(t, hq + 2 * hkv, d)
    qk = x[:, : hq + hkv]
    w = torch.cat((s["q_w"].float().expand(hq, d), s["k_w"].float().expand(hkv, d)))
    qk = qk * torch.rsqrt((qk * qk).mean(-1, keepdim=True) + EPS) * w
    pos = s["pos"].long()
    if s["rope"]:
        c, sn = s["cos"][pos][:, None].float(), s["sin"][pos][:, None].float()
        if s["rope"] == 1:
            h = d // 2
            qk = qk * c + torch.cat((-qk[..., h:], qk[..., :h]), -1) * sn
        else:
            a, b = qk[..., 0::2], qk[..., 1::2]
            qk = torch.stack((a * c - b * sn, b * c + a * sn), -1).flatten(-2)
    s["q_out"].copy_(qk[:, :hq].reshape(t, -1))
    row = s["table"][s["slot"].long(), pos // BS].long() * BS + pos % BS
    s["pool"][0, 0, row] = qk[:, hq:].bfloat16()
    s["pool"][0, 1, row] = x[:, hq + hkv :].bfloat16()
    return {"q": s["q_out"], "pool": s["pool"]}


def _prefix(s):
    if own:
        _ops().prefix_decode_attention(s["q"], s["out"], s["pool"], 0, s["table"], s["slot"], s["pos"], s["group_start"], s["prefix_len"], s["heads"], s["scale"])
        return s["out"]
    hq, hkv, d = s["heads"], s["kv_heads"], s["dim"]
    cache = s["pool"][0].view(2, -1, BS, hkv, d)
    most = (s["own_max"] + BS - 1) // BS
    out, at = [], 0
    for size, prefix in zip(s["sizes"], s["prefix_host"]):
        pages = prefix // BS
        rows = s["table"][s["slot"][at : at + size].long()].long()
        last = s["pos"][at : at + size].long()
        q = s["q"][at : at + size].float().view(size, hkv, hq // hkv, d)
        # the shared pages once, every request's own pages beside them
        ks, vs = (cache[i][rows[0, :pages]].float().view(pages * BS, hkv, d) for i in range(2))
        ids = rows[:, pages : pages + most].clamp(min=0)
        ko, vo = (cache[i][ids].float().view(size, -1, hkv, d) for i in range(2))
        live = pages * BS + torch.arange(ko.shape[1], device=DEV) <= last[:, None]
        xs = torch.matmul(q.permute(1, 0, 2, 3).reshape(hkv, -1, d), ks.permute(1, 2, 0)).view(hkv, size, hq // hkv, pages * BS).transpose(0, 1) * s["scale"]
        xo = torch.matmul(q, ko.permute(0, 2, 3, 1)) * s["scale"]
        xo = xo.masked_fill(~live[:, None, None], -math.inf)
        m = xo.amax(-1, keepdim=True)
        if pages:
            m = torch.maximum(m, xs.amax(-1, keepdim=True))
        ps, po = torch.exp(xs - m), torch.exp(xo - m)
        o = torch.matmul(po, vo.transpose(1, 2))
        if pages:
            o = o + torch.matmul(ps.transpose(0, 1).reshape(hkv, -1, pages * BS), vs.transpose(0, 1)).view(hkv, size, hq // hkv, d).transpose(0, 1)
        out.append((o / (ps.sum(-1, keepdim=True) + po.sum(-1, keepdim=True))).reshape(size, -1).bfloat16())
        at += size
    return torch.cat(out)


def _sample(s):
    if own:
        _ops().sample_tokens(s["logits"], s["u"], s["temperature"], s["k"], s["p"], s["m"], s["ids"], s["logp"])
        return {"ids": s["ids"], "logp": s["logp"]}
    x = s["logits"].double()  # running sums next to a border want 64 bits
    n, v = x.shape
    top = x.amax(-1, keepdim=True)
    t = s["temperature"].double()[:, None]
    w = torch.where(t > 0, torch.exp((x - top) / t), (x == top).double())
    _, order = torch.sort(s["logits"], dim=-1, descending=True, stable=True)
    ranked = w.gather(1, order)
    rank = torch.arange(v, device=DEV)
    keep = torch.where(t > 0, torch.ones_like(ranked, dtype=torch.bool), rank < 1)
    if s["k"] is not None:
        k = s["k"].long()[:, None]
        keep &= (k <= 0) | (rank < k)
    ranked = ranked * keep
    if s["p"] is not None:
        before = ranked.cumsum(-1) - ranked
        keep &= (before < s["p"].double()[:, None] * ranked.sum(-1, keepdim=True)) | (rank < 1)
    if s["m"] is not None:
        keep &= (ranked >= s["m"].double()[:, None]) | (rank < 1)
    kept = torch.zeros_like(w).scatter_(1, order, ranked * keep)
    run_sum = kept.cumsum(-1)
    total = run_sum[:, -1:]
    ids = (run_sum <= s["u"].double()[:, None] * total).sum(-1)
    logp = torch.log(kept.gather(1, ids[:, None]) / total)[:, 0].float()
    return {"ids": ids, "logp": logp}


# ---------------------------------------------------------------- work and definition


def work(case):
    if case["op"] == "sample":
        size = 2 if case["dtype"] == "bf16" else 4
        # the logits once; a subtraction, an exponential and a sum a logit
        return {"bytes": case["rows"] * (case["vocab"] * size + 5 * 4 + 12), "flops": 3 * case["rows"] * case["vocab"]}
    hq, hkv, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "norm":
        rows = case["requests"] * (1 + case["max_new"]) / 2
        # q, k, v in, q and the cache's rows out
        return {"bytes": rows * d * 4 * (hq + 2 * hkv), "flops": rows * d * 7 * (hq + hkv)}
    sizes, prefix, _ = _groups(case)
    extra = case["requests"] * (1 + case["own"]) / 2
    keys = sum(n * p for n, p in zip(sizes, prefix)) + extra
    return {"bytes": (sum(prefix) + extra) * hkv * d * 4 + case["requests"] * hq * d * 4, "flops": 4 * keys * hq * d}


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "prefix": _exact_prefix, "sample": _exact_sample}[case["op"]](s)


def _exact_norm(s):
    hq, hkv, d, t = s["heads"], s["kv_heads"], s["dim"], s["qkv"].shape[0]
    x = s["qkv"].double().reshape(t, -1, d)
    pos = s["pos"].long()

    def head(y, weight):
        y = y / torch.sqrt(torch.einsum("thd,thd->th", y, y)[..., None] / d + EPS) * weight.double()
        if not s["rope"]:
            return y
        z = torch.empty_like(y)
        half = d // 2
        pair = [slice(0, half), slice(half, d)] if s["rope"] == 1 else [slice(0, d, 2), slice(1, d, 2)]
        c, sn = s["cos"].double()[pos][:, None, :half], s["sin"].double()[pos][:, None, :half]
        z[..., pair[0]] = y[..., pair[0]] * c - y[..., pair[1]] * sn
        z[..., pair[1]] = y[..., pair[0]] * sn + y[..., pair[1]] * c
        return z

    pool = s["pool"].double()
    block = torch.gather(s["table"].long()[s["slot"].long()], 1, torch.div(pos, BS, rounding_mode="floor")[:, None])[:, 0]
    row = block * BS + pos - torch.div(pos, BS, rounding_mode="floor") * BS
    pool[0, 0].index_copy_(0, row, head(x[:, hq : hq + hkv], s["k_w"]))
    pool[0, 1].index_copy_(0, row, x[:, hq + hkv :])
    return {"q": head(x[:, :hq], s["q_w"]).reshape(t, -1), "pool": pool}


def _exact_prefix(s):
    hq, hkv, d = s["heads"], s["kv_heads"], s["dim"]
    out = []
    for i, (slot, pos) in enumerate(zip(s["slot"].tolist(), s["pos"].tolist())):  # each request by itself, every key its own
        at = torch.arange(pos + 1, device=DEV)
        row = s["table"][slot].long()[at // BS] * BS + at % BS
        k, v = s["pool"][0, 0, row].double(), s["pool"][0, 1, row].double()
        x = torch.einsum("hgd,lhd->hgl", s["q"][i].double().view(hkv, hq // hkv, d), k) * s["scale"]
        out.append(torch.einsum("hgl,lhd->hgd", torch.softmax(x, -1), v).reshape(-1))
    return torch.stack(out)


def _exact_sample(s):
    ids, logp = [], []
    value = lambda name, i, off: off if s[name] is None else s[name][i].item()  # noqa: E731
    for i in range(s["rows"]):
        x = s["logits"][i].double()
        t, u = s["temperature"][i].item(), s["u"][i].item()
        if t <= 0:
            ids.append(int(torch.nonzero(x == x.max())[0]))
            logp.append(0.0)
            continue
        # by distinct logits, largest first: how many tokens have it, how many of them stay
        level, index, count = torch.unique(x, return_inverse=True, return_counts=True)
        level, count, index = level.flip(0), count.flip(0), level.numel() - 1 - index
        w = torch.exp((level - level[0]) / t)
        k = value("k", i, 0)
        stay = count if k <= 0 else (k - (count.cumsum(0) - count)).clamp(min=0).minimum(count)
        p = value("p", i, 1.0)
        if p < 1:
            mass = w * stay
            room = p * mass.sum() - (mass.cumsum(0) - mass)  # of the share, before each level
            stay = torch.ceil(room / w).nan_to_num(0.0, posinf=0.0).clamp(min=0).minimum(stay.double()).long()
            stay[0] = stay[0].clamp(min=1)
        m = value("m", i, 0.0)
        if m > 0:
            stay = torch.where(w >= min(m, 1.0), stay, 0)
        kept = stay[index] == count[index]
        part = torch.nonzero((stay > 0) & (stay < count))
        for level_at in part[:, 0].tolist():
            kept[torch.nonzero(index == level_at)[: int(stay[level_at]), 0]] = True
        token = torch.nonzero(kept)[:, 0]
        running = torch.cumsum(w[index[token]], 0)
        j = int(torch.searchsorted(running, u * running[-1], right=True))
        ids.append(int(token[j]))
        logp.append(float(torch.log(w[index[token[j]]] / running[-1])))
    return {"ids": torch.tensor(ids, device=DEV), "logp": torch.tensor(logp, dtype=torch.float64, device=DEV)}
