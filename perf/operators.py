"""Serving in 4 bits, as measurable cases: keys and values appended to a paged 4-bit cache, attention of one new token a
sequence over such a cache, and products with 4-bit weights.

A group of values is held as codes ``c`` of 4 bits with two bf16 numbers, ``value = m + s * c``: ``m`` the smallest value of
the group, ``s`` a fifteenth of its range.  The cache has a group for every 32 dims of a head, weights for every 64 or 128
rows of a column.  ``listed()`` names the cases, ``draw(rng)`` gives another one of the same ranges; ``prepare`` builds what a
program holds before the call, ``run`` is one pass, ``work`` what a pass cannot do without, ``exact`` the outputs in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

_CACHE_GROUP = 32


# ------------------------------------------------------------------------------------------
# Cases.
# ------------------------------------------------------------------------------------------


def listed() -> list:
    return [
        # One conversation at a small model's widths: launches and the chain length -> page -> key -> merge count.
        dict(name="attend 1 x 300", op="attend", batch=1, heads=16, kv=16, dim=128, tokens=300, page=16, ragged=False),
        # A served batch with grouped queries at the 8B widths, sequences of all ages.
        dict(name="attend 16 x 2048 grouped", op="attend", batch=16, heads=32, kv=8, dim=128, tokens=2048, page=16,
             ragged=True),
        # A full batch of a model with one query head per KV head: the cache's bytes.
        dict(name="attend 64 x 2000", op="attend", batch=64, heads=32, kv=32, dim=128, tokens=2000, page=16, ragged=False),
        # One long document, few heads: the cache is split along its length.
        dict(name="attend 1 x 130001 long", op="attend", batch=1, heads=32, kv=8, dim=128, tokens=130001, page=64,
             ragged=False),
        # A short prompt of a model with heads of 64.
        dict(name="append 1 x 333, dim 64", op="append", batch=1, tokens=333, kv=8, dim=64, page=16, start=0, ragged=False),
        # A decoding step's new tokens, every sequence at its own place.
        dict(name="append 64 x 1", op="append", batch=64, tokens=1, kv=32, dim=128, page=16, start=1000, ragged=True),
        # A batch of right-padded prompts.
        dict(name="append 8 x 2048", op="append", batch=8, tokens=2048, kv=8, dim=128, page=16, start=0, ragged=True),
        # Output projection of one token at the 1B widths: latency.
        dict(name="linear 1 x 2048 x 2048", op="linear", rows=1, k=2048, n=2048, group=128),
        # Gate and up projection of one token at the 8B widths.
        dict(name="linear 1 x 4096 x 28672", op="linear", rows=1, k=4096, n=28672, group=128),
        # Down projection of a batch of 16.
        dict(name="linear 16 x 14336 x 4096", op="linear", rows=16, k=14336, n=4096, group=128),
        # Gate and up projection of a batch of 64 at the 7B widths, finer groups.
        dict(name="linear 64 x 4096 x 22016", op="linear", rows=64, k=4096, n=22016, group=64),
        # A prompt's output projection: many rows.
        dict(name="linear 2048 x 4096 x 4096", op="linear", rows=2048, k=4096, n=4096, group=128),
    ]


def _log_uniform(rng, low: float, high: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng) -> dict:
    op = rng.choice(["attend", "append", "linear"])
    if op == "linear":
        rows, group = _log_uniform(rng, 1, 2048), rng.choice([64, 128])
        k, n = (8 * _log_uniform(rng, 32, 1792) for _ in range(2))
        while rows * k * n > 2048 * 4096 * 4096:
            rows = max(1, rows // 2)
        return dict(op=op, rows=rows, k=k, n=n, group=group)
    kv, dim = rng.choice([1, 2, 3, 4, 8, 16, 32]), rng.choice([64, 128])
    batch, page = _log_uniform(rng, 1, 64), rng.choice([8, 12, 16, 32, 64])
    if op == "append":
        tokens = 1 if rng.random() < 0.3 else _log_uniform(rng, 2, 2048)
        while batch * tokens * kv * dim > 8 * 2048 * 8 * 128:
            tokens = max(1, tokens // 2)
        return dict(op=op, batch=batch, tokens=tokens, kv=kv, dim=dim, page=page, start=rng.choice([0, _log_uniform(rng, 1, 900)]),
                    ragged=rng.random() < 0.6)
    tokens, group = _log_uniform(rng, 1, 60000), rng.choice([1, 1, 2, 3, 4, 6, 8, 12, 16])
    while batch * tokens * kv * dim * max(1, group / 4) > 64 * 2000 * 32 * 128:
        tokens = max(1, tokens // 2)
    return dict(op=op, batch=batch, heads=kv * group, kv=kv, dim=dim, tokens=tokens, page=page, ragged=rng.random() < 0.6)


def _counts(case: dict, most: int) -> list:
    """Tokens of every sequence: all ``most``, or the first that and the others spread over 1 to ``most``."""
    if not case["ragged"]:
        return [most] * case["batch"]
    return [most] + [1 + int((most - 1) * (0.618034 * i % 1.0)) for i in range(1, case["batch"])]


# ------------------------------------------------------------------------------------------
# The format, in plain operations.
# ------------------------------------------------------------------------------------------


def _quantize(x: torch.Tensor) -> tuple:
    """Groups along the last dim: codes (whole numbers), step and smallest value (bf16) of every group."""
    x = x.float()
    m = x.amin(-1).bfloat16()
    s = ((x.amax(-1) - m.float()) * (1.0 / 15.0)).bfloat16()
    s = torch.where(s < torch.finfo(torch.float32).tiny, torch.zeros_like(s), s)
    level = (x - m.float()[..., None]) / torch.where(s > 0, s.float(), torch.inf)[..., None]
    return level.round().clamp(0, 15).to(torch.uint8), s, m


def _pack_rows(c: torch.Tensor) -> torch.Tensor:
    """Codes of heads ``[..., H]`` as cache rows ``[..., H / 2]``: chunk r holds dims 4r .. 4r + 3 of every group of 32, group
    by group, the lower dim in the lower half of a byte."""
    h = c.shape[-1]
    x = c.reshape(*c.shape[:-1], h // 32, 8, 2, 2).movedim(-4, -3)
    return (x[..., 0] | (x[..., 1] << 4)).reshape(*c.shape[:-1], h // 2)


def _unpack_rows(b: torch.Tensor) -> torch.Tensor:
    h = 2 * b.shape[-1]
    x = torch.stack((b & 15, b >> 4), -1).reshape(*b.shape[:-1], 8, h // 32, 2, 2)
    return x.movedim(-4, -3).reshape(*b.shape[:-1], h)


def _cache_values(codes: torch.Tensor, scales: torch.Tensor, dtype) -> torch.Tensor:
    """Values of cache rows ``[..., H]``; ``scales [..., H / 32, 2]`` are (step, smallest)."""
    c = _unpack_rows(codes).to(dtype).unflatten(-1, (-1, _CACHE_GROUP))
    return (scales[..., 1, None].to(dtype) + scales[..., 0, None].to(dtype) * c).flatten(-2)


def _pack_weight(c: torch.Tensor) -> torch.Tensor:
    """Codes ``[N, K]`` (multiples of 16 and 64) as blocks ``[N / 16, K / 64, 512]``: bytes run over feature mod 8, k in
    sixteens, fours, singles, pairs, with feature + 8 in the upper half of a byte."""
    n, k = c.shape
    x = c.reshape(n // 16, 2, 8, k // 64, 4, 4, 2, 2)        # [N/16, half, r, K/64, c, j, pair, odd]
    x = x.permute(0, 3, 2, 4, 5, 7, 6, 1)                    # [N/16, K/64, r, c, j, odd, pair, half]
    return (x[..., 0] | (x[..., 1] << 4)).reshape(n // 16, k // 64, 512)


def _unpack_weight(b: torch.Tensor) -> torch.Tensor:
    n16, k64, _ = b.shape
    x = torch.stack((b & 15, b >> 4), -1).reshape(n16, k64, 8, 4, 4, 2, 2, 2)
    return x.permute(0, 7, 2, 1, 3, 4, 6, 5).reshape(n16 * 16, k64 * 64)


def _weight_values(state: dict, dtype) -> torch.Tensor:
    """``[K, N]``; ``scales [N / 16, groups, 8, 2, 2]`` run over feature mod 8, feature / 8, (step, smallest)."""
    scales = state["scales"].to(dtype)
    n16, groups = scales.shape[:2]
    s, m = scales.permute(0, 3, 2, 1, 4).reshape(n16 * 16, groups, 2).unbind(-1)
    c = _unpack_weight(state["codes"]).to(dtype)
    k = min(c.shape[1], groups * state["group"])
    s, m = (x.repeat_interleave(state["group"], 1)[:, :k] for x in (s, m))
    return (m + s * c[:, :k]).t()[:state["k"], :state["n"]]


# ------------------------------------------------------------------------------------------
# States.
# ------------------------------------------------------------------------------------------


def _generator(seed: int, salt: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed * 1000003 + salt)


def _normal(gen, *shape) -> torch.Tensor:
    return torch.randn(*shape, device="cuda", generator=gen)


def _heads_like(gen, rows: tuple, kv: int, dim: int, head_axis: int) -> torch.Tensor:
    """Keys or values: some channels of a head are larger than others, and not centred."""
    gain, mean = torch.exp(0.5 * _normal(gen, kv, dim)), 0.5 * _normal(gen, kv, dim)
    x = _normal(gen, *rows, dim)
    shape = [1] * x.dim()
    shape[head_axis], shape[-1] = kv, dim
    return (x * gain.reshape(shape) + mean.reshape(shape)).bfloat16()


def prepare(case: dict, seed: int) -> dict:
    gen = _generator(seed, 1)
    if case["op"] == "linear":
        k, n, group = case["k"], case["n"], case["group"]
        kp, np_ = -(-k // 128) * 128, -(-n // 16) * 16
        w = torch.zeros(np_, kp, device="cuda")
        w[:n, :k] = _normal(gen, n, k) * k ** -0.5
        c, s, m = _quantize(w.unflatten(1, (-1, group)))
        scales = torch.stack((s, m), -1).reshape(np_ // 16, 2, 8, kp // group, 2).permute(0, 3, 2, 1, 4).contiguous()
        x = (_normal(gen, case["rows"], k) * torch.exp(0.3 * _normal(gen, k))).bfloat16()
        return dict(op="linear", x=x, codes=_pack_weight(c.flatten(1)), scales=scales, k=k, n=n, group=group)
    b, kv, dim, page = case["batch"], case["kv"], case["dim"], case["page"]
    if case["op"] == "append":
        # A step's sequences stand at places of their own, prompts and chunks at one place and are of different lengths.
        start = _counts(case, case["start"]) if case["tokens"] == 1 and case["start"] else [case["start"]] * b
        live = [1] * b if case["tokens"] == 1 else _counts(case, case["tokens"])
        pages = -(-(case["start"] + case["tokens"]) // page)
    else:
        lengths = _counts(case, case["tokens"])
        pages = -(-case["tokens"] // page)
    table = torch.randperm(b * pages, device="cuda", generator=gen).to(torch.int32).reshape(b, pages)
    if case["op"] == "append":
        qkv = torch.cat([_heads_like(gen, (b, case["tokens"], kv), kv, dim, 2) for _ in range(2)], 2)
        empty = [(torch.zeros(b * pages, kv, page, dim // 2, dtype=torch.uint8, device="cuda"),
                  torch.zeros(b * pages, kv, page, dim // 32, 2, dtype=torch.bfloat16, device="cuda")) for _ in range(2)]
        return dict(op="append", k=qkv[:, :, :kv], v=qkv[:, :, kv:], k_pages=empty[0], v_pages=empty[1], table=table,
                    start=torch.tensor(start, dtype=torch.int32, device="cuda"),
                    live=torch.tensor(live, dtype=torch.int32, device="cuda"))
    pools = []
    for _ in range(2):
        c, s, m = _quantize(_heads_like(gen, (b * pages, kv, page), kv, dim, 1).unflatten(-1, (-1, _CACHE_GROUP)))
        pools.append((_pack_rows(c.flatten(-2)), torch.stack((s, m), -1)))
    q = _normal(gen, b, case["heads"], dim).bfloat16()
    return dict(op="attend", q=q, k_pages=pools[0], v_pages=pools[1], table=table,
                lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"))


# ------------------------------------------------------------------------------------------
# Passes.
# ------------------------------------------------------------------------------------------


def _attend(state: dict) -> torch.Tensor:
    q, table, lengths = state["q"], state["table"].long(), state["lengths"]
    b, heads, dim = q.shape
    k, v = (_cache_values(codes[table], scales[table], torch.float32).transpose(1, 2).flatten(2, 3)
            for codes, scales in (state["k_pages"], state["v_pages"]))           # [B, Nkv, S, H]
    qf = q.float().unflatten(1, (k.shape[1], -1))                                 # [B, Nkv, G, H]
    scores = qf @ k.transpose(2, 3) * dim ** -0.5
    seen = (torch.arange(k.shape[2], device=q.device) < lengths[:, None])[:, None, None]
    top = scores.masked_fill(~seen, -torch.inf).amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = torch.where(seen, torch.exp(scores - top), 0.0)
    out = p @ v / p.sum(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).tiny)
    return out.reshape(b, heads, dim).bfloat16()


def _places(state: dict) -> tuple:
    """Which tokens are appended ``[B, T]``, and their pages and rows there."""
    t = torch.arange(state["k"].shape[1], device="cuda")
    live = t < state["live"][:, None]
    pos = (state["start"][:, None] + t).long()
    page = state["k_pages"][0].shape[2]
    return live, state["table"].long().gather(1, (pos // page).clamp(max=state["table"].shape[1] - 1)), pos % page


def _append(state: dict) -> dict:
    live, pages, rows = _places(state)
    out = {}
    for name in ("k", "v"):
        x, (codes, scales) = state[name], state[name + "_pages"]
        c, s, m = _quantize(x.unflatten(-1, (-1, _CACHE_GROUP)))
        packed, pair = _pack_rows(c.flatten(-2)), torch.stack((s, m), -1)
        codes[pages[live], :, rows[live]] = packed[live]
        scales[pages[live], :, rows[live]] = pair[live]
        values = _cache_values(packed, pair, torch.float32).to(x.dtype)
        out[name] = torch.where(live[..., None, None], values, 0)
    return out


def run(state: dict):
    if own:
        from axlearn_b200.ops import int4_ops

        if state["op"] == "linear":
            w = int4_ops.Int4Weight(state["codes"], state["scales"], k=state["k"], n=state["n"], group=state["group"])
            return int4_ops.int4_linear(state["x"], w)
        k_pages, v_pages = int4_ops.Int4Pages(*state["k_pages"]), int4_ops.Int4Pages(*state["v_pages"])
        if state["op"] == "attend":
            return int4_ops.paged_decode_attention_int4(state["q"], k_pages, v_pages, state["table"], state["lengths"])
        k, v = int4_ops.append_int4(state["k"], state["v"], k_pages, v_pages, state["table"], state["start"],
                                    live=state["live"], values=True)
        return dict(k=k, v=v)
    if state["op"] == "linear":
        return (state["x"].float() @ _weight_values(state, torch.float32)).bfloat16()
    return _attend(state) if state["op"] == "attend" else _append(state)


def work(case: dict) -> dict:
    if case["op"] == "linear":
        rows, k, n = case["rows"], case["k"], case["n"]
        return {"bytes": k * n / 2 + 4 * n * -(-k // case["group"]) + 2 * rows * (k + n), "flops": 2 * rows * k * n}
    kv, dim = case["kv"], case["dim"]
    row = dim // 2 + dim // 8
    if case["op"] == "append":
        tokens = case["batch"] * case["tokens"]
        live = tokens if case["tokens"] == 1 else sum(_counts(case, case["tokens"]))
        return {"bytes": 2 * kv * (live * (2 * dim + row) + tokens * 2 * dim), "flops": 0}
    tokens = sum(_counts(case, case["tokens"]))
    return {"bytes": 2 * kv * row * tokens + 4 * case["batch"] * case["heads"] * dim, "flops": 4 * tokens * case["heads"] * dim}


# ------------------------------------------------------------------------------------------
# 64 bits.
# ------------------------------------------------------------------------------------------


def _rounded64(x: torch.Tensor) -> torch.Tensor:
    """The values that groups of 32 along the last dim are held as."""
    g = x.double().unflatten(-1, (-1, _CACHE_GROUP))
    low = g.min(-1, keepdim=True).values.bfloat16().double()
    step = ((g.max(-1, keepdim=True).values - low) / 15).bfloat16().double()
    level = torch.where(step > 0, torch.round((g - low) / torch.where(step > 0, step, 1.0)), 0.0)
    return (low + step * torch.clamp(level, 0, 15)).flatten(-2)


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    if case["op"] == "linear":
        scales, codes = state["scales"].double(), state["codes"]
        k, n, group = state["k"], state["n"], state["group"]
        y = torch.zeros(case["rows"], codes.shape[0] * 16, dtype=torch.float64, device="cuda")
        x = torch.zeros(case["rows"], codes.shape[1] * 64, dtype=torch.float64, device="cuda")
        x[:, :k] = state["x"].double()
        place = torch.arange(512, device="cuda")                    # byte of a block: feature mod 8, and its k
        feature, at = place // 64, place // 16 % 4 * 16 + place // 4 % 4 * 4 + place % 2 * 2 + place // 2 % 2
        for block in range(codes.shape[1]):
            w = torch.zeros(codes.shape[0], 16, 64, dtype=torch.float64, device="cuda")
            b = codes[:, block].long()
            w[:, feature, at], w[:, feature + 8, at] = (b % 16).double(), (b // 16).double()
            pair = scales[:, block * 64 // group].transpose(1, 2).reshape(-1, 16, 2)
            w = pair[..., 1:] + pair[..., :1] * w
            y += x[:, block * 64:block * 64 + 64] @ w.reshape(-1, 64).t()
        return y[:, :n]
    if case["op"] == "append":
        live = torch.arange(case["tokens"], device="cuda") < state["live"][:, None]
        return {name: _rounded64(state[name]) * live[..., None, None] for name in ("k", "v")}
    q, out = state["q"].double(), torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    dim, group = case["dim"], case["heads"] // case["kv"]
    place = torch.arange(dim, device="cuda")                        # dim: its byte of a row and its half
    byte = place % 32 // 4 * (dim // 16) + place // 32 * 2 + place % 4 // 2
    for i, length in enumerate(state["lengths"].tolist()):
        if not length:
            continue
        pages = state["table"][i, :-(-length // case["page"])].long()
        rows = []
        for codes, scales in (state["k_pages"], state["v_pages"]):
            c = codes[pages].transpose(0, 1).flatten(1, 2)[:, :length][..., byte].long() >> 4 * (place % 2) & 15
            pair = scales[pages].transpose(0, 1).flatten(1, 2)[:, :length].double()[:, :, place // 32]
            rows.append(pair[..., 1] + pair[..., 0] * c)
        scores = torch.einsum("kgd,ksd->kgs", q[i].reshape(-1, group, dim), rows[0]) / math.sqrt(dim)
        out[i] = torch.einsum("kgs,ksd->kgd", torch.softmax(scores, -1), rows[1]).reshape(-1, dim)
    return out
