"""Serving in 8 bits, as measurable cases: a norm whose output is held in 8 bits, products of 8-bit rows with 8-bit weights, keys
and values appended to a paged 8-bit cache, and attention of one new token a sequence over such a cache.

A block of values with the largest magnitude ``A`` is held as whole numbers ``c = round(127 x / A)`` of -127 to 127 and stands
for ``c A / 127``.  Rows of activations and columns of weights are blocks; in the cache a page's tokens of one KV head are one,
so that ``A`` grows while a page fills and the codes that are there follow it.  ``listed()`` names the cases, ``draw(rng)``
gives another one of the same ranges; ``prepare`` builds what a program holds before the call, ``run`` is one pass, ``work``
what a pass cannot do without, ``exact`` the outputs in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

_EPS = 1e-5


# ------------------------------------------------------------------------------------------
# Cases.
# ------------------------------------------------------------------------------------------


def listed() -> list:
    return [
        # One token at the 1B widths: launch and the row's sums.
        dict(name="norm 1 x 2048", op="norm", rows=1, dim=2048, residual=True),
        # A batch of prompts at the 7B and 8B widths: bytes.
        dict(name="norm 8192 x 4096", op="norm", rows=8192, dim=4096, residual=True),
        # Gate and up projection of one token at the 8B widths: the weight's bytes.
        dict(name="linear 1 x 4096 x 28672", op="linear", rows=1, k=4096, n=28672, held=True),
        # Down projection of a batch of 16 whose activations are still in 16 bits.
        dict(name="linear 16 x 14336 x 4096", op="linear", rows=16, k=14336, n=4096, held=False),
        # A short prompt at the 1B widths.
        dict(name="linear 333 x 2048 x 8192", op="linear", rows=333, k=2048, n=8192, held=True),
        # Gate and up projection of prompts at the 7B widths: the tensor cores.
        dict(name="linear 8192 x 4096 x 22016", op="linear", rows=8192, k=4096, n=22016, held=True),
        # A decoding step's new tokens, every sequence at its own place in a page.
        dict(name="append 64 x 1", op="append", batch=64, tokens=1, kv=32, dim=128, page=16, start=1000, ragged=True),
        # A batch of right-padded prompts.
        dict(name="append 8 x 2048", op="append", batch=8, tokens=2048, kv=8, dim=128, page=16, start=0, ragged=True),
        # One conversation at a small model's widths: launches and the chain length -> page -> key -> merge count.
        dict(name="attend 1 x 300", op="attend", batch=1, heads=16, kv=16, dim=128, tokens=300, page=16, ragged=False),
        # A served batch with grouped queries at the 8B widths, sequences of all ages.
        dict(name="attend 16 x 2048 grouped", op="attend", batch=16, heads=32, kv=8, dim=128, tokens=2048, page=16, ragged=True),
        # A full batch of a model with one query head per KV head: the cache's bytes.
        dict(name="attend 64 x 2000", op="attend", batch=64, heads=32, kv=32, dim=128, tokens=2000, page=16, ragged=False),
        # One long document, few heads: the cache is split along its length.
        dict(name="attend 1 x 130001 long", op="attend", batch=1, heads=32, kv=8, dim=128, tokens=130001, page=64, ragged=False),
    ]


def _log_uniform(rng, low: float, high: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng) -> dict:
    op = rng.choice(["norm", "linear", "append", "attend"])
    if op == "norm":
        rows, dim = _log_uniform(rng, 1, 8192), 8 * _log_uniform(rng, 32, 1024)
        while rows * dim > 8192 * 4096:
            rows = max(1, rows // 2)
        return dict(op=op, rows=rows, dim=dim, residual=rng.random() < 0.7)
    if op == "linear":
        rows, k, n = _log_uniform(rng, 1, 8192), 16 * _log_uniform(rng, 16, 1024), 8 * _log_uniform(rng, 32, 4096)
        while rows * k * n > 8192 * 4096 * 22016:
            rows = max(1, rows // 2)
        return dict(op=op, rows=rows, k=k, n=n, held=rng.random() < 0.6)
    kv, dim, page = rng.choice([1, 2, 3, 4, 8, 16, 32]), rng.choice([64, 128]), rng.choice([16, 16, 32, 48, 64, 128])
    batch = _log_uniform(rng, 1, 64)
    if op == "append":
        tokens = 1 if rng.random() < 0.4 else _log_uniform(rng, 2, 2048)
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


def _levels(x: torch.Tensor, top: torch.Tensor) -> torch.Tensor:
    """Codes of ``x`` (32 bits) under largest magnitudes ``top``, as fp32 whole numbers."""
    return (x * 127.0 / torch.where(top > 0, top, torch.inf)).round()


def _rows(x: torch.Tensor) -> tuple:
    """A block a row: codes (fp32 whole numbers) and scales."""
    top = x.abs().amax(-1, keepdim=True)
    return _levels(x, top), top / 127.0


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


def _hold_pages(x: torch.Tensor) -> tuple:
    """Pages ``[pages, Nkv, page, H]`` in 8 bits: codes, and the largest magnitudes ``[pages, Nkv]`` in bf16."""
    top = x.abs().amax((2, 3))
    return _levels(x.float(), top.float()[..., None, None]).to(torch.int8), top


def prepare(case: dict, seed: int) -> dict:
    gen, op = _generator(seed, 1), case["op"]
    if op == "norm":
        rows, dim = case["rows"], case["dim"]
        gain = torch.exp(0.5 * _normal(gen, dim))  # some channels of a residual stream are larger than others
        x = (_normal(gen, rows, dim) * gain).bfloat16()
        residual = (0.3 * _normal(gen, rows, dim)).bfloat16() if case["residual"] else None
        return dict(op=op, x=x, residual=residual, scale=(1 + 0.2 * _normal(gen, dim)).bfloat16())
    if op == "linear":
        rows, k, n = case["rows"], case["k"], case["n"]
        codes, scales = _rows(_normal(gen, n, k) * k ** -0.5)
        x = (_normal(gen, rows, k) * torch.exp(0.3 * _normal(gen, k))).bfloat16()
        state = dict(op=op, codes=codes.to(torch.int8), scales=scales[:, 0].contiguous())
        if not case["held"]:
            return dict(state, x=x)
        held, held_scales = _rows(x.float())
        return dict(state, x=None, x_codes=held.to(torch.int8), x_scales=held_scales[:, 0].contiguous())
    b, kv, dim, page = case["batch"], case["kv"], case["dim"], case["page"]
    if op == "attend":
        lengths = _counts(case, case["tokens"])
        pages = -(-case["tokens"] // page)
        table = torch.randperm(b * pages, device="cuda", generator=gen).to(torch.int32).reshape(b, pages)
        pools = [_hold_pages(_heads_like(gen, (b * pages, kv, page), kv, dim, 1)) for _ in range(2)]
        return dict(op=op, q=_normal(gen, b, case["heads"], dim).bfloat16(), k_pages=pools[0], v_pages=pools[1], table=table,
                    lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    # A step's sequences stand at places of their own, prompts and chunks at one place and are of different lengths.
    start = _counts(case, case["start"]) if case["tokens"] == 1 and case["start"] else [case["start"]] * b
    live = [1] * b if case["tokens"] == 1 else _counts(case, case["tokens"])
    pages = -(-(case["start"] + case["tokens"]) // page)
    table = torch.randperm(b * pages, device="cuda", generator=gen).to(torch.int32).reshape(b, pages)
    start = torch.tensor(start, dtype=torch.int32, device="cuda")
    qkv = torch.cat([_heads_like(gen, (b, case["tokens"], kv), kv, dim, 2) for _ in range(2)], 2)
    first = table.long().gather(1, (start // page).long()[:, None])[:, 0]  # holds the tokens of its sequence so far
    there = (torch.arange(page, device="cuda") < (start % page)[:, None])[:, None, :, None]
    state = dict(op=op, k=qkv[:, :, :kv], v=qkv[:, :, kv:], table=table, start=start,
                 live=torch.tensor(live, dtype=torch.int32, device="cuda"))
    for name in ("k_pages", "v_pages"):
        codes = torch.zeros(b * pages, kv, page, dim, dtype=torch.int8, device="cuda")
        tops = torch.zeros(b * pages, kv, dtype=torch.bfloat16, device="cuda")
        codes[first], tops[first] = _hold_pages(torch.where(there, _heads_like(gen, (b, kv, page), kv, dim, 1), 0))
        state[name] = (codes, tops)
    return state


# ------------------------------------------------------------------------------------------
# Passes.
# ------------------------------------------------------------------------------------------


def _norm(state: dict) -> dict:
    x = state["x"]
    if state["residual"] is not None:
        x = (x.float() + state["residual"].float()).bfloat16()
    t = x.float()
    y = t * torch.rsqrt((t * t).mean(-1, keepdim=True) + _EPS) * state["scale"].float()
    codes, scales = _rows(y)
    return dict(total=x, values=(codes * scales).bfloat16())


def _linear(state: dict) -> torch.Tensor:
    if state["x"] is not None:
        codes, scales = _rows(state["x"].float())
    else:
        codes, scales = state["x_codes"].float(), state["x_scales"][:, None]
    return (codes @ state["codes"].float().t() * scales * state["scales"]).bfloat16()


def _attend(state: dict) -> torch.Tensor:
    q, table, lengths = state["q"], state["table"].long(), state["lengths"]
    b, heads, dim = q.shape
    k, v = ((codes[table].float() * (tops[table].float() / 127.0)[..., None, None]).transpose(1, 2).flatten(2, 3)
            for codes, tops in (state["k_pages"], state["v_pages"]))             # [B, Nkv, S, H]
    qf = q.float().unflatten(1, (k.shape[1], -1))                                 # [B, Nkv, G, H]
    scores = qf @ k.transpose(2, 3) * dim ** -0.5
    seen = (torch.arange(k.shape[2], device=q.device) < lengths[:, None])[:, None, None]
    top = scores.masked_fill(~seen, -torch.inf).amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = torch.where(seen, torch.exp(scores - top), 0.0)
    out = p @ v / p.sum(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).tiny)
    return out.reshape(b, heads, dim).bfloat16()


def _append(state: dict) -> dict:
    table, start = state["table"].long(), state["start"].long()
    b, t, kv, dim = state["k"].shape
    page = state["k_pages"][0].shape[2]
    cols = table.shape[1]
    at = torch.arange(t, device="cuda")
    live = at < state["live"][:, None]
    pos = start[:, None] + at
    col = (pos // page).clamp(max=cols - 1)
    first = (start // page).clamp(max=cols - 1)[:, None]
    owner = table.gather(1, first)[:, 0]                                          # the page that a sequence goes on with
    before = (torch.arange(page, device="cuda") < (start % page)[:, None])[:, None, :, None]
    touched = torch.zeros(b, cols, dtype=torch.int32, device="cuda").scatter_add_(1, col, live.int()) > 0
    out = {}
    for name in ("k", "v"):
        x, (codes, tops) = state[name].float(), state[name + "_pages"]
        size = torch.where(live[..., None], x.abs().amax(-1), 0.0)                # [B, T, Nkv]
        top = torch.zeros(b, cols, kv, device="cuda")
        old = torch.where((start % page > 0)[:, None], tops[owner].float(), 0.0)  # of the tokens that are there
        top.scatter_(1, first[..., None].expand(b, 1, kv), old[:, None])
        top.scatter_reduce_(1, col[..., None].expand(b, t, kv), size, "amax")
        grown = top.gather(1, first[..., None].expand(b, 1, kv))[:, 0]            # [B, Nkv]
        held = codes[owner].float() * old[..., None, None] / torch.where(grown > 0, grown, torch.inf)[..., None, None]
        goes_on = (live[:, 0] & (start % page > 0))[:, None, None, None]
        codes[owner] = torch.where(goes_on & before, held.round().to(torch.int8), codes[owner])
        mine = top.gather(1, col[..., None].expand(b, t, kv))[..., None]
        new = _levels(x, mine)
        codes[table.gather(1, col)[live], :, (pos % page)[live]] = new.to(torch.int8)[live]
        tops[table[touched]] = top[touched].bfloat16()
        out[name] = torch.where(live[..., None, None], new * mine / 127.0, 0).bfloat16()
        out[name + "_tops"] = tops
    return out


def run(state: dict):
    if own:
        from axlearn_b200.ops import int8_ops

        if state["op"] == "norm":
            _, total, values = int8_ops.add_rms_norm_int8(state["x"], state["residual"], state["scale"], _EPS, values=True)
            return dict(total=total, values=values)
        if state["op"] == "linear":
            w = int8_ops.Int8Weight(state["codes"], state["scales"])
            x = state["x"] if state["x"] is not None else int8_ops.Int8Rows(state["x_codes"], state["x_scales"])
            return int8_ops.int8_linear(x, w)
        k_pages, v_pages = int8_ops.Int8Pages(*state["k_pages"]), int8_ops.Int8Pages(*state["v_pages"])
        if state["op"] == "attend":
            return int8_ops.paged_decode_attention_int8(state["q"], k_pages, v_pages, state["table"], state["lengths"])
        k, v = int8_ops.append_int8(state["k"], state["v"], k_pages, v_pages, state["table"], state["start"], live=state["live"],
                                    values=True)
        return dict(k=k, k_tops=k_pages.tops, v=v, v_tops=v_pages.tops)
    return {"norm": _norm, "linear": _linear, "attend": _attend, "append": _append}[state["op"]](state)


def work(case: dict) -> dict:
    if case["op"] == "norm":
        size = case["rows"] * case["dim"]
        return {"bytes": size * (8 if case["residual"] else 4) + 2 * case["dim"], "flops": 8 * size}
    if case["op"] == "linear":
        rows, k, n = case["rows"], case["k"], case["n"]
        return {"bytes": n * (k + 4) + rows * (k + 4 if case["held"] else 2 * k) + 2 * rows * n, "flops": 2 * rows * k * n}
    kv, dim, page = case["kv"], case["dim"], case["page"]
    if case["op"] == "append":
        tokens = case["batch"] * case["tokens"]
        live = [1] * tokens if case["tokens"] == 1 else _counts(case, case["tokens"])
        blocks = sum(-(-n // page) for n in live)
        return {"bytes": 2 * kv * (sum(live) * 3 * dim + tokens * 2 * dim + 4 * blocks), "flops": 0}
    lengths = _counts(case, case["tokens"])
    tokens, blocks = sum(lengths), sum(-(-n // page) for n in lengths)
    return {"bytes": 2 * kv * (dim * tokens + 2 * blocks) + 4 * case["batch"] * case["heads"] * dim,
            "flops": 4 * tokens * case["heads"] * dim}


# ------------------------------------------------------------------------------------------
# 64 bits.
# ------------------------------------------------------------------------------------------


def _held64(x: torch.Tensor) -> tuple:
    """Codes and largest magnitudes of rows, in 64 bits."""
    top = x.abs().max(-1, keepdim=True).values
    return torch.where(top > 0, torch.round(x * 127 / torch.where(top > 0, top, 1.0)), 0.0), top


def _append64(state: dict, name: str) -> tuple:
    """Values of the new tokens, and the largest magnitudes of all blocks behind the call."""
    x, (codes, tops) = state[name].double(), state[name + "_pages"]
    page, tops = codes.shape[2], tops.double().clone()
    out = torch.zeros_like(x)
    for i, (start, live) in enumerate(zip(state["start"].tolist(), state["live"].tolist())):
        done = 0
        while done < live:
            block = int(state["table"][i, (start + done) // page])
            row = (start + done) % page
            new = x[i, done:done + min(page - row, live - done)]
            top = new.abs().amax((0, 2))
            if row:
                top = torch.maximum(top, tops[block])
            tops[block] = top
            safe = torch.where(top > 0, top, 1.0)[:, None]
            out[i, done:done + len(new)] = torch.round(127 * new / safe) * top[:, None] / 127
            done += len(new)
    return out, tops


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    if case["op"] == "norm":
        total = state["x"]
        if state["residual"] is not None:
            total = (total.double() + state["residual"].double()).bfloat16()  # the stream itself is kept in 16 bits
        t = total.double()
        y = t / torch.sqrt(t.square().sum(-1, keepdim=True) / case["dim"] + _EPS) * state["scale"].double()
        codes, top = _held64(y)
        return dict(total=t, values=codes * top / 127)
    if case["op"] == "linear":
        if case["held"]:
            codes, scales = state["x_codes"].double(), state["x_scales"].double()[:, None]
        else:
            codes, top = _held64(state["x"].double())
            scales = top / 127
        return torch.einsum("mk,nk->mn", codes, state["codes"].double()) * (scales * state["scales"].double())
    if case["op"] == "append":
        (k, k_tops), (v, v_tops) = (_append64(state, name) for name in ("k", "v"))
        return dict(k=k, k_tops=k_tops, v=v, v_tops=v_tops)
    q, out = state["q"].double(), torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    dim, group = case["dim"], case["heads"] // case["kv"]
    for i, length in enumerate(state["lengths"].tolist()):
        pages = state["table"][i, :-(-length // case["page"])].long()
        rows = []
        for codes, tops in (state["k_pages"], state["v_pages"]):
            values = codes[pages].double() * tops[pages].double()[..., None, None] / 127
            rows.append(values.transpose(0, 1).flatten(1, 2)[:, :length])
        scores = torch.einsum("kgd,ksd->kgs", q[i].reshape(-1, group, dim), rows[0]) / math.sqrt(dim)
        out[i] = torch.einsum("kgs,ksd->kgd", torch.softmax(scores, -1), rows[1]).reshape(-1, dim)
    return out
