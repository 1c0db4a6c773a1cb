"""8-bit rows, weights and cache: the format, the plain statements and the refusals (no GPU)."""

import math
from fractions import Fraction

import pytest
import torch

from axlearn_b200.ops import int4_ops, int8_ops


def _values(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def _level(x: float, top: float, factor: int = 127) -> int:
    """The code of one value, in exact arithmetic (ties to even)."""
    return round(Fraction(x) * factor / Fraction(top)) if top else 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("dim", [8, 40, 256])
def test_rows_hold_the_nearest_level(dim, dtype):
    x = torch.cat([_values(4, dim) * s for s in (1, 1e-3, 300)]).to(dtype)
    x[1] = x[1].abs().amax() * torch.linspace(-1, 1, dim).to(dtype)  # many ties
    rows = int8_ops.quantize_rows(x)
    assert rows.codes.dtype == torch.int8 and rows.codes.shape == x.shape and rows.scales.shape == (12,)
    for row, codes, scale in zip(x.double().tolist(), rows.codes.tolist(), rows.scales.double().tolist()):
        top = max(abs(value) for value in row)
        assert codes == [_level(value, top) for value in row]
        assert abs(scale - top / 127) <= 2.0 ** -24 * top / 127
    # Half a level, and the rounding of the scale.
    error = (int8_ops.row_values(rows).double() - x.double()).abs()
    assert (error <= (0.5 + 127 * 2.0 ** -23) * rows.scales.double()[:, None]).all()


def test_rows_of_zeros_and_rows_that_are_not_finite():
    x = torch.zeros(6, 16)
    x[1, 3], x[2, 4], x[3, 5] = float("nan"), float("inf"), -float("inf")
    x[4] = 2.0 ** -120
    x[5, 1], x[5, 2] = 2.0 ** -119, -(2.0 ** -120)
    rows = int8_ops.quantize_rows(x)
    values = int8_ops.row_values(rows)
    assert not values[0].any() and values[1:4].isnan().all() and not rows.codes[:5].any() and not values[4].any()
    assert rows.codes[5].tolist()[:4] == [0, 127, -64, 0]  # -63.5 to the even number


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_norm_is_its_formula(residual, dtype):
    x, r, w = _values(5, 24, seed=1).to(dtype), _values(5, 24, seed=2).to(dtype), (1 + 0.2 * _values(24, seed=3)).to(dtype)
    rows, total, values = int8_ops.add_rms_norm_int8(x, r if residual else None, w, 1e-5, values=True)
    assert torch.equal(total, x + r if residual else x)
    y = total.double() / torch.sqrt(total.double().square().mean(-1, keepdim=True) + 1e-5) * w.double()
    top = y.abs().amax(-1, keepdim=True)
    # Half a level; in 32 bits a sum of 24 squares, its root and four products around it, one of them 127 times a level's size.
    slack = (24 + 8) * 2.0 ** -24
    assert ((int8_ops.row_values(rows).double() - y).abs() <= (0.5 + 127 * slack) * top / 127).all()
    assert torch.equal(values, int8_ops.row_values(rows, dtype)) and values.dtype == dtype
    assert len(int8_ops.add_rms_norm_int8(x, None, w, 1e-5)) == 2
    assert int8_ops.add_rms_norm_int8(x[:0], None, w, 1e-5)[0].codes.shape == (0, 24)


def test_swiglu_is_its_formula():
    gu = _values(3, 2, 32, seed=4) * 2
    rows = int8_ops.swiglu_int8(gu)
    gate, up = gu.double().chunk(2, -1)
    y = gate * torch.sigmoid(gate) * up
    top = y.abs().amax(-1, keepdim=True)
    assert rows.codes.shape == (3, 2, 16) and rows.scales.shape == (3, 2)
    assert ((int8_ops.row_values(rows).double() - y).abs() <= (0.5 + 127 * 2.0 ** -20) * top / 127).all()


def test_swiglu_of_gates_far_below_zero():
    gate = torch.linspace(-90, -79, 64).view(4, 16)
    up = torch.full((4, 16), 2.0 ** 20)
    up[1], up[2, 1::2] = 2.0 ** 100, -1
    rows = int8_ops.swiglu_int8(torch.cat([gate, up], 1))
    y = gate.double() * torch.sigmoid(gate.double()) * up.double()
    top = y.abs().amax(-1, keepdim=True)
    # Half a level; three products in 32 bits, and exponentials of a unit that are denormal from 2^-130 on (20 bits).
    assert rows.codes.any(1).all() and ((int8_ops.row_values(rows).double() - y).abs() <= (0.5 + 127 * 2.0 ** -18) * top / 127).all()
    gu = torch.tensor([[-float("inf"), 1.0] * 8, [float("inf"), 1.0] * 8, [-200.0] * 16, [0.0, -0.0] * 8])
    rows = int8_ops.swiglu_int8(torch.cat([gu, torch.ones_like(gu)], 1))
    assert rows.scales[:2].isnan().all() and not rows.codes.any() and not rows.scales[2:].any()


@pytest.mark.parametrize("k,n", [(16, 8), (48, 24), (272, 40)])
def test_linear_is_the_product_of_what_both_stand_for(k, n):
    w = int8_ops.quantize_weight(_values(k, n, seed=5) * 0.1)
    assert w.shape == (k, n)
    x = _values(2, 3, k, seed=6)
    rows = int8_ops.quantize_rows(x)
    want = int8_ops.row_values(rows).double() @ int8_ops.dequantize_weight(w, torch.float32).double()
    # Integer sums; they, two scales' products and values held in 32 bits for the comparison: ten roundings of sums of magnitudes.
    bound = 10 * 2.0 ** -24 * (int8_ops.row_values(rows).double().abs() @ int8_ops.dequantize_weight(w, torch.float32).double().abs())
    got = int8_ops.int8_linear(x, w)
    assert got.shape == (2, 3, n) and got.dtype == torch.float32 and ((got - want).abs() <= bound).all()
    assert torch.equal(int8_ops.int8_linear(rows, w, dtype=torch.float32), got)
    assert int8_ops.int8_linear(rows, w).dtype == torch.bfloat16
    out = torch.ones(2, 3, n)
    assert int8_ops.int8_linear(rows, w, out=out, accumulate=True) is out
    assert ((out - 1 - want).abs() <= bound + 2.0 ** -23 * (1 + want.abs())).all()
    assert int8_ops.int8_linear(x[:0], w).shape == (0, 3, n)
    square = int8_ops.quantize_weight(_values(48, 48, seed=7))
    x = _values(3, 48, seed=8)
    want = int8_ops.int8_linear(x, square)
    assert torch.equal(int8_ops.int8_linear(x, square, out=x), want)


def _cache(b, max_pages, page_size, kv, dim, seed=0, spare=2):
    gen = torch.Generator().manual_seed(seed)
    pools = [int8_ops.int8_pages(b * max_pages + spare, page_size, kv, dim) for _ in range(2)]
    table = torch.randperm(b * max_pages + spare, generator=gen)[:b * max_pages].to(torch.int32).reshape(b, max_pages)
    return pools[0], pools[1], table


def _append_loop(x, codes, tops, table, start, live):
    """One pool's append, block by block, in exact arithmetic; returns the values of the new tokens."""
    page_size, out = codes.shape[2], torch.zeros_like(x)
    for b, (first, count) in enumerate(zip(start, live)):
        done = 0
        while done < count:
            page, row = int(table[b, (first + done) // page_size]), (first + done) % page_size
            new = x[b, done:done + min(page_size - row, count - done)]
            for head in range(x.shape[2]):
                old = float(tops[page, head]) if row else 0.0
                top = max(old, float(new[:, head].abs().max()))
                if row and top != old:
                    turned = [[_level(int(c) * old, top, 1) for c in line] for line in codes[page, head, :row].tolist()]
                    codes[page, head, :row] = torch.tensor(turned, dtype=torch.int8)
                held = torch.tensor([[_level(v, top) for v in line] for line in new[:, head].double().tolist()])
                codes[page, head, row:row + len(new)] = held.to(torch.int8)
                tops[page, head] = top
                out[b, done:done + len(new), head] = (held.double() * top / 127).to(x.dtype)
            done += len(new)
    return out


@pytest.mark.parametrize("dim,page_size", [(64, 16), (128, 32)])
def test_append_is_its_definition_and_writes_nothing_else(dim, page_size):
    b, kv = 4, 2
    k_pages, v_pages, table = _cache(b, 4, page_size, kv, dim)
    for pages in (k_pages, v_pages):
        pages.codes.random_(-127, 128)
        pages.tops.uniform_(0.5, 2)
    calls = [([0, 0, 0, 0], [page_size + 3, 5, 0, 1], 2 * page_size), ([page_size + 3, 5, 0, 1], [7, 1, 4, 0], 7),
             ([page_size + 10, 6, 4, 1], [1, 1, 1, 1], 1), ([page_size + 11, 7, 5, 2], [1, 1, 1, 1], 1)]
    for i, (start, live, t) in enumerate(calls):
        k, v = (_values(b, t, kv, dim, seed=10 * i + s).mul(1 + i).bfloat16() for s in (5, 6))
        want = [(x.codes.clone(), x.tops.clone()) for x in (k_pages, v_pages)]
        values = [_append_loop(x, *held, table, start, live) for x, held in zip((k, v), want)]
        got = int8_ops.append_int8(k, v, k_pages, v_pages, table, torch.tensor(start, dtype=torch.int32),
                                   live=torch.tensor(live, dtype=torch.int32), values=True)
        for pages, (codes, tops), x, y in zip((k_pages, v_pages), want, got, values):
            assert torch.equal(pages.codes, codes) and torch.equal(pages.tops, tops) and torch.equal(x, y)


def test_a_page_that_grows_keeps_its_tokens_within_its_roundings():
    k_pages, v_pages, table = _cache(1, 1, 16, 1, 64)
    tokens = _values(16, 64, seed=9).bfloat16() * torch.linspace(0.2, 3, 16).bfloat16()[:, None]  # growing all the time
    for t in range(16):
        x = tokens[t][None, None, None]
        int8_ops.append_int8(x, x, k_pages, v_pages, table, torch.tensor([t], dtype=torch.int32))
    top = tokens.float().abs().amax()
    assert k_pages.tops[table[0, 0], 0] == top
    held = int8_ops.page_values(k_pages)[table[0, 0].long(), 0]
    tops = torch.cummax(tokens.float().abs().amax(-1), 0).values
    for t in range(16):
        grown = [float(tops[t])] + [float(a) for a, b in zip(tops[t + 1:], tops[t:]) if a > b]
        assert (held[t] - tokens[t].float()).abs().max() <= sum(0.5 * a / 127 for a in grown) * (1 + 2.0 ** -20)


@pytest.mark.parametrize("old,new", [(2.0 ** 121, 1.5 * 2.0 ** 121), (2.0 ** 122, 2.0 ** 124), (2.0 ** 126, 1.9921875 * 2.0 ** 127),
                                     (2.0 ** -119, 2.0 ** 127), (2.0 ** -119, 1.0078125 * 2.0 ** -119), (2.0 ** -119, 2.0 ** -118)])
def test_pages_at_the_ends_of_the_range(old, new):
    """Codes, magnitudes and what they stand for, of a page that goes on and of a new one."""
    k_pages, v_pages, table = _cache(1, 2, 16, 1, 128)
    for pages in (k_pages, v_pages):
        pages.codes[:, :, :5] = torch.randint(-127, 128, (1, 1, 5, 128), generator=torch.Generator().manual_seed(3), dtype=torch.int8)
        pages.tops.fill_(old)
    x = _values(1, 20, 1, 128, seed=13)
    x = (x / x.abs().amax(-1, keepdim=True) * new).bfloat16()
    want = [(p.codes.clone(), p.tops.clone()) for p in (k_pages, v_pages)]
    values = [_append_loop(y, *held, table, [5], [20]) for y, held in zip((x, -x), want)]
    got = int8_ops.append_int8(x, -x, k_pages, v_pages, table, torch.tensor([5], dtype=torch.int32), values=True)
    for pages, (codes, tops), y, z in zip((k_pages, v_pages), want, got, values):
        assert torch.equal(pages.codes, codes) and torch.equal(pages.tops, tops) and torch.equal(y, z) and y.isfinite().all()
        exact = codes.double() * tops.double()[..., None, None] / 127
        # A product of 15 bits, which is exact, and a quotient in 32.
        assert ((int8_ops.page_values(pages).double() - exact).abs() <= 2.0 ** -24 * exact.abs()).all()


def test_blocks_that_are_not_finite_and_blocks_of_zeros():
    k_pages, v_pages, table = _cache(1, 2, 16, 2, 64)
    page = int(table[0, 0])
    x = _values(1, 5, 2, 64, seed=10).bfloat16()
    x[0, 2, 1, 7] = float("inf")
    y = torch.zeros_like(x)
    k, v = int8_ops.append_int8(x, y, k_pages, v_pages, table, torch.zeros(1, dtype=torch.int32), values=True)
    assert k[:, :, 1].isnan().all() and not k[:, :, 0].isnan().any() and not v.any()
    assert k_pages.tops[page, 1].isnan() and v_pages.tops[page].tolist() == [0, 0]
    x = _values(1, 1, 2, 64, seed=11).bfloat16()
    k, v = int8_ops.append_int8(x, x, k_pages, v_pages, table, torch.tensor([5], dtype=torch.int32), values=True)
    assert k[:, :, 1].isnan().all() and not k[:, :, 0].isnan().any() and not v.isnan().any()
    assert not int8_ops.page_values(v_pages)[page, :, :5].any()
    # The first token of a page starts it anew.
    int8_ops.append_int8(x, x, k_pages, v_pages, table, torch.tensor([0], dtype=torch.int32))
    assert torch.equal(k_pages.tops[page], x.abs().amax(-1)[0, 0])


def test_places_that_are_not_there():
    k_pages, v_pages, table = _cache(2, 2, 16, 1, 64, spare=0)
    x = _values(2, 3, 1, 64, seed=12).bfloat16()
    for start, live in (([30, 0], [3, 3]), ([-1, 0], [1, 3]), ([2 ** 31 - 2, 0], [3, 3])):
        before = k_pages.codes.clone()
        with pytest.raises(IndexError):
            int8_ops.append_int8(x, x, k_pages, v_pages, table, torch.tensor(start, dtype=torch.int32),
                                 live=torch.tensor(live, dtype=torch.int32))
        assert torch.equal(before, k_pages.codes)
    bad = table.clone()
    bad[1, 0] = 4
    with pytest.raises(IndexError):
        int8_ops.append_int8(x, x, k_pages, v_pages, bad, torch.zeros(2, dtype=torch.int32))
    none = torch.zeros(2, 0, dtype=torch.int32)
    with pytest.raises(IndexError):
        int8_ops.append_int8(x, x, k_pages, v_pages, none, torch.zeros(2, dtype=torch.int32))
    int8_ops.append_int8(x, x, k_pages, v_pages, none, torch.zeros(2, dtype=torch.int32), live=torch.zeros(2, dtype=torch.int32))
    q = _values(2, 1, 64)
    for lengths in ([33, 1], [0, 17]):
        with pytest.raises(IndexError):
            int8_ops.paged_decode_attention_int8(q, k_pages, v_pages, torch.tensor([[0, 1], [1, 9]], dtype=torch.int32),
                                                 torch.tensor(lengths, dtype=torch.int32))


def _fill(pages, seed):
    gen = torch.Generator().manual_seed(seed)
    pages.codes.copy_(torch.randint(-127, 128, pages.codes.shape, generator=gen))
    pages.tops.copy_(0.5 + 2 * torch.rand(pages.tops.shape, generator=gen))


@pytest.mark.parametrize("heads,kv,dim", [(4, 4, 64), (6, 2, 128)])
def test_attention_over_the_cache_matches_a_loop(heads, kv, dim):
    k_pages, v_pages, table = _cache(3, 3, 16, kv, dim)
    _fill(k_pages, 1), _fill(v_pages, 2)
    lengths = torch.tensor([0, 17, 48], dtype=torch.int32)
    q = _values(3, heads, dim, seed=7)
    got = int8_ops.paged_decode_attention_int8(q, k_pages, v_pages, table, lengths, softmax_scale=0.05)
    assert not got[0].any()
    k, v = (int8_ops.page_values(p, torch.float64) for p in (k_pages, v_pages))
    for b in range(1, 3):
        for head in range(heads):
            rows = [(int(table[b, t // 16]), head // (heads // kv), t % 16) for t in range(int(lengths[b]))]
            scores = torch.stack([k[i] @ q[b, head].double() for i in rows]) * 0.05
            want = torch.softmax(scores, 0) @ torch.stack([v[i] for i in rows])
            # 128 products a score of up to 12: 130 * 2^-24 * 12 in the exponent, as much again in both sums; values up to 2.5.
            assert (got[b, head] - want).abs().max() <= 4 * 130 * 12 * 2.0 ** -24 * 2.5
    poisoned = [int8_ops.Int8Pages(p.codes.clone(), p.tops.clone()) for p in (k_pages, v_pages)]
    for p in poisoned:
        used = torch.cat([table[1, :2], table[2]]).long()
        others = torch.ones(len(p.tops), dtype=torch.bool)
        others[used] = False
        p.tops[others] = float("nan")
    assert torch.equal(int8_ops.paged_decode_attention_int8(q, *poisoned, table, lengths, softmax_scale=0.05), got)


def test_a_decoding_step_is_rotation_append_and_attention():
    b, nq, kv, dim = 3, 4, 2, 64
    k_pages, v_pages, table = _cache(b, 2, 16, kv, dim)
    _fill(k_pages, 3), _fill(v_pages, 4)
    rope = _values(32, dim // 2, 2, seed=5)
    lengths = torch.tensor([1, 20, 0], dtype=torch.int32)
    qkv = _values(b, (nq + 2 * kv) * dim, seed=6)
    pools = [int8_ops.Int8Pages(p.codes.clone(), p.tops.clone()) for p in (k_pages, v_pages)]
    got = int8_ops.rope_decode_attention_int8(qkv, k_pages, v_pages, table, lengths, rope, num_q_heads=nq, softmax_scale=0.1)
    q, k, v = qkv.view(b, 1, -1, dim).split((nq, kv, kv), 2)
    pos = (lengths[:, None] - 1).long()
    q, k = (int4_ops._rotate(x, rope, pos) for x in (q, k))  # pylint: disable=protected-access
    int8_ops.append_int8(k, v, *pools, table, lengths - 1, live=(lengths > 0).to(torch.int32))
    want = int8_ops.paged_decode_attention_int8(q[:, 0], *pools, table, lengths, softmax_scale=0.1)
    assert torch.equal(got, want) and not got[2].any()
    for p, w in zip((k_pages, v_pages), pools):
        assert torch.equal(p.codes, w.codes) and torch.equal(p.tops, w.tops)
    before = k_pages.codes.clone()
    with pytest.raises(IndexError):
        int8_ops.rope_decode_attention_int8(qkv, k_pages, v_pages, table, torch.tensor([1, 33, 1], dtype=torch.int32), rope,
                                            num_q_heads=nq, softmax_scale=0.1)
    assert torch.equal(before, k_pages.codes)


@pytest.mark.parametrize("live", [None, [20, 3]])
def test_prompts_attend_to_what_the_cache_stands_for(live):
    b, t, nq, kv, dim = 2, 20, 4, 2, 64
    k_pages, v_pages, table = _cache(b, 2, 16, kv, dim)
    rope = _values(32, dim // 2, 2, seed=5)
    qkv = _values(b, t, (nq + 2 * kv) * dim, seed=6)
    given = qkv.clone()
    counts = None if live is None else torch.tensor(live, dtype=torch.int32)
    got = int8_ops.prompt_attention_int8(qkv, k_pages, v_pages, table, rope, num_q_heads=nq, softmax_scale=0.1, live=counts)
    q, k, v = qkv.view(b, t, -1, dim).split((nq, kv, kv), 2)
    for i in range(b):
        n = t if live is None else live[i]
        rows = torch.tensor([[int(table[i, p // 16]), p % 16] for p in range(n)])
        for x, pages in ((k, k_pages), (v, v_pages)):
            assert torch.equal(x[i, :n], int8_ops.page_values(pages)[rows[:, 0], :, rows[:, 1]])
            assert not x[i, n:].any()
        assert torch.equal(q[i], int4_ops._rotate(given.view(b, t, -1, dim)[i:i + 1, :, :nq], rope, torch.arange(t)[None])[0])  # pylint: disable=protected-access
    kf, vf = (x.double().repeat_interleave(nq // kv, 2) for x in (k, v))
    scores = torch.einsum("bqhd,bkhd->bhqk", q.double(), kf) * 0.1
    scores = scores.masked_fill(torch.ones(t, t).triu(1).bool(), -math.inf)
    want = torch.einsum("bhqk,bkhd->bqhd", torch.softmax(scores, -1), vf).reshape(b, t, -1)
    # As over the cache, with rotations by a table of numbers up to 4: scores up to 200.
    assert (got - want).abs().max() <= 4 * 130 * 200 * 2.0 ** -24 * 4


def _attend_args(**change):
    k_pages, v_pages, table = _cache(2, 2, 16, 2, 64)
    args = dict(q=_values(2, 4, 64), k_pages=k_pages, v_pages=v_pages, page_table=table, lengths=torch.tensor([3, 20], dtype=torch.int32))
    return {**args, **{name: f(args) for name, f in change.items()}}


@pytest.mark.parametrize("change", [
    dict(q=lambda a: a["q"][:, :3]), dict(q=lambda a: _values(2, 4, 128)), dict(lengths=lambda a: a["lengths"].long()),
    dict(lengths=lambda a: a["lengths"][:1]), dict(page_table=lambda a: a["page_table"].long()),
    dict(page_table=lambda a: a["page_table"][:1]), dict(page_table=lambda a: a["page_table"].t()),
    dict(k_pages=lambda a: int8_ops.Int8Pages(a["k_pages"].codes.float(), a["k_pages"].tops)),
    dict(k_pages=lambda a: int8_ops.Int8Pages(a["k_pages"].codes, a["k_pages"].tops.float())),
    dict(v_pages=lambda a: int8_ops.Int8Pages(a["v_pages"].codes[1:], a["v_pages"].tops[1:])),
    dict(v_pages=lambda a: int8_ops.Int8Pages(a["v_pages"].codes[:, :, ::2], a["v_pages"].tops)),
    dict(softmax_scale=lambda a: 0.0), dict(softmax_scale=lambda a: float("nan")), dict(softmax_scale=lambda a: 2.0 ** 20),
    dict(splits=lambda a: 0), dict(splits=lambda a: 1025),
    dict(out=lambda a: torch.zeros(2, 4, 32)), dict(out=lambda a: torch.zeros(2, 4, 64, dtype=torch.bfloat16)),
])
def test_attention_refuses(change):
    with pytest.raises(ValueError):
        int8_ops.paged_decode_attention_int8(**_attend_args(**change))


@pytest.mark.parametrize("change", [
    dict(v=lambda a: a["v"][:, :2]), dict(k=lambda a: a["k"][:, :, :1], v=lambda a: a["v"][:, :, :1]),
    dict(start=lambda a: a["start"].long()), dict(live=lambda a: torch.zeros(3, dtype=torch.int32)),
    dict(k=lambda a: a["k"][..., :32], v=lambda a: a["v"][..., :32]), dict(v_pages=lambda a: a["k_pages"]),
    dict(v_pages=lambda a: int8_ops.Int8Pages(a["v_pages"].codes, a["k_pages"].tops)),
])
def test_append_refuses(change):
    k_pages, v_pages, table = _cache(2, 2, 16, 2, 64)
    args = dict(k=_values(2, 3, 2, 64), v=_values(2, 3, 2, 64), k_pages=k_pages, v_pages=v_pages, page_table=table,
                start=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError):
        int8_ops.append_int8(**{**args, **{name: f(args) for name, f in change.items()}})


def test_sizes_and_types_that_are_refused():
    for dim in (4, 12, 65544):
        with pytest.raises(ValueError):
            int8_ops.quantize_rows(torch.zeros(2, dim))
    with pytest.raises(ValueError):
        int8_ops.swiglu_int8(torch.zeros(2, 24))
    x, w = torch.zeros(2, 16), torch.ones(16)
    for bad in (dict(scale=w[:8]), dict(residual=x[:1]), dict(residual=x.double())):
        with pytest.raises(ValueError):
            int8_ops.add_rms_norm_int8(**{**dict(x=x, residual=None, scale=w, eps=1e-5), **bad})
    for shape in ((8, 8), (24, 8), (16, 12), (16,)):
        with pytest.raises(ValueError):
            int8_ops.quantize_weight(torch.zeros(shape))
    with pytest.raises(ValueError):
        int8_ops.Int8Weight(torch.zeros(8, 16, dtype=torch.uint8), torch.zeros(8))
    with pytest.raises(ValueError):
        int8_ops.Int8Weight(torch.zeros(8, 16, dtype=torch.int8), torch.zeros(8).bfloat16())
    weight = int8_ops.quantize_weight(_values(16, 8))
    for call in (lambda: int8_ops.int8_linear(torch.zeros(2, 32), weight), lambda: int8_ops.int8_linear(x, weight, accumulate=True),
                 lambda: int8_ops.int8_linear(x, weight, out=torch.zeros(2, 16)), lambda: int8_ops.int8_linear(x, weight, out=torch.zeros(8, 2).t()),
                 lambda: int8_ops.int8_linear(int8_ops.Int8Rows(x.to(torch.int8), torch.zeros(2, 1)), weight),
                 lambda: int8_ops.int8_linear(int8_ops.Int8Rows(x, torch.zeros(2)), weight)):
        with pytest.raises(ValueError):
            call()
    for page_size, dim in ((8, 64), (24, 64), (0, 64), (16, 96)):
        with pytest.raises(ValueError):
            int8_ops.int8_pages(2, page_size, 1, dim)
    k_pages, v_pages, table = _cache(2, 2, 16, 2, 64)
    rope = torch.zeros(32, 32, 2)
    lengths = torch.ones(2, dtype=torch.int32)
    step = lambda qkv, rope: int8_ops.rope_decode_attention_int8(  # noqa: E731
        qkv, k_pages, v_pages, table, lengths, rope, num_q_heads=2, softmax_scale=0.1)
    for qkv, angles in ((torch.zeros(2, 1, 384), rope), (torch.zeros(2, 320), rope), (torch.zeros(2, 384), rope[:, :16]),
                        (torch.zeros(2, 384), rope[:0]), (torch.zeros(2, 384), rope.double())):
        with pytest.raises(ValueError):
            step(qkv, angles)
    with pytest.raises(ValueError):
        int8_ops.prompt_attention_int8(torch.zeros(2, 33, 384), k_pages, v_pages, table, rope, num_q_heads=2, softmax_scale=0.1)
    with pytest.raises(ValueError):
        int8_ops.prompt_attention_int8(torch.zeros(2, 3, 384), k_pages, v_pages, table, rope, num_q_heads=2, softmax_scale=0.1,
                                       live=torch.ones(2))


@pytest.mark.parametrize("scale", [0.0, -0.1, math.nan, math.inf, 2.0 ** 20])
def test_scales_that_are_refused_leave_the_cache_as_it_was(scale):
    k_pages, v_pages, table = _cache(2, 2, 16, 2, 64)
    _fill(k_pages, 1), _fill(v_pages, 2)
    kept = [x.clone() for x in (*k_pages, *v_pages)]
    rope, qkv = torch.zeros(32, 32, 2), _values(2, 3, 384)
    given = qkv.clone()
    with pytest.raises(ValueError, match="softmax_scale"):
        int8_ops.prompt_attention_int8(qkv, k_pages, v_pages, table, rope, num_q_heads=2, softmax_scale=scale)
    with pytest.raises(ValueError, match="softmax_scale"):
        int8_ops.rope_decode_attention_int8(qkv[:, 0].contiguous(), k_pages, v_pages, table, torch.ones(2, dtype=torch.int32), rope,
                                            num_q_heads=2, softmax_scale=scale)
    assert torch.equal(qkv, given) and all(torch.equal(x, y) for x, y in zip((*k_pages, *v_pages), kept))


def test_formats_of_the_environment(monkeypatch):
    from axlearn_b200.inference import decode_engine

    bits = decode_engine._bits  # pylint: disable=protected-access
    assert (bits("WEIGHT"), bits("CACHE")) == (16, 16)
    for value, want in (("weights", (8, 16)), ("cache", (16, 8)), ("weights,cache", (8, 8)), (" cache, weights ", (8, 8)), ("", (16, 16))):
        monkeypatch.setenv("AXB200_DECODE_INT8", value)
        assert (bits("WEIGHT"), bits("CACHE")) == want
    monkeypatch.setenv("AXB200_DECODE_CACHE_BITS", "8")
    with pytest.raises(ValueError, match="4 or 16.*AXB200_DECODE_INT8"):
        bits("CACHE")
    for value in ("4", "16"):
        monkeypatch.setenv("AXB200_DECODE_CACHE_BITS", value)
        assert bits("CACHE") == int(value)
    monkeypatch.setenv("AXB200_DECODE_INT8", "caches")
    with pytest.raises(ValueError, match="AXB200_DECODE_INT8"):
        bits("CACHE")


def _calls_with_operands():
    k_pages, v_pages, table = _cache(1, 2, 16, 1, 64)
    weight = int8_ops.quantize_weight(_values(16, 8))
    one = torch.ones(1, dtype=torch.int32)
    rope = torch.zeros(32, 32, 2)
    return [
        (lambda x: int8_ops.quantize_rows(x), _values(2, 16)),
        (lambda x: int8_ops.swiglu_int8(x), _values(2, 16)),
        (lambda x: int8_ops.add_rms_norm_int8(x, None, torch.ones(16), 1e-5), _values(2, 16)),
        (lambda x: int8_ops.add_rms_norm_int8(torch.ones(2, 16), None, x, 1e-5), _values(16)),
        (lambda x: int8_ops.int8_linear(x, weight), _values(2, 16)),
        (lambda x: int8_ops.append_int8(x, x, k_pages, v_pages, table, one), _values(1, 1, 1, 64)),
        (lambda x: int8_ops.paged_decode_attention_int8(x, k_pages, v_pages, table, one), _values(1, 1, 64)),
        (lambda x: int8_ops.rope_decode_attention_int8(x, k_pages, v_pages, table, one, rope, num_q_heads=1, softmax_scale=0.1),
         _values(1, 192)),
        (lambda x: int8_ops.prompt_attention_int8(x, k_pages, v_pages, table, rope, num_q_heads=1, softmax_scale=0.1),
         _values(1, 2, 192)),
    ]


@pytest.mark.parametrize("call", range(9))
def test_differentiated_operands_are_refused(call):
    f, x = _calls_with_operands()[call]
    with pytest.raises(ValueError, match="no gradient"):
        f(x.clone().requires_grad_())
    with torch.no_grad():
        f(x.clone().requires_grad_())
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(ValueError, match="no gradient"):
            f(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)))


def test_empty_calls():
    k_pages, v_pages, table = _cache(2, 2, 16, 2, 64)
    none, rope = torch.zeros(0, dtype=torch.int32), torch.zeros(32, 32, 2)
    assert int8_ops.quantize_rows(torch.zeros(0, 16)).codes.shape == (0, 16)
    assert int8_ops.swiglu_int8(torch.zeros(0, 16)).codes.shape == (0, 8)
    k, v = int8_ops.append_int8(torch.zeros(0, 3, 2, 64), torch.zeros(0, 3, 2, 64), k_pages, v_pages, table[:0], none, values=True)
    assert k.shape == v.shape == (0, 3, 2, 64)
    x = torch.zeros(2, 0, 2, 64)
    assert int8_ops.append_int8(x, x, k_pages, v_pages, table, torch.zeros(2, dtype=torch.int32), values=True)[0].shape == x.shape
    assert int8_ops.paged_decode_attention_int8(torch.zeros(0, 2, 64), k_pages, v_pages, table[:0], none).shape == (0, 2, 64)
    assert int8_ops.rope_decode_attention_int8(torch.zeros(0, 384), k_pages, v_pages, table[:0], none, rope, num_q_heads=2,
                                               softmax_scale=0.1).shape == (0, 2, 64)
    for shape in ((0, 3, 384), (2, 0, 384)):
        got = int8_ops.prompt_attention_int8(torch.zeros(shape), k_pages, v_pages, table[:shape[0]], rope, num_q_heads=2,
                                             softmax_scale=0.1)
        assert got.shape == shape[:2] + (128,)


def test_splits_have_keys_and_fit():
    for ctas in (1, 2, 3, 5, 8, 14, 16, 17, 40, 148, 600):
        for tokens in (1, 63, 64, 127, 128, 500, 4095, 4096, 8192, 8193, 8208, 12000, 16384, 60000, 2 ** 18 - 1, 2 ** 18, 10 ** 6):
            splits = int8_ops.attention_splits(1, ctas, 1, tokens)
            assert 1 <= splits <= int8_ops.MAX_SPLITS
            if splits <= 8:  # a cluster
                assert splits in (1, 2, 4, 8) and (splits == 1 or splits * 64 <= tokens)
                assert splits <= 2 or splits * ctas <= (6 if tokens > 8192 else 3) * 148
            else:            # twelve warps a split, a tile of 32 keys for each; a CTA an SM
                assert tokens > 8192 and (splits - 1) * 12 * 32 < tokens and splits * ctas <= 148
    assert [int8_ops.attention_splits(1, 1, 1, tokens) for tokens in (8192, 8208, 16384, 60000, 10 ** 6)] == [8, 22, 43, 48, 96]
    assert [int8_ops.attention_splits(1, 8, 4, tokens) for tokens in (300, 16384, 130048)] == [4, 16, 16]


@pytest.mark.parametrize("rows,k,n,few", [(96, 4096, 4096, True), (97, 4096, 4096, False), (128, 4096, 4096, False), (128, 4112, 4096, True),
                                          (129, 4112, 4096, False), (128, 4096, 74 * 128, False), (128, 4096, 74 * 128 + 8, True),
                                          (1, 16, 8, True), (129, 131072, 40000, False)])
def test_products_that_stream_the_weight(rows, k, n, few):
    """96 rows, and 128 where K is above 4096 or tiles of 128 columns are more than the 74 pairs of SMs."""
    assert int8_ops.few_rows(rows, k, n) is few


@pytest.mark.parametrize("rows,n,features", [
    (256, 74 * 128, 128), (256, 74 * 128 + 8, 256),      # one wave of narrow tiles, or two (1.24 of a wide one's time)
    (512, 37 * 128, 128), (512, 37 * 128 + 8, 256),
    (256, 74 * 256, 256), (256, 74 * 256 + 8, 128),      # two narrow waves for one wide one; three for two
    (333, 8192, 256), (8192, 22016, 256), (129, 8, 128),
])
def test_features_of_a_tile(rows, n, features):
    assert int8_ops.pair_features(rows, n) == features


@pytest.mark.parametrize("batch,kv,group,tokens", [(1, 16, 1, 300), (16, 8, 4, 2048), (64, 32, 1, 2000), (1, 8, 4, 130048), (0, 8, 1, 64),
                                                   (1, 1, 1, 1), (1, 1, 40, 10 ** 6)])
def test_splits_of_attention(batch, kv, group, tokens):
    splits = int8_ops.attention_splits(batch, kv, group, tokens)
    assert splits in (1, 2, 4, 8) or (splits > 8 and tokens > 8192)
    assert int8_ops.pair_features(129, 8) in (128, 256)
