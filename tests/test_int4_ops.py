"""4-bit weights and cache: the format, the plain statements and the refusals (no GPU)."""

import math

import pytest
import torch

from axlearn_b200.ops import int4_ops


def _values(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def _level(x: float, low: float, step: float) -> int:
    """The code of one value, by Python's own rounding (ties to even)."""
    return min(15, max(0, round((x - low) / step))) if step else 0


@pytest.mark.parametrize("group", [32, 64])
def test_groups_hold_the_nearest_level(group):
    x = torch.cat([_values(5, 3 * group) * s + o for s, o in ((1, 0), (1e-3, 7), (300, -900))]).bfloat16()
    codes, scales = int4_ops.quantize_groups(x, group)
    assert codes.shape == x.shape and scales.shape == (15, 3, 2) and scales.dtype == torch.bfloat16
    for row in range(15):
        for g in range(3):
            part = x[row, g * group:(g + 1) * group].double().tolist()
            step, low = scales[row, g].double().tolist()
            assert low == min(part)
            # A fifteenth of the range: to half a unit of bf16, and the range and its product with 1 / 15 in 32 bits.
            assert abs(step - (max(part) - low) / 15) <= (2.0 ** -8 + 2.0 ** -20) * (max(part) - low) / 15
            for value, code in zip(part, codes[row, g * group:(g + 1) * group].tolist()):
                assert code == _level(value, low, step)
    # Half a step, and what the rounding of the step leaves behind level 15: 15 * 2^-8 of a step; sums in 32 bits.
    step = scales[..., :1].double()
    error = (int4_ops.group_values(codes, scales).double() - x.double()).abs().unflatten(-1, (-1, group))
    assert (error <= step * (0.5 + 15 * 2.0 ** -8) + 2.0 ** -22 * x.double().abs().amax()).all()


def test_groups_without_a_range_and_groups_that_are_not_finite():
    x = torch.zeros(8, 32).bfloat16()
    x[1] = 3.25
    x[2, 4], x[3, 5], x[4, 6] = float("nan"), float("inf"), -float("inf")
    x[5, 0], x[5, 1] = 3e38, -3e38                    # the range overflows
    x[6] = torch.linspace(0, 1, 32).bfloat16() * 2.0 ** -126   # a step below the smallest normal number
    x[7, 31] = 15.0
    codes, scales = int4_ops.quantize_groups(x, 32)
    values = int4_ops.group_values(codes, scales)
    assert torch.equal(values[:2], x[:2].float()) and not codes[:6].any()
    assert values[2:6].isnan().all()
    assert (values[6] == 0).all() and not scales[6].any()
    assert torch.equal(values[7], x[7].float()) and codes[7, 31] == 15


@pytest.mark.parametrize("dim", [64, 128])
def test_rows_of_the_cache_are_in_the_documented_order(dim):
    codes = torch.randint(0, 16, (3, 5, dim), dtype=torch.uint8, generator=torch.Generator().manual_seed(1))
    rows = int4_ops._pack_rows(codes)  # pylint: disable=protected-access
    assert rows.shape == (3, 5, dim // 2) and torch.equal(int4_ops._unpack_rows(rows), codes)  # pylint: disable=protected-access
    groups = dim // 32
    for d in range(dim):
        g, chunk, rest = d // 32, d % 32 // 4, d % 4
        byte = rows[..., chunk * 2 * groups + 2 * g + rest // 2]
        assert torch.equal(byte >> 4 if rest % 2 else byte & 15, codes[..., d])


@pytest.mark.parametrize("k,n,group", [(8, 8, 64), (72, 24, 64), (128, 16, 128), (200, 40, 128), (384, 56, 64)])
def test_weights_hold_their_groups_and_keep_their_order(k, n, group):
    w = _values(k, n, seed=k) * 0.1
    q = int4_ops.quantize_weight(w, group=group)
    assert q.shape == (k, n) and q.codes.shape == (-(-n // 16), -(-k // 128) * 2, 512)
    got = int4_ops.dequantize_weight(q, torch.float32)
    assert got.shape == (k, n)
    for lo in range(0, k, group):
        part = torch.zeros(group, n)
        part[:min(group, k - lo)] = w[lo:lo + group]
        codes, scales = int4_ops.quantize_groups(part.t(), group)
        want = int4_ops.group_values(codes, scales).t()[:min(group, k - lo)]
        assert torch.equal(got[lo:lo + group], want)
    # One column and one row of a block by the documented places.
    column, row = n - 1, min(k - 1, 63)
    block = q.codes[column // 16, 0].view(8, 4, 4, 2, 2)[column % 8, row // 16, row % 16 // 4, row % 2, row % 4 // 2]
    code = int(block) >> 4 if column % 16 >= 8 else int(block) & 15
    step, low = q.scales[column // 16, 0, column % 8, column % 16 // 8].float().tolist()
    assert got[row, column].item() == pytest.approx(low + step * code, rel=1e-6)


def test_linear_matches_its_formula_and_adds_to_out():
    w = int4_ops.quantize_weight(_values(72, 24, seed=2), group=64)
    x = _values(2, 3, 72, seed=3)
    want = x.double() @ int4_ops.dequantize_weight(w, torch.float32).double()
    # 72 products and sums in 32 bits.
    bound = 74 * 2.0 ** -24 * (x.double().abs() @ int4_ops.dequantize_weight(w, torch.float32).double().abs())
    got = int4_ops.int4_linear(x, w)
    assert got.shape == (2, 3, 24) and ((got - want).abs() <= bound).all()
    out = torch.ones(2, 3, 24)
    assert int4_ops.int4_linear(x, w, out=out, accumulate=True) is out
    assert ((out - 1 - want).abs() <= bound + 2.0 ** -23 * (1 + want.abs())).all()
    assert int4_ops.int4_linear(x[:0], w).shape == (0, 3, 24)


def test_memory_that_tensors_have_in_common():
    x = torch.zeros(10, 16)
    for a, b, want in ((x, x, True), (x[:4], x[4:], False), (x[:4], x[3:], True), (x[:, :8], x[:, 8:], True),  # (spans, not rows)
                       (x[:0], x, False), (x[2], x.view(-1)[47:48], True), (x[2], x.view(-1)[48:49], False), (x, x.clone(), False)):
        assert int4_ops._overlap(a, b) == int4_ops._overlap(b, a) == want  # pylint: disable=protected-access


def test_products_and_attention_in_place():
    w, x = int4_ops.quantize_weight(_values(64, 64, seed=4)), _values(3, 64, seed=5)
    want = int4_ops.int4_linear(x, w)
    flat = torch.cat([torch.zeros(64), x.flatten()])
    assert torch.equal(int4_ops.int4_linear(flat[64:].view(3, 64), w, out=flat[:-64].view(3, 64)), want)
    assert torch.equal(int4_ops.int4_linear(x, w, out=x), want)
    args = _attend_args()
    want = int4_ops.paged_decode_attention_int4(**args)
    assert torch.equal(int4_ops.paged_decode_attention_int4(**args, out=args["q"]), want)


def _cache(b, max_pages, page_size, kv, dim, seed=0, spare=2):
    gen = torch.Generator().manual_seed(seed)
    pools = [int4_ops.int4_pages(b * max_pages + spare, page_size, kv, dim) for _ in range(2)]
    table = torch.randperm(b * max_pages + spare, generator=gen)[:b * max_pages].to(torch.int32).reshape(b, max_pages)
    return pools[0], pools[1], table


@pytest.mark.parametrize("dim,page_size", [(64, 5), (128, 16)])
def test_append_writes_live_tokens_and_nothing_else(dim, page_size):
    b, t, kv = 3, 7, 2
    k_pages, v_pages, table = _cache(b, 4, page_size, kv, dim)
    for pages in (k_pages, v_pages):
        pages.codes.random_(0, 255)
        pages.scales.normal_()
    before = [x.clone() for x in (*k_pages, *v_pages)]
    start, live = torch.tensor([0, 3, 9], dtype=torch.int32), torch.tensor([7, 0, 4], dtype=torch.int32)
    k, v = (_values(b, t, kv, dim, seed=s).bfloat16() for s in (5, 6))
    kv_values = int4_ops.append_int4(k, v, k_pages, v_pages, table, start, live=live, values=True)
    touched = torch.zeros(k_pages.codes.shape[0], page_size, dtype=torch.bool)
    for x, pages, got in zip((k, v), (k_pages, v_pages), kv_values):
        held = int4_ops.page_values(pages)
        for i in range(b):
            for j in range(t):
                if j >= live[i]:
                    assert not got[i, j].any()
                    continue
                pos = int(start[i]) + j
                page, row = int(table[i, pos // page_size]), pos % page_size
                touched[page, row] = True
                codes, scales = int4_ops.quantize_groups(x[i, j], 32)
                assert torch.equal(held[page, :, row], int4_ops.group_values(codes, scales))
                assert torch.equal(got[i, j], held[page, :, row].bfloat16())
    for old, new in zip(before, (*k_pages, *v_pages)):
        assert torch.equal(old.transpose(1, 2)[~touched], new.transpose(1, 2)[~touched])


def test_places_written_are_inside_the_pool():
    """What the plain append writes to on any device."""
    table = torch.tensor([[3, 9], [0, 6], [5, -1]], dtype=torch.int32)
    start, live = torch.tensor([2, 6, -1], dtype=torch.int32), torch.tensor([4, 3, 2], dtype=torch.int32)
    page, row, keep, inside = int4_ops._write_places(table, start, live, 4, 4, 7)  # pylint: disable=protected-access
    assert keep.tolist() == [[True] * 4, [True] * 3 + [False], [True] * 2 + [False] * 2]
    assert inside.tolist() == [[True, True, False, False], [True, True, False, False], [False, True, False, False]]
    assert page[inside].tolist() == [3, 3, 6, 6, 5] and row[inside].tolist() == [2, 3, 2, 3, 0]
    _, _, keep, inside = int4_ops._write_places(table[:, :0], start, None, 4, 4, 7)  # pylint: disable=protected-access
    assert keep.all() and not inside.any()


def test_append_refuses_a_table_without_pages():
    k_pages, v_pages, table = _cache(2, 3, 4, 2, 64)
    rows, start = _values(2, 1, 2, 64).bfloat16(), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(IndexError, match="page table"):
        int4_ops.append_int4(rows, rows, k_pages, v_pages, table[:, :0].contiguous(), start)
    int4_ops.append_int4(rows, rows, k_pages, v_pages, table[:, :0].contiguous(), start, live=start)


@pytest.mark.parametrize("heads,kv,dim", [(4, 4, 64), (6, 2, 128)])
def test_attention_over_the_cache_matches_a_loop(heads, kv, dim):
    b, page_size, lengths = 4, 6, [0, 1, 13, 18]
    k_pages, v_pages, table = _cache(b, 3, page_size, kv, dim, seed=7)
    k, v = (_values(b, 18, kv, dim, seed=s).bfloat16() for s in (8, 9))
    lens = torch.tensor(lengths, dtype=torch.int32)
    int4_ops.append_int4(k, v, k_pages, v_pages, table, torch.zeros(b, dtype=torch.int32), live=lens)
    k_pages.scales[table[2, 2].long(), :, 2:] = torch.nan  # behind the third sequence's last token
    q = _values(b, heads, dim, seed=10).bfloat16()
    out = int4_ops.paged_decode_attention_int4(q, k_pages, v_pages, table, lens)
    assert not out[0].any()
    kk, vv = int4_ops.page_values(k_pages, torch.float64), int4_ops.page_values(v_pages, torch.float64)
    for i in range(1, b):
        for h in range(heads):
            at = [(int(table[i, p // page_size]), h // (heads // kv), p % page_size) for p in range(lengths[i])]
            keys, vals = (torch.stack([x[j] for j in at]) for x in (kk, vv))
            p = torch.softmax(keys @ q[i, h].double() / math.sqrt(dim), 0)
            # The output's rounding, and a few hundred operations in 32 bits.
            assert ((out[i, h].double() - p @ vals).abs() <= 2.0 ** -8 * (p @ vals).abs() + 2.0 ** -14 * vals.abs().max()).all()


def test_places_read_are_those_of_the_sequences_alone():
    """What the plain attention gathers on any device: entries behind a sequence may be anything."""
    table = torch.tensor([[3, 10 ** 9, -7], [0, 6, 2 ** 31 - 1], [-2 ** 31, 7, 7], [1, 2, 3]], dtype=torch.int32)
    lengths = torch.tensor([4, 5, 0, -3], dtype=torch.int32)
    pages, seen, bad = int4_ops._read_places(table, lengths, 4, 7)  # pylint: disable=protected-access
    assert pages.tolist() == [[3, 0, 0], [0, 6, 0], [0, 0, 0], [0, 0, 0]] and not bad
    assert torch.equal(seen, torch.arange(12) < lengths[:, None])
    # A page that a sequence needs and the pool does not have, a length behind the table: no key of theirs, nothing outside.
    for row, page in ((0, 7), (1, -1)):
        wrong = table.clone()
        wrong[row, 0] = page
        pages, seen, bad = int4_ops._read_places(wrong, lengths, 4, 7)  # pylint: disable=protected-access
        assert bad and pages.min() >= 0 and pages.max() < 7 and not seen[row, :4].any()
    pages, seen, bad = int4_ops._read_places(table[3:], torch.tensor([13], dtype=torch.int32), 4, 7)  # pylint: disable=protected-access
    assert bad and pages.tolist() == [[1, 2, 3]] and seen.all()
    assert int4_ops._read_places(table[:, :0], lengths, 4, 7)[2]  # pylint: disable=protected-access


def test_attention_takes_tables_with_anything_behind_a_sequence():
    args = _attend_args(lengths=torch.tensor([3, 0], dtype=torch.int32))
    want = int4_ops.paged_decode_attention_int4(**args)
    args["page_table"][0, 1:], args["page_table"][1] = 10 ** 9, -7
    assert torch.equal(int4_ops.paged_decode_attention_int4(**args), want)


def test_a_decoding_step_is_rotation_append_and_attention():
    b, heads, kv, dim, page_size = 3, 4, 2, 64, 4
    k_pages, v_pages, table = _cache(b, 3, page_size, kv, dim, seed=11)
    past = [_values(b, 12, kv, dim, seed=s).bfloat16() for s in (12, 13)]
    lens = torch.tensor([0, 5, 12], dtype=torch.int32)
    int4_ops.append_int4(*past, k_pages, v_pages, table, torch.zeros(b, dtype=torch.int32), live=(lens - 1).clamp(min=0))
    angle = torch.arange(12)[:, None] * 0.3 ** torch.arange(dim // 2)
    rope = torch.stack((angle.sin(), angle.cos()), -1)
    qkv = _values(b, (heads + 2 * kv) * dim, seed=14).bfloat16()
    out = int4_ops.rope_decode_attention_int4(qkv, k_pages, v_pages, table, lens, rope, num_q_heads=heads, softmax_scale=0.1)
    q, k, v = qkv.view(b, -1, dim).split((heads, kv, kv), 1)

    def turned(x, pos):
        z = torch.view_as_complex(x.float().unflatten(-1, (-1, 2)).contiguous()) * torch.polar(torch.ones(dim // 2), angle[pos])
        return torch.view_as_real(z).flatten(-2).bfloat16()

    for i, n in ((1, 5), (2, 12)):
        page, row = int(table[i, (n - 1) // page_size]), (n - 1) % page_size
        for x, pages in ((turned(k[i], n - 1), k_pages), (v[i], v_pages)):
            codes, scales = int4_ops.quantize_groups(x, 32)
            assert torch.equal(int4_ops.page_values(pages)[page, :, row], int4_ops.group_values(codes, scales))
        want = int4_ops.paged_decode_attention_int4(turned(q[i], n - 1)[None], k_pages, v_pages, table[i:i + 1], lens[i:i + 1],
                                                    softmax_scale=0.1)
        assert torch.equal(out[i], want[0])
    assert not out[0].any()


def test_prompts_attend_to_what_the_cache_stands_for():
    b, t, heads, kv, dim = 2, 9, 4, 2, 64
    k_pages, v_pages, table = _cache(b, 3, 4, kv, dim, seed=15)
    angle = torch.arange(t)[:, None] * 0.5 ** torch.arange(dim // 2)
    rope = torch.stack((angle.sin(), angle.cos()), -1)
    qkv = _values(b, t, (heads + 2 * kv) * dim, seed=16).bfloat16()
    given = qkv.clone()
    out = int4_ops.prompt_attention_int4(qkv, k_pages, v_pages, table, rope, num_q_heads=heads, softmax_scale=0.2)
    step_pages = _cache(b, 3, 4, kv, dim, seed=15)
    for i in range(t):
        lens = torch.full((b,), i + 1, dtype=torch.int32)
        one = int4_ops.rope_decode_attention_int4(given[:, i].contiguous(), step_pages[0], step_pages[1], table, lens, rope,
                                                  num_q_heads=heads, softmax_scale=0.2)
        # The prompt reads values rounded to bf16: a score moves by up to 2^-8 of its terms, a probability by e^(2 move), a
        # value by 2^-8; then both outputs are rounded.
        terms = 0.2 * dim * qkv[:, i, :heads * dim].abs().max() * int4_ops.page_values(k_pages).abs().max()
        bound = (torch.expm1(2 * 2.0 ** -8 * terms) + 3 * 2.0 ** -8) * int4_ops.page_values(v_pages).abs().max()
        assert (one.flatten(1).float() - out[:, i].float()).abs().max() <= bound
    for x, y in zip((*k_pages, *v_pages), (*step_pages[0], *step_pages[1])):
        assert torch.equal(x, y)


def _attention64(q, k, v, scale):
    """One query ``[N, H]`` over ``k, v [S, Nkv, H]`` in 64 bits, and what 32-bit sums and the output's rounding to bf16 may add."""
    q, k, v = q.double(), k.double().transpose(0, 1), v.double().transpose(0, 1)
    qg = q.unflatten(0, (k.shape[0], -1))
    p = torch.softmax(qg @ k.transpose(1, 2) * scale, -1)
    out, size = p @ v, p @ v.abs()
    # A score: products of bf16 are exact, H sums and a factor, each 2^-24 of the terms; a probability moves by e^(2 move).  Then exp
    # and the division, a few 2^-24, and sums of S terms twice.
    move = (q.shape[1] + 2) * 2.0 ** -24 * scale * (qg.abs() @ k.abs().transpose(1, 2)).amax(-1, keepdim=True)
    bound = (torch.expm1(2 * move) + (2 * k.shape[1] + 16) * 2.0 ** -24) * size
    return out.flatten(0, 1), (1.01 * bound + 2.0 ** -8 * (out.abs() + bound)).flatten(0, 1)


@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (3, 1, 128)])
def test_prompts_and_steps_have_the_values_of_their_formula(heads, kv, dim):
    """Prompts attend to the cache's values rounded to bf16, steps to the values themselves; a token that is missing, or one too
    many, is far outside the bounds."""
    b, t, scale = 2, 11, 0.15
    k_pages, v_pages, table = _cache(b, 3, 4, kv, dim, seed=15)
    angle = torch.arange(t)[:, None] * 0.5 ** torch.arange(dim // 2)
    rope = torch.stack((angle.sin(), angle.cos()), -1)
    qkv = _values(b, t, (heads + 2 * kv) * dim, seed=16).bfloat16()
    given = qkv.clone()
    out = int4_ops.prompt_attention_int4(qkv, k_pages, v_pages, table, rope, num_q_heads=heads, softmax_scale=scale).unflatten(-1, (heads, dim))
    q, k, v = qkv.unflatten(-1, (-1, dim)).split((heads, kv, kv), 2)
    held = [int4_ops.page_values(p)[table.long()].transpose(2, 3).flatten(1, 2)[:, :t] for p in (k_pages, v_pages)]
    assert torch.equal(k, held[0].bfloat16()) and torch.equal(v, held[1].bfloat16())
    step_pages = _cache(b, 3, 4, kv, dim, seed=15)
    far = 0
    for i in range(t):
        lens = torch.full((b,), i + 1, dtype=torch.int32)
        one = int4_ops.rope_decode_attention_int4(given[:, i].contiguous(), step_pages[0], step_pages[1], table, lens, rope,
                                                  num_q_heads=heads, softmax_scale=scale)
        for j in range(b):
            want, bound = _attention64(q[j, i], k[j, :i + 1], v[j, :i + 1], scale)
            assert ((out[j, i].double() - want).abs() <= bound).all()
            want, bound = _attention64(q[j, i], held[0][j, :i + 1], held[1][j, :i + 1], scale)
            assert ((one[j].double() - want).abs() <= bound).all()
            for n in {i, i + 2} & set(range(1, t + 1)):
                other, _ = _attention64(q[j, i], held[0][j, :n], held[1][j, :n], scale)
                far += ((other - want).abs() > 4 * bound).float().mean() > 0.5
    assert far >= 0.9 * 2 * b * (t - 1)


def _attend_args(**change):
    k_pages, v_pages, table = _cache(2, 3, 4, 2, 64)
    args = dict(q=_values(2, 4, 64).bfloat16(), k_pages=k_pages, v_pages=v_pages, page_table=table,
                lengths=torch.tensor([3, 12], dtype=torch.int32))
    args.update(change)
    return args


@pytest.mark.parametrize("change,error", [
    (dict(q=torch.zeros(2, 3, 64).bfloat16()), ValueError),                          # heads are no multiple of the cache's
    (dict(q=torch.zeros(2, 4, 128).bfloat16()), ValueError),                         # another head size
    (dict(q=torch.zeros(1, 4, 64).bfloat16()), ValueError),                          # another batch
    (dict(lengths=torch.tensor([3, 12])), ValueError),                               # int64
    (dict(lengths=torch.tensor([3, 13], dtype=torch.int32)), IndexError),            # behind the table
    (dict(page_table=torch.zeros(2, 3, dtype=torch.int64)), ValueError),
    (dict(page_table=torch.zeros(3, 2, dtype=torch.int32).t()), ValueError),         # not contiguous
    (dict(page_table=torch.full((2, 3), 8, dtype=torch.int32)), IndexError),         # pages that the pool does not have
    (dict(page_table=torch.full((2, 3), -1, dtype=torch.int32)), IndexError),
    (dict(out=torch.zeros(2, 4, 64)), ValueError),                                   # out of another type
    (dict(k_pages=int4_ops.int4_pages(8, 4, 2, 128)), ValueError),
    (dict(v_pages=int4_ops.int4_pages(7, 4, 2, 64)), ValueError),                    # pools of two sizes
])
def test_attention_refuses(change, error):
    int4_ops.paged_decode_attention_int4(**_attend_args())
    with pytest.raises(error):
        int4_ops.paged_decode_attention_int4(**_attend_args(**change))


@pytest.mark.parametrize("change,error", [
    (dict(v=torch.zeros(2, 5, 2, 64)), ValueError),                                  # another type than k
    (dict(k=torch.zeros(2, 5, 4, 64).bfloat16(), v=torch.zeros(2, 5, 4, 64).bfloat16()), ValueError),
    (dict(start=torch.tensor([0, 0])), ValueError),
    (dict(start=torch.tensor([0], dtype=torch.int32)), ValueError),
    (dict(live=torch.tensor([5.0, 5.0])), ValueError),
    (dict(start=torch.tensor([0, 8], dtype=torch.int32)), IndexError),               # position 12 of 12
    (dict(start=torch.tensor([-1, 0], dtype=torch.int32)), IndexError),
    (dict(page_table=torch.full((2, 3), 8, dtype=torch.int32)), IndexError),
])
def test_append_refuses(change, error):
    k_pages, v_pages, table = _cache(2, 3, 4, 2, 64)
    args = dict(k=_values(2, 5, 2, 64).bfloat16(), v=_values(2, 5, 2, 64).bfloat16(), k_pages=k_pages, v_pages=v_pages,
                page_table=table, start=torch.zeros(2, dtype=torch.int32))
    int4_ops.append_int4(**args)
    with pytest.raises(error):
        int4_ops.append_int4(**{**args, **change})


def test_a_step_refuses_tokens_it_does_not_take():
    k_pages, v_pages, table = _cache(2, 3, 4, 2, 64)
    rope, lengths = torch.zeros(8, 32, 2), torch.tensor([8, 0], dtype=torch.int32)
    args = dict(num_q_heads=4, softmax_scale=0.1)
    qkv = _values(2, 8 * 64).bfloat16()
    int4_ops.rope_decode_attention_int4(qkv, k_pages, v_pages, table, lengths, rope, **args)
    with pytest.raises(ValueError):  # two tokens a sequence
        int4_ops.rope_decode_attention_int4(_values(2, 2, 8 * 64).bfloat16(), k_pages, v_pages, table, lengths, rope, **args)
    with pytest.raises(IndexError):  # position 8 of 8
        int4_ops.rope_decode_attention_int4(qkv, k_pages, v_pages, table, lengths + 1, rope, **args)


def test_a_step_refused_for_its_position_leaves_the_cache():
    k_pages, v_pages, table = _cache(2, 3, 4, 2, 64)
    before = [x.clone() for x in (*k_pages, *v_pages)]
    qkv = _values(2, 8 * 64).bfloat16()
    for positions, length in ((8, 9), (20, 13)):     # behind the rotation table, behind the page table
        with pytest.raises(IndexError):
            int4_ops.rope_decode_attention_int4(qkv, k_pages, v_pages, table, torch.tensor([3, length], dtype=torch.int32),
                                                torch.zeros(positions, 32, 2), num_q_heads=4, softmax_scale=0.1)
        assert all(torch.equal(x, y) for x, y in zip(before, (*k_pages, *v_pages)))
    with pytest.raises(ValueError):                  # a rotation table without a position
        int4_ops.rope_decode_attention_int4(qkv, k_pages, v_pages, table, torch.zeros(2, dtype=torch.int32), torch.zeros(0, 32, 2),
                                            num_q_heads=4, softmax_scale=0.1)


def test_a_pool_without_pages_is_refused():
    empty, table = int4_ops.int4_pages(0, 4, 2, 64), torch.zeros(2, 3, dtype=torch.int32)
    lengths = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        int4_ops.paged_decode_attention_int4(torch.zeros(2, 4, 64).bfloat16(), empty, empty, table, lengths)
    rows = torch.zeros(2, 1, 2, 64).bfloat16()
    with pytest.raises(ValueError):
        int4_ops.append_int4(rows, rows, empty, empty, table, lengths)


def _calls_with_operands():
    """``(name, call, operands)``: each operand may be differentiated by a caller who does not know better."""
    k_pages, v_pages, table = _cache(2, 3, 4, 2, 64)
    lengths, start, rope = torch.tensor([3, 8], dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(8, 32, 2)
    w = int4_ops.quantize_weight(_values(64, 16))
    args = dict(num_q_heads=4, softmax_scale=0.1)
    rows, packed = _values(2, 1, 2, 64).bfloat16(), _values(2, 512).bfloat16()
    return [
        ("int4_linear", lambda x, out: int4_ops.int4_linear(x, w, out=out, accumulate=True), (_values(3, 64), torch.zeros(3, 16))),
        ("append_int4", lambda k, v: int4_ops.append_int4(k, v, k_pages, v_pages, table, start, values=True), (rows, rows.clone())),
        ("paged_decode_attention_int4", lambda q, out: int4_ops.paged_decode_attention_int4(q, k_pages, v_pages, table, lengths, out=out),
         (_values(2, 4, 64).bfloat16(), torch.zeros(2, 4, 64).bfloat16())),
        ("rope_decode_attention_int4",
         lambda qkv: int4_ops.rope_decode_attention_int4(qkv, k_pages, v_pages, table, lengths, rope, **args), (packed,)),
        ("prompt_attention_int4",
         lambda qkv: int4_ops.prompt_attention_int4(qkv, k_pages, v_pages, table, rope, **args), (packed[:, None].clone(),)),
    ]


@pytest.mark.parametrize("call", range(5))
def test_differentiated_operands_are_refused(call):
    name, fn, operands = _calls_with_operands()[call]
    fn(*operands)
    for i, x in enumerate(operands):
        given = [t.clone() for t in operands]
        given[i].requires_grad_()
        with pytest.raises(ValueError, match=f"{name} has no gradient"):
            fn(*given)
        with torch.no_grad():
            fn(*given)
        given = [t.clone() for t in operands]
        with torch.autograd.forward_ad.dual_level():
            fn(*given)
            given[i] = torch.autograd.forward_ad.make_dual(given[i], torch.ones_like(x))
            with pytest.raises(ValueError, match=f"{name} has no gradient"):
                fn(*given)


def test_weights_and_products_refuse():
    w = int4_ops.quantize_weight(_values(64, 16))
    for shape, group in (((60, 16), 128), ((64, 12), 128), ((64, 16), 32)):
        with pytest.raises(ValueError):
            int4_ops.quantize_weight(_values(*shape), group=group)
    with pytest.raises(ValueError):
        int4_ops.quantize_weight(_values(2, 64, 16))
    with pytest.raises(ValueError):
        int4_ops.Int4Weight(w.codes, w.scales, k=64, n=16, group=64)
    with pytest.raises(ValueError):
        int4_ops.int4_linear(_values(3, 72), w)
    with pytest.raises(ValueError):
        int4_ops.int4_linear(_values(3, 64).requires_grad_(), w)
    with pytest.raises(ValueError):
        int4_ops.int4_linear(_values(3, 64), w, accumulate=True)
    with pytest.raises(ValueError):
        int4_ops.int4_linear(_values(3, 64), w, out=torch.zeros(3, 24))
    with pytest.raises(ValueError):
        int4_ops.int4_pages(2, 16, 2, 96)


@pytest.mark.parametrize("rows", [9, 64, 65, 512])
@pytest.mark.parametrize("k,n", [(8, 8), (128, 136), (4096, 4096), (4096, 22016), (4096, 28672), (16384, 2048), (2048, 6144), (8, 10 ** 6)])
def test_plans_of_products(rows, k, n):
    warps, splits = int4_ops.fused_plan(rows, k, n)
    assert 1 <= warps <= 8 and 1 <= splits <= min(8, -(-k // 128))
    assert splits == 1 or -(-n // (16 * warps)) * -(-rows // 128) * splits <= 2 * 148


@pytest.mark.parametrize("tokens", [1, 64, 575, 576, 2048, 130048])
@pytest.mark.parametrize("kv,group", [(1, 1), (8, 4), (32, 16)])
def test_splits_of_an_empty_batch(kv, group, tokens):
    assert int4_ops.attention_splits(0, kv, group, tokens) >= 1


def test_empty_calls():
    k_pages, v_pages, _ = _cache(2, 3, 4, 2, 64)
    before = [x.clone() for x in (*k_pages, *v_pages)]
    table, none, rope = torch.zeros(0, 200, dtype=torch.int32), torch.zeros(0, dtype=torch.int32), torch.zeros(8, 32, 2)
    assert int4_ops.paged_decode_attention_int4(torch.zeros(0, 4, 64).bfloat16(), k_pages, v_pages, table, none).shape == (0, 4, 64)
    args = dict(num_q_heads=4, softmax_scale=0.1)
    assert int4_ops.rope_decode_attention_int4(torch.zeros(0, 512).bfloat16(), k_pages, v_pages, table, none, rope, **args).shape == (0, 4, 64)
    for b, t in ((0, 5), (2, 0)):
        table, start = torch.zeros(b, 200, dtype=torch.int32), torch.zeros(b, dtype=torch.int32)
        rows = torch.zeros(b, t, 2, 64).bfloat16()
        assert int4_ops.append_int4(rows, rows, k_pages, v_pages, table, start, values=True)[0].shape == rows.shape
        qkv = torch.zeros(b, t, 512).bfloat16()
        assert int4_ops.prompt_attention_int4(qkv, k_pages, v_pages, table, rope, **args).shape == (b, t, 256)
    assert all(torch.equal(x, y) for x, y in zip(before, (*k_pages, *v_pages)))


@pytest.mark.parametrize("batch,kv,group,tokens", [(1, 16, 1, 300), (16, 8, 4, 2048), (64, 32, 1, 2000), (1, 8, 4, 130048),
                                                   (1, 1, 1, 1), (0, 4, 1, 64), (300, 32, 16, 4096)])
def test_splits_of_attention(batch, kv, group, tokens):
    splits = int4_ops.attention_splits(batch, kv, group, tokens)
    assert splits >= 1 and (splits == 1 or (tokens >= 32 * splits and batch * kv * -(-group // 8) * splits <= 4 * 148))
