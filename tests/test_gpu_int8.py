"""8-bit rows, weights and cache on the GPU, against 64 bits or the plain statements."""

import math

import pytest
import torch

from axlearn_b200.ops import cuda_ops, decode_ops, dispatch, int8_ops

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, *shape):
    return torch.randn(*shape, device="cuda", generator=gen)


def _plain(fn, *args, **kwargs):
    with dispatch.use_reference_ops():
        return fn(*args, **kwargs)


@pytest.fixture(autouse=True)
def _status():
    yield
    cuda_ops.check_status()


# ------------------------------------------------------------------------------------------
# Rows.
# ------------------------------------------------------------------------------------------


@pytest.mark.parametrize("rows", [1, 3, 300])
@pytest.mark.parametrize("dim", [8, 264, 2048, 4096, 5000, 16384, 40000, 65536])
def test_rows_have_the_bits_of_the_plain_statement(rows, dim):
    gen = _gen(rows + dim)
    x = (_normal(gen, rows, dim) * torch.exp(_normal(gen, rows, 1))).bfloat16()
    x[0, ::2] = x[0].abs().amax() * 0.5  # ties
    got, want = int8_ops.quantize_rows(x), _plain(int8_ops.quantize_rows, x)
    assert torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales)


def test_rows_with_a_pitch_out_of_line_and_not_finite():
    gen = _gen(5)
    wide = _normal(gen, 20, 200).bfloat16()
    for x in (wide[:, :64], wide[:, 8:72], wide[:, 1:65], wide[::3, :64], wide.t()[:, :16], wide[:1, 8:72], wide.view(4, 5, 200)[:, :, :64]):
        got, want = int8_ops.quantize_rows(x), _plain(int8_ops.quantize_rows, x)
        assert torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales)
    x = wide.clone()
    x[1, 3], x[2, 4], x[3, 5] = float("nan"), float("inf"), -float("inf")
    x[4], x[5] = 0, 2.0 ** -120
    x[6] *= 2.0 ** -117
    x[7] *= 2.0 ** 120
    got, want = int8_ops.quantize_rows(x), _plain(int8_ops.quantize_rows, x)
    assert torch.equal(got.codes, want.codes) and torch.equal(got.scales.isnan(), want.scales.isnan())
    assert torch.equal(got.scales.nan_to_num(0), want.scales.nan_to_num(0)) and got.scales[1:4].isnan().all()


@pytest.mark.parametrize("rows", [1, 5, 400])
@pytest.mark.parametrize("dim", [8, 512, 2048, 5000, 8192, 40000])
@pytest.mark.parametrize("residual", [False, True])
def test_norms_have_the_codes_of_exact_arithmetic(rows, dim, residual):
    gen = _gen(rows * dim)
    x, r = (_normal(gen, 2, rows, dim) * torch.exp(0.5 * _normal(gen, dim))).bfloat16()
    w = (1 + 0.2 * _normal(gen, dim)).bfloat16()
    got, total, values = int8_ops.add_rms_norm_int8(x, r if residual else None, w, 1e-5, values=True)
    assert torch.equal(total, x + r if residual else x)
    t = total.double()
    y = t * w.double()
    top = y.abs().amax(-1, keepdim=True)
    assert torch.equal(got.codes.double(), torch.round(y * 127 / top))
    scale = (top / 127 / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-5))[:, 0]
    # Sums of at most 64 squares a thread, then ten of a tree; half of that behind the root, and five roundings.
    assert ((got.scales - scale).abs() <= (37 + 5) * 2.0 ** -24 * scale).all()
    # The product in 32 bits and its rounding to bf16.
    exact = got.codes.double() * got.scales.double()[:, None]
    assert ((values - exact).abs() <= (2.0 ** -8 + 2.0 ** -23) * exact.abs()).all()


def test_norms_of_rows_that_are_not_finite_or_zero():
    gen = _gen(6)
    x, w = _normal(gen, 6, 512).bfloat16(), torch.ones(512, device="cuda").bfloat16()
    x[1, 3], x[2, 4], x[3] = float("nan"), float("inf"), 0
    rows, _, values = int8_ops.add_rms_norm_int8(x, None, w, 1e-5, values=True)
    assert rows.scales[1].isnan() and not rows.scales[2].isfinite() and not values[3].any() and rows.scales[3] == 0
    assert values[[0, 4, 5]].isfinite().all()
    rows3, total3 = int8_ops.add_rms_norm_int8(x.view(2, 3, 512), x.view(2, 3, 512), w.float(), 1e-5)
    assert rows3.codes.shape == (2, 3, 512) and rows3.scales.shape == (2, 3) and total3.shape == (2, 3, 512)
    assert torch.equal(rows3.codes.view(6, 512)[4:], int8_ops.add_rms_norm_int8((x + x)[4:], None, w, 1e-5)[0].codes)


@pytest.mark.parametrize("rows", [1, 7, 320])
@pytest.mark.parametrize("dim", [8, 1032, 11008, 14336, 32768])
def test_swiglu_is_its_formula(rows, dim):
    gu = (2 * _normal(_gen(dim), rows, 2 * dim)).bfloat16()
    got = int8_ops.swiglu_int8(gu)
    gate, up = gu.double().chunk(2, -1)
    y = gate * torch.sigmoid(gate) * up
    top = y.abs().amax(-1, keepdim=True)
    # Half a level; exp to two units, a sum, a quotient and a product in 32 bits.
    assert ((int8_ops.row_values(got).double() - y).abs() <= (0.5 + 127 * 2.0 ** -20) * top / 127).all()


# ------------------------------------------------------------------------------------------
# Products.
# ------------------------------------------------------------------------------------------


def _weight(gen, k, n):
    return int8_ops.quantize_weight(_normal(gen, k, n) * k ** -0.5)


def _linear64(rows, w):
    return (rows.codes.double() @ w.codes.double().t()) * (rows.scales.double()[..., None] * w.scales.double())


def _close(got, want, old=None):
    """Rounded once to bf16, from a sum and two products (and an addition) in 32 bits."""
    whole = want if old is None else want + old.double()
    slack = 2.0 ** -22 * (want.abs() + whole.abs())
    assert ((got.double() - whole).abs() <= 2.0 ** -8 * whole.abs() + slack).all()


@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 32, 33, 64, 65, 128])
@pytest.mark.parametrize("k,n", [(16, 8), (48, 24), (208, 40), (1104, 328), (2048, 96), (4096, 4104)])
def test_linear_of_few_rows(rows, k, n):
    gen = _gen(rows + k)
    w, x = _weight(gen, k, n), _normal(gen, rows, k).bfloat16()
    held = int8_ops.quantize_rows(x)
    want = _linear64(held, w)
    got = int8_ops.int8_linear(held, w)
    _close(got, want)
    assert torch.equal(int8_ops.int8_linear(x, w), got)
    out = _normal(gen, rows, n).bfloat16()
    old = out.clone()
    int8_ops.int8_linear(held, w, out=out, accumulate=True)
    _close(out, want, old)


@pytest.mark.parametrize("rows", [129, 255, 256, 257, 513, 1500])
@pytest.mark.parametrize("k,n", [(16, 8), (208, 136), (1104, 392), (4096, 1032), (272, 9480)])
def test_linear_of_many_rows(rows, k, n):
    gen = _gen(rows + n)
    w, x = _weight(gen, k, n), _normal(gen, rows, k).bfloat16()
    held = int8_ops.quantize_rows(x)
    want = _linear64(held, w)
    got = int8_ops.int8_linear(held, w)
    _close(got, want)
    out = _normal(gen, rows, n).bfloat16()
    old = out.clone()
    int8_ops.int8_linear(held, w, out=out, accumulate=True)
    _close(out, want, old)


@pytest.mark.parametrize("features", [128, 256])
def test_linear_with_either_tile_and_every_tile_of_a_wave(features, monkeypatch):
    monkeypatch.setattr(int8_ops, "pair_features", lambda rows, n: features)
    gen = _gen(features)
    w, held = _weight(gen, 144, 20000), int8_ops.quantize_rows(_normal(gen, 1100, 144).bfloat16())
    _close(int8_ops.int8_linear(held, w), _linear64(held, w))


@pytest.mark.parametrize("rows", [4, 200])
def test_linear_at_the_ends_of_the_integers(rows):
    """127 x 127 all along the longest K: 2114060288, of 31 bits."""
    k = int8_ops.MAX_K
    w = int8_ops.Int8Weight(torch.full((16, k), 127, dtype=torch.int8, device="cuda"), torch.full((16,), 2.0 ** -10, device="cuda"))
    codes = torch.full((rows, k), 127, dtype=torch.int8, device="cuda")
    codes[1] = -127
    got = int8_ops.int8_linear(int8_ops.Int8Rows(codes, torch.full((rows,), 2.0 ** -20, device="cuda")), w)
    want = torch.full((rows, 16), 127 * 127 * k * 2.0 ** -30, device="cuda", dtype=torch.float64)
    want[1] *= -1
    _close(got, want)


@pytest.mark.parametrize("rows", [3, 200])
@pytest.mark.parametrize("accumulate", [False, True])
def test_linear_into_and_from_places_out_of_line(rows, accumulate):
    gen = _gen(rows)
    w, held = _weight(gen, 208, 40), int8_ops.quantize_rows(_normal(gen, rows, 208).bfloat16())
    base = _normal(gen, rows * 40 + 9).bfloat16()
    before, out = base.clone(), base[1:1 + rows * 40].view(rows, 40)
    old = out.clone()
    int8_ops.int8_linear(held, w, out=out, accumulate=accumulate)
    _close(out, _linear64(held, w), old if accumulate else None)
    assert torch.equal(base[:1], before[:1]) and torch.equal(base[1 + rows * 40:], before[1 + rows * 40:])
    room = torch.zeros(rows * 208 + 1, dtype=torch.int8, device="cuda")
    codes = room[1:].view(rows, 208)
    codes.copy_(held.codes)
    assert torch.equal(int8_ops.int8_linear(int8_ops.Int8Rows(codes, held.scales), w), int8_ops.int8_linear(held, w))
    odd = torch.zeros(40 * 208 + 1, dtype=torch.int8, device="cuda")[1:].view(40, 208)
    odd.copy_(w.codes)
    assert torch.equal(int8_ops.int8_linear(held, int8_ops.Int8Weight(odd, w.scales)), int8_ops.int8_linear(held, w))


@pytest.mark.parametrize("rows", [3, 70, 300])
def test_linear_in_place_and_rows_apart(rows):
    gen = _gen(rows)
    w, x = _weight(gen, 256, 256), _normal(gen, rows, 256).bfloat16()
    want = int8_ops.int8_linear(x, w)
    y = x.clone()
    assert torch.equal(int8_ops.int8_linear(y, w, out=y), want)
    poisoned = x.clone()
    poisoned[1] = float("nan")
    got = int8_ops.int8_linear(poisoned, w)
    assert got[1].isnan().all() and torch.equal(got[[0, 2]], want[[0, 2]]) and torch.equal(got[3:], want[3:])
    x3 = x[:rows // 3 * 3].view(3, -1, 256)
    assert torch.equal(int8_ops.int8_linear(x3, w).flatten(0, 1), want[:rows // 3 * 3])


# ------------------------------------------------------------------------------------------
# Cache.
# ------------------------------------------------------------------------------------------


def _cache(b, max_pages, page_size, kv, dim, seed=0, spare=3):
    """Pools of random pages, and a table of pages in any order."""
    gen = _gen(seed)
    pools = []
    for _ in range(2):
        pages = int8_ops.int8_pages(b * max_pages + spare, page_size, kv, dim, device="cuda")
        pages.codes.copy_(torch.randint(-127, 128, pages.codes.shape, generator=gen, device="cuda"))
        pages.tops.copy_(0.5 + 2 * torch.rand(pages.tops.shape, generator=gen, device="cuda"))
        pools.append(pages)
    table = torch.randperm(b * max_pages + spare, generator=gen, device="cuda")[:b * max_pages].to(torch.int32).reshape(b, max_pages)
    return pools[0], pools[1], table


def _attention64(q, k_pages, v_pages, table, lengths, scale):
    """``(out, bound)``: P is rounded to bf16 (2^-8 of it) ahead of its product with the values, and normalised by the sum of what it
    was rounded to, so what is off is values' distance from the result; the result's own rounding; sums of c + 128 in 32 bits."""
    b, nq, h = q.shape
    page_size, kv = k_pages.codes.shape[2], k_pages.codes.shape[1]
    out = torch.zeros(b, nq, h, dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(out)
    for i, n in enumerate(lengths.tolist()):
        if not n:
            continue
        pages = table[i, :-(-n // page_size)].long()
        k, v = (int8_ops.page_values(int8_ops.Int8Pages(p.codes[pages], p.tops[pages]), torch.float64).transpose(0, 1).flatten(1, 2)[:, :n]
                for p in (k_pages, v_pages))
        scores = torch.einsum("kgd,ksd->kgs", q[i].double().reshape(kv, -1, h), k) * scale
        p = torch.softmax(scores, -1)
        o = p @ v
        spread = torch.stack([torch.einsum("ks,ksd->kd", p[:, g], (v - o[:, g, None]).abs()) for g in range(nq // kv)], 1)
        tops = v_pages.tops[pages].double().amax(0)[:, None, None]
        slack = 2.0 ** -14 * tops * (1 + scores.abs().amax(-1, keepdim=True) / 16)
        out[i] = o.reshape(nq, h)
        bound[i] = (1.02 * 2.0 ** -8 * (spread + o.abs()) + slack).reshape(nq, h)
    return out, bound


@pytest.mark.parametrize("nq,kv,dim", [(4, 4, 128), (8, 4, 64), (3, 1, 128), (8, 2, 128), (16, 2, 64), (12, 1, 128), (40, 2, 128)])
@pytest.mark.parametrize("page_size,splits", [(16, 1), (48, 2), (16, 3), (64, 8), (32, 9), (16, 17)])
def test_attention_at_tile_split_and_page_edges(nq, kv, dim, page_size, splits):
    lengths = torch.tensor([0, 1, 15, 16, 17, 31, 33, 64, 100, 129, 500, 1030], dtype=torch.int32, device="cuda")
    b = len(lengths)
    k_pages, v_pages, table = _cache(b, -(-1030 // page_size), page_size, kv, dim, seed=nq + dim)
    q = _normal(_gen(3), b, nq, dim).bfloat16()
    got = int8_ops.paged_decode_attention_int8(q, k_pages, v_pages, table, lengths, splits=splits)
    want, bound = _attention64(q, k_pages, v_pages, table, lengths, dim ** -0.5)
    assert not got[0].any()
    assert ((got.double() - want).abs() <= bound).all(), ((got.double() - want).abs() / bound.clamp(min=1e-30)).max()


@pytest.mark.parametrize("b,nq,kv,dim,tokens,page_size", [(1, 16, 16, 128, 300, 16), (1, 8, 2, 128, 40000, 64), (33, 32, 8, 64, 700, 16),
                                                          (7, 32, 8, 128, 1, 16), (1, 1, 1, 64, 30000, 16)])
def test_attention_with_splits_of_its_own(b, nq, kv, dim, tokens, page_size):
    k_pages, v_pages, table = _cache(b, -(-tokens // page_size), page_size, kv, dim, seed=b)
    lengths = torch.tensor([max(1, tokens - 17 * i) for i in range(b)], dtype=torch.int32, device="cuda")
    q = _normal(_gen(4), b, nq, dim).bfloat16()
    got = int8_ops.paged_decode_attention_int8(q, k_pages, v_pages, table, lengths)
    want, bound = _attention64(q, k_pages, v_pages, table, lengths, dim ** -0.5)
    assert ((got.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("splits", [1, 3, 16])
def test_rows_behind_a_sequence_and_other_pages_are_not_read(dim, splits):
    lengths = torch.tensor([5, 40, 0, 64], dtype=torch.int32, device="cuda")
    k_pages, v_pages, table = _cache(4, 5, 16, 2, dim)
    q = _normal(_gen(5), 4, 4, dim).bfloat16()
    want = int8_ops.paged_decode_attention_int8(q, k_pages, v_pages, table, lengths, splits=splits)
    used = torch.cat([table[i, :-(-n // 16)] for i, n in enumerate(lengths.tolist())]).long()
    others = torch.ones(len(k_pages.tops), dtype=torch.bool, device="cuda")
    others[used] = False
    for p in (k_pages, v_pages):
        p.tops[others] = float("nan")
        p.codes[others] = 77
        for i, n in enumerate(lengths.tolist()):
            if n % 16:
                p.codes[table[i, n // 16].long(), :, n % 16:] = -128
    table = table.clone()
    for i, n in enumerate(lengths.tolist()):
        table[i, -(-n // 16):] = 2 ** 31 - 1
    assert torch.equal(int8_ops.paged_decode_attention_int8(q, k_pages, v_pages, table, lengths, splits=splits), want)


@pytest.mark.parametrize("b,t,kv,dim,page_size,packed", [(1, 1, 1, 128, 16, False), (3, 37, 2, 64, 16, True), (5, 9, 3, 128, 48, True),
                                                         (2, 300, 4, 128, 64, True), (2, 300, 2, 64, 128, False), (3, 200, 5, 128, 32, True),
                                                         (64, 1, 8, 128, 16, True)])
@pytest.mark.parametrize("ragged", [False, True])
def test_append_has_the_bits_of_the_plain_statement(b, t, kv, dim, page_size, packed, ragged):
    gen = _gen(t)
    max_pages = -(-(t + 150) // page_size)
    k_pages, v_pages, table = _cache(b, max_pages, page_size, kv, dim, seed=t)
    qkv = _normal(gen, b, t, 2 * kv + 1, dim).bfloat16() * torch.exp(0.5 * _normal(gen, b, t, 1, 1)).bfloat16()
    k, v = qkv[:, :, 1:1 + kv], qkv[:, :, 1 + kv:]
    if not packed:
        k, v = k.contiguous(), v.contiguous()
    k[0, 0, 0, ::2] = k[0, :, 0].abs().amax() / 2  # ties
    start = torch.randint(0, 150, (b,), generator=gen, device="cuda", dtype=torch.int32) if ragged else torch.zeros(b, dtype=torch.int32, device="cuda")
    live = torch.randint(0, t + 1, (b,), generator=gen, device="cuda", dtype=torch.int32) if ragged else None
    other = [int8_ops.Int8Pages(p.codes.clone(), p.tops.clone()) for p in (k_pages, v_pages)]
    for i in range(2):
        got = int8_ops.append_int8(k, v, k_pages, v_pages, table, start, live=live, values=True)
        want = _plain(int8_ops.append_int8, k, v, *other, table, start, live=live, values=True)
        for x, y, p, o in zip(got, want, (k_pages, v_pages), other):
            assert torch.equal(x, y) and torch.equal(p.codes, o.codes) and torch.equal(p.tops, o.tops)
        k, v = 1.3 * k, 0.9 * v
        start = start + 1 if ragged else start
        if live is not None:
            live = (live - 1).clamp(min=0)
    int8_ops.append_int8(k, v, k_pages, v_pages, table, start, live=live)
