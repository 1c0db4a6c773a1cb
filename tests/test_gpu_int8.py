"""8-bit rows, weights and cache on the GPU, against 64 bits or the plain statements."""

import gc
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


@pytest.fixture(autouse=True, scope="module")
def _memory():
    """Gives memory back: other tests count the segments that the allocator makes."""
    yield
    gc.collect()
    torch.cuda.empty_cache()


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


def test_swiglu_of_gates_far_below_zero():
    """Rows whose largest product is one of a gate beyond -87.3 = log 2^-126."""
    gate = torch.linspace(-90, -86, 4 * 64, device="cuda").bfloat16().view(4, 64)
    up = torch.full((4, 64), 2.0 ** 20, device="cuda").bfloat16()
    up[1], up[2, 1::2] = 2.0 ** 100, -1
    gu = torch.cat([gate, up], 1)
    got = int8_ops.swiglu_int8(gu)
    gate, up = gu.double().chunk(2, -1)
    y = gate * torch.sigmoid(gate) * up
    top = y.abs().amax(-1, keepdim=True)
    # Half a level; |t| 2^-24 and two units of the exponential, whose denormal values (from 2^-131 = exp(-90.8) on) have 19 bits.
    assert got.codes.any(1).all() and ((int8_ops.row_values(got).double() - y).abs() <= (0.5 + 127 * 2.0 ** -16) * top / 127).all()
    gu = torch.tensor([[-float("inf"), 1.0] * 8, [float("inf"), 1.0] * 8, [-200.0] * 16, [0.0, -0.0] * 8], device="cuda").bfloat16()
    rows = int8_ops.swiglu_int8(torch.cat([gu, torch.ones_like(gu)], 1))
    assert rows.scales[:2].isnan().all() and not rows.codes.any() and not rows.scales[2:].any()


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


@pytest.mark.parametrize("rows", [1, 16, 31, 50, 96])
@pytest.mark.parametrize("k,n", [(16, 18952), (1104, 19208), (400, 25000), (2064, 37888), (144, 37896), (272, 56840)])
def test_linear_of_few_rows_and_more_features_than_a_tile_an_sm(rows, k, n):
    gen = _gen(rows + n)
    w, held = _weight(gen, k, n), int8_ops.quantize_rows(_normal(gen, rows, k).bfloat16())
    want = _linear64(held, w)
    _close(int8_ops.int8_linear(held, w), want)
    room = _normal(gen, rows + 1, n).bfloat16()  # (its last row has to stay)
    old = room.clone()
    int8_ops.int8_linear(held, w, out=room[:rows], accumulate=True)
    _close(room[:rows], want, old[:rows])
    assert torch.equal(room[rows], old[rows])


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


@pytest.mark.parametrize("nq,kv,dim,page_size", [(4, 2, 128, 16), (9, 1, 64, 48)])
@pytest.mark.parametrize("splits", [1, 2, 5, 11])
def test_attention_over_many_tiles_a_warp(nq, kv, dim, page_size, splits):
    lengths = torch.tensor([2048, 2049, 9001, 4097 * splits, 3, 6144], dtype=torch.int32, device="cuda")
    k_pages, v_pages, table = _cache(len(lengths), -(-int(lengths.max()) // page_size), page_size, kv, dim, seed=splits)
    q = _normal(_gen(splits), len(lengths), nq, dim).bfloat16()
    got = int8_ops.paged_decode_attention_int8(q, k_pages, v_pages, table, lengths, splits=splits)
    want, bound = _attention64(q, k_pages, v_pages, table, lengths, dim ** -0.5)
    assert ((got.double() - want).abs() <= bound).all()


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


@pytest.mark.parametrize("old,new", [(2.0 ** 121, 1.5 * 2.0 ** 121), (1.5 * 2.0 ** 121, 2.0 ** 122), (2.0 ** 122, 2.0 ** 124),
                                     (2.0 ** 126, 1.9921875 * 2.0 ** 127), (2.0 ** -119, 2.0 ** 127), (2.0 ** 100, 1.5 * 2.0 ** 100),
                                     (2.0 ** -119, 1.0078125 * 2.0 ** -119), (2.0 ** -119, 2.0 ** -118), (2.0 ** -118, 1.5 * 2.0 ** -117)])
@pytest.mark.parametrize("dim,page_size,t", [(128, 16, 1), (64, 128, 20)])
def test_codes_of_pages_that_grow_at_the_ends_of_the_range(old, new, dim, page_size, t):
    """Every code under every pair of magnitudes, in 64 bits."""
    k_pages, v_pages, table = _cache(2, 2, page_size, 2, dim)
    row = torch.arange(128, device="cuda")[-dim:].to(torch.int8)
    for p in (k_pages, v_pages):
        p.codes[:, :, 0], p.codes[:, :, 1], p.codes[:, :, 2] = row, -row, row - 64
        p.tops.fill_(old)
    x = _normal(_gen(1), 2, t, 2, dim)
    x = (x / x.abs().amax(-1, keepdim=True) * new).bfloat16()
    start = torch.tensor([5, 3], dtype=torch.int32, device="cuda")
    want = [torch.round(p.codes.double() * (old / new)) for p in (k_pages, v_pages)]
    int8_ops.append_int8(x, -x, k_pages, v_pages, table, start)
    for sign, p, turned in zip((1, -1), (k_pages, v_pages), want):
        for i, first in enumerate(start.tolist()):
            page = table[i, 0].long()
            assert (p.tops[page].double() == new).all() and torch.equal(p.codes[page, :, :first].double(), turned[page, :, :first])
            count = min(t, page_size - first)
            codes = torch.round(127 * (sign * x[i, :count].double().transpose(0, 1)) / new)
            assert torch.equal(p.codes[page, :, first:first + count].double(), codes)


@pytest.mark.parametrize("nq,kv,dim,splits", [(4, 4, 128, 1), (8, 2, 64, 3), (20, 2, 128, 9), (32, 8, 128, None)])
def test_a_step_is_rotation_append_and_attention(nq, kv, dim, splits):
    lengths = torch.tensor([1, 16, 17, 200, 0, 63, 144], dtype=torch.int32, device="cuda")
    b, gen = len(lengths), _gen(nq)
    k_pages, v_pages, table = _cache(b, 13, 16, kv, dim, seed=nq)
    rope = decode_ops.rope_table(208, dim, 1e4, torch.device("cuda"))
    qkv = (2 * _normal(gen, b, (nq + 2 * kv) * dim)).bfloat16()
    kept = qkv.clone()
    pools = [int8_ops.Int8Pages(p.codes.clone(), p.tops.clone()) for p in (k_pages, v_pages)]
    got = int8_ops.rope_decode_attention_int8(qkv, k_pages, v_pages, table, lengths, rope, num_q_heads=nq, softmax_scale=0.08,
                                              splits=splits)
    assert torch.equal(qkv, kept) and not got[4].any()
    # The same as separate calls: a prompt's rotation of one token, append, attention.
    turned = qkv.clone().view(b, 1, -1, dim)
    angle = rope[(lengths.long() - 1).clamp(min=0)][:, None, None]
    x = turned[..., :nq + kv, :].float().unflatten(-1, (-1, 2))
    sn, cs = angle[..., 0], angle[..., 1]
    both = torch.stack((x[..., 0].double() * cs - x[..., 1].double() * sn, x[..., 1].double() * cs + x[..., 0].double() * sn), -1).flatten(-2)
    turned[..., :nq + kv, :] = both.bfloat16()
    q, k, v = turned.split((nq, kv, kv), 2)
    int8_ops.append_int8(k, v, *pools, table, lengths - 1, live=(lengths > 0).int())
    # (A rotation in 32 bits may round the other way: by a step of bf16, or of codes.)
    for p, o in zip((k_pages, v_pages), pools):
        assert (p.tops.float() / o.tops.float() - 1).abs().max() <= 2.0 ** -7
        assert (int8_ops.page_values(p) - int8_ops.page_values(o)).abs().max() <= 2.1 * o.tops.float().max() / 127
    assert torch.equal(v_pages.codes, pools[1].codes)
    out = int8_ops.paged_decode_attention_int8(got.clone(), k_pages, v_pages, table, lengths, softmax_scale=0.08, splits=splits)
    assert out.shape == got.shape
    want, bound = _attention64(q[:, 0], k_pages, v_pages, table, lengths, 0.08)
    # Queries that round the other way move scores, by 2^-8 of a few of their products.
    assert ((got.double() - want).abs() <= bound + 2.0 ** -6).all()


@pytest.mark.parametrize("nq,kv,dim,splits", [(4, 4, 128, 1), (8, 2, 64, 3), (20, 2, 128, 9), (32, 8, 128, None)])
def test_a_step_attends_to_the_cache_that_it_leaves(nq, kv, dim, splits):
    """Bit for bit: its rotated queries are those of the same token as the last one of a prompt."""
    b, t, gen = 3, 77, _gen(nq + dim)
    rope = decode_ops.rope_table(96, dim, 1e4, torch.device("cuda"))
    qkv = _normal(gen, b, t, (nq + 2 * kv) * dim).bfloat16()
    lengths = torch.tensor([77, 1, 33], dtype=torch.int32, device="cuda")
    k_pages, v_pages, table = _cache(b, 6, 16, kv, dim, seed=nq)
    whole = qkv.clone()
    int8_ops.prompt_attention_int8(whole, k_pages, v_pages, table, rope, num_q_heads=nq, softmax_scale=0.08)
    int8_ops.prompt_attention_int8(qkv.clone(), k_pages, v_pages, table, rope, num_q_heads=nq, softmax_scale=0.08, live=lengths - 1)
    at = torch.arange(b, device="cuda")
    got = int8_ops.rope_decode_attention_int8(qkv[at, lengths.long() - 1], k_pages, v_pages, table, lengths, rope, num_q_heads=nq,
                                              softmax_scale=0.08, splits=splits)
    q = whole[at, lengths.long() - 1, :nq * dim].view(b, nq, dim)
    assert torch.equal(got, int8_ops.paged_decode_attention_int8(q, k_pages, v_pages, table, lengths, softmax_scale=0.08, splits=splits))
    want, bound = _attention64(q, k_pages, v_pages, table, lengths, 0.08)
    assert ((got.double() - want).abs() <= bound).all()


def test_a_step_without_a_place_appends_nothing():
    k_pages, v_pages, table = _cache(4, 2, 16, 2, 64)
    rope = decode_ops.rope_table(24, 64, 1e4, torch.device("cuda"))
    lengths = torch.tensor([25, 20, 33, 0], dtype=torch.int32, device="cuda")
    table = table.clone()
    before = [p.codes.clone() for p in (k_pages, v_pages)]
    qkv = _normal(_gen(7), 4, 8 * 64).bfloat16()
    got = int8_ops.rope_decode_attention_int8(qkv, k_pages, v_pages, table, lengths, rope, num_q_heads=4, softmax_scale=0.1)
    with pytest.raises(RuntimeError, match="status 5"):
        cuda_ops.check_status()
    assert not got[[0, 2, 3]].any() and got[1].any()
    for p, old in zip((k_pages, v_pages), before):
        others = torch.ones(len(old), dtype=torch.bool, device="cuda")
        others[table[1, 1].long()] = False
        assert torch.equal(p.codes[others], old[others])


def test_bad_places_are_reported_and_not_touched():
    k_pages, v_pages, table = _cache(3, 3, 16, 2, 128)
    table = table.clone()
    q = _normal(_gen(8), 3, 4, 128).bfloat16()
    lengths = torch.tensor([20, 48, 30], dtype=torch.int32, device="cuda")
    want = int8_ops.paged_decode_attention_int8(q, k_pages, v_pages, table, lengths)
    cuda_ops.check_status()
    for bad in (-1, 12, 2 ** 31 - 1):
        at = table.clone()
        at[1, 1] = bad
        for splits in (1, 4, 16):
            got = int8_ops.paged_decode_attention_int8(q, k_pages, v_pages, at, lengths, splits=splits)
            with pytest.raises(RuntimeError, match="status 5"):
                cuda_ops.check_status()
            assert got.isfinite().all() and (got[[0, 2]].float() - want[[0, 2]].float()).abs().max() < 0.05
    got = int8_ops.paged_decode_attention_int8(q, k_pages, v_pages, table, lengths + 30)
    with pytest.raises(RuntimeError, match="status 5"):
        cuda_ops.check_status()
    x = _normal(_gen(9), 3, 20, 2, 128).bfloat16()
    at = table.clone()
    at[2, 1] = 12
    start = torch.tensor([-5, 40, 0], dtype=torch.int32, device="cuda")
    live = torch.tensor([20, 20, 20], dtype=torch.int32, device="cuda")
    other = [int8_ops.Int8Pages(p.codes.clone(), p.tops.clone()) for p in (k_pages, v_pages)]
    got = int8_ops.append_int8(x, x, k_pages, v_pages, at, start, live=live, values=True)
    with pytest.raises(RuntimeError, match="status 5"):
        cuda_ops.check_status()
    want = _plain(int8_ops.append_int8, x, x, *other, at, start, live=live, values=True)
    with pytest.raises(RuntimeError, match="status 5"):
        cuda_ops.check_status()
    for a, o, p, y in zip(got, want, (k_pages, v_pages), other):
        assert torch.equal(a, o) and torch.equal(p.codes, y.codes) and torch.equal(p.tops, y.tops)


def _report_a_bad_place(plain):
    k_pages, v_pages, table = _cache(1, 1, 16, 1, 64)
    x = _normal(_gen(1), 1, 1, 1, 64).bfloat16()
    args = (x, x, k_pages, v_pages, torch.full_like(table, 99), torch.zeros(1, dtype=torch.int32, device="cuda"))
    _plain(int8_ops.append_int8, *args) if plain else int8_ops.append_int8(*args)


@pytest.mark.parametrize("plain", [False, True])
def test_a_bad_place_does_not_hide_a_wait_that_gave_up(plain):
    word = cuda_ops.status_word()
    word[0] = 2  # as a kernel whose wait gave up leaves it
    try:
        _report_a_bad_place(plain)
        with pytest.raises(RuntimeError, match="status 2"):
            cuda_ops.check_status()
        cuda_ops.check_status()
        _report_a_bad_place(plain)
        with pytest.raises(RuntimeError, match="status 5"):
            cuda_ops.check_status()
    finally:
        word.zero_()


@pytest.mark.parametrize("product", ["int8", "bf16"])
def test_products_behind_a_bad_place_take_no_longer(product):
    """A kernel waits 2 ms on its way out where a wait gave up, not where an index was bad."""
    gen = _gen(2)
    w, x = _weight(gen, 256, 256), _normal(gen, 300, 256).bfloat16()
    held, plain = int8_ops.quantize_rows(x), _normal(gen, 256, 256).bfloat16()
    call = (lambda: int8_ops.int8_linear(held, w)) if product == "int8" else (lambda: cuda_ops.gemm(x, plain))
    want = call()
    _report_a_bad_place(False)
    times = []
    for _ in range(5):
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        start.record()
        got = call()
        end.record()
        end.synchronize()
        times.append(start.elapsed_time(end))
    with pytest.raises(RuntimeError, match="status 5"):
        cuda_ops.check_status()
    assert torch.equal(got, want) and min(times) < 1


@pytest.mark.parametrize("b,t,nq,kv,dim", [(2, 300, 8, 2, 128), (1, 1, 4, 4, 64), (3, 130, 12, 4, 64), (3, 1300, 6, 2, 128)])
@pytest.mark.parametrize("ragged", [False, True])
def test_prompts_attend_to_what_the_cache_stands_for(b, t, nq, kv, dim, ragged):
    gen = _gen(t)
    max_pages = -(-t // 16)
    k_pages, v_pages, table = _cache(b, max_pages, 16, kv, dim, seed=t)
    rope = decode_ops.rope_table(t, dim, 1e4, torch.device("cuda"))
    qkv = _normal(gen, b, t, (nq + 2 * kv) * dim).bfloat16()
    live = torch.randint(1, t + 1, (b,), generator=gen, device="cuda", dtype=torch.int32) if ragged else None
    mine = qkv.clone()
    got = int8_ops.prompt_attention_int8(mine, k_pages, v_pages, table, rope, num_q_heads=nq, softmax_scale=dim ** -0.5, live=live)
    q, k, v = mine.view(b, t, -1, dim).split((nq, kv, kv), 2)
    given = qkv.view(b, t, -1, dim)[:, :, nq:]
    for i in range(b):
        n = t if live is None else int(live[i])
        pos = torch.arange(n, device="cuda")
        for x, pages, raw in ((k, k_pages, None), (v, v_pages, given[:, :, kv:])):
            held = int8_ops.page_values(pages, torch.bfloat16)[table[i, pos // 16].long(), :, pos % 16]
            assert torch.equal(x[i, :n], held) and not x[i, n:].any()
            if raw is not None:
                tops = pages.tops[table[i, pos // 16].long()].float()[..., None]
                assert ((held.float() - raw[i, :n].float()).abs() <= tops * (0.5 / 127 + 2.0 ** -8) + 1e-6).all()
    want = dispatch.reference.attention(q.double(), k.double(), v.double(), causal=True, softmax_scale=dim ** -0.5).reshape(b, t, -1)
    # Probabilities and the output rounded to bf16, of values of up to five.
    assert (got.double() - want).abs().max() <= 2 * 2.0 ** -8 * 5


def test_scratch_that_does_not_fit_is_refused():
    k_pages, v_pages, table = _cache(1, 64, 16, 1, 128)
    q, lengths = _normal(_gen(1), 1, 2, 128).bfloat16(), torch.tensor([1000], dtype=torch.int32, device="cuda")
    floats = int8_ops.attention_scratch_floats(1, 2, 128, 16)
    assert floats == 2 * 16 * 130 and int8_ops.attention_scratch_floats(1, 2, 128, 8) == 0
    call = lambda scratch: int8_ops.paged_decode_attention_int8(q, k_pages, v_pages, table, lengths, splits=16, scratch=scratch)  # noqa: E731
    for bad in (torch.empty(floats - 1, device="cuda"), torch.empty(floats, device="cuda").half(), torch.empty(floats),
                torch.empty(2 * floats, device="cuda")[::2], torch.empty(floats + 1, device="cuda")[1:]):
        with pytest.raises(ValueError):
            call(bad)
    assert torch.equal(call(torch.empty(floats, device="cuda")), call(None))


def test_a_step_that_is_refused_appends_nothing():
    k_pages, v_pages, table = _cache(1, 64, 16, 1, 64)
    rope = decode_ops.rope_table(1024, 64, 1e4, torch.device("cuda"))
    kept = [x.clone() for x in (*k_pages, *v_pages)]
    many = int8_ops.MAX_GRID + 1
    lengths = torch.zeros(many, dtype=torch.int32, device="cuda")
    lengths[0] = 1000
    qkv = _normal(_gen(1), many, 3 * 64).bfloat16()
    for b, scratch in ((1, torch.empty(8, device="cuda")), (many, None)):
        with pytest.raises(ValueError):
            int8_ops.rope_decode_attention_int8(qkv[:b], k_pages, v_pages, table.expand(b, -1).contiguous(), lengths[:b], rope,
                                                num_q_heads=1, softmax_scale=0.1, splits=16, scratch=scratch)
    given = qkv.clone()
    with pytest.raises(ValueError):
        int8_ops.prompt_attention_int8(qkv[:, None], k_pages, v_pages, table.expand(many, -1).contiguous(), rope, num_q_heads=1,
                                       softmax_scale=0.1, live=torch.zeros_like(lengths))
    with pytest.raises(ValueError):
        int8_ops.paged_decode_attention_int8(qkv.view(many, 3, 64)[:, :1], k_pages, v_pages, table.expand(many, -1).contiguous(), lengths)
    assert torch.equal(qkv, given) and all(torch.equal(x, y) for x, y in zip((*k_pages, *v_pages), kept))


@pytest.mark.parametrize("nq,kv,dim,splits", [(8, 2, 128, 1), (8, 8, 64, 8), (40, 2, 128, 3), (4, 1, 128, 16)])
def test_attention_in_place(nq, kv, dim, splits):
    k_pages, v_pages, table = _cache(3, 40, 16, kv, dim)
    lengths = torch.tensor([600, 3, 0], dtype=torch.int32, device="cuda")
    q = _normal(_gen(2), 3, nq, dim).bfloat16()
    want = int8_ops.paged_decode_attention_int8(q, k_pages, v_pages, table, lengths, splits=splits)
    room = torch.cat([torch.zeros(nq * dim, device="cuda").bfloat16(), q.flatten()])
    moved = room[nq * dim:].view(3, nq, dim)
    assert torch.equal(int8_ops.paged_decode_attention_int8(moved, k_pages, v_pages, table, lengths, splits=splits,
                                                            out=room[:-nq * dim].view(3, nq, dim)), want)
    assert torch.equal(int8_ops.paged_decode_attention_int8(q, k_pages, v_pages, table, lengths, splits=splits, out=q), want)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q_scale,v_scale", [(2.0 ** 50, 2.0 ** 45), (2.0 ** -40, 2.0 ** -40), (1.0, 2.0 ** -40)])
def test_attention_over_small_and_large_values(dim, q_scale, v_scale):
    k_pages, v_pages, table = _cache(2, 20, 16, 2, dim)
    k_pages = int8_ops.Int8Pages(k_pages.codes, (k_pages.tops.float() / max(q_scale, 1.0)).bfloat16())
    v_pages = int8_ops.Int8Pages(v_pages.codes, (v_pages.tops.float() * v_scale).bfloat16())
    lengths = torch.tensor([300, 45], dtype=torch.int32, device="cuda")
    q = (_normal(_gen(3), 2, 4, dim) * q_scale).bfloat16()
    got = int8_ops.paged_decode_attention_int8(q, k_pages, v_pages, table, lengths)
    want, bound = _attention64(q, k_pages, v_pages, table, lengths, dim ** -0.5)
    assert ((got.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("splits", [1, 8, 16])
def test_scores_far_apart(splits):
    """One key of a sequence takes all the weight, wherever it stands; the others' scores are hundreds below."""
    k_pages, v_pages, table = _cache(1, 40, 16, 1, 128)
    q = _normal(_gen(4), 1, 8, 128).bfloat16()
    lengths = torch.tensor([640], dtype=torch.int32, device="cuda")
    for at in (0, 17, 33, 639):
        page, row = table[0, at // 16].long(), at % 16
        kept = k_pages.codes[page, 0, row].clone()
        k_pages.codes[page, 0, row] = (q[0, 0].float() * 127 / q[0, 0].abs().amax()).round().to(torch.int8)
        got = int8_ops.paged_decode_attention_int8(q, k_pages, v_pages, table, lengths, splits=splits, softmax_scale=3.0)
        want, bound = _attention64(q, k_pages, v_pages, table, lengths, 3.0)
        # Scores of some 3000 in 32 bits: 2^-12 in the exponent, and as much again of weights of other heads' keys.
        assert ((got.double() - want).abs() <= bound + 2.0 ** -9).all()
        k_pages.codes[page, 0, row] = kept


def test_values_that_are_not_numbers_stay_where_they_belong():
    k_pages, v_pages, table = _cache(3, 4, 16, 2, 128)
    lengths = torch.tensor([40, 33, 64], dtype=torch.int32, device="cuda")
    q = _normal(_gen(5), 3, 8, 128).bfloat16()
    want = int8_ops.paged_decode_attention_int8(q, k_pages, v_pages, table, lengths)
    q = q.clone()
    q[0, 1, 5] = float("nan")
    k_pages.tops[table[1, 1].long(), 0] = float("nan")
    v_pages.tops[table[2, 3].long(), 1] = float("nan")
    got = int8_ops.paged_decode_attention_int8(q, k_pages, v_pages, table, lengths)
    bad = got.isnan().any(-1)
    expect = torch.zeros_like(bad)
    expect[0, 1], expect[1, :4], expect[2, 4:] = True, True, True
    assert torch.equal(bad, expect) and torch.equal(got[~expect], want[~expect])


@pytest.mark.parametrize("dim,page_size", [(128, 64), (64, 128)])
def test_pools_beyond_32_bits(dim, page_size):
    """Pages whose bytes lie behind 2^32: appended to and attended to like any others."""
    if torch.cuda.mem_get_info()[0] < 30e9:
        pytest.skip("needs 15 GB")
    kv, pages = 8, 2 ** 32 // (8 * page_size * dim) + 40
    k_pages, v_pages = (int8_ops.int8_pages(pages, page_size, kv, dim, device="cuda") for _ in range(2))
    table = torch.tensor([[pages - 1, pages - 3, pages - 20], [2, pages - 30, 5]], dtype=torch.int32, device="cuda")
    x = _normal(_gen(6), 2, 2 * page_size + 9, 2 * kv, dim).bfloat16()
    start = torch.zeros(2, dtype=torch.int32, device="cuda")
    k, v = int8_ops.append_int8(x[:, :, :kv], x[:, :, kv:], k_pages, v_pages, table, start, values=True)
    held = int8_ops.page_values(int8_ops.Int8Pages(k_pages.codes[table.long()].flatten(0, 1), k_pages.tops[table.long()].flatten(0, 1)),
                                torch.bfloat16).view(2, 3, kv, page_size, dim).transpose(2, 3).flatten(1, 2)
    assert torch.equal(held[:, :x.shape[1]], k)
    q, lengths = _normal(_gen(7), 2, 16, dim).bfloat16(), torch.full((2,), x.shape[1], dtype=torch.int32, device="cuda")
    got = int8_ops.paged_decode_attention_int8(q, k_pages, v_pages, table, lengths)
    want, bound = _attention64(q, k_pages, v_pages, table, lengths, dim ** -0.5)
    assert ((got.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("rows", [3, 200])
def test_linear_of_codes_beyond_32_bits(rows):
    """A weight of 4.3 GB: its last columns."""
    if torch.cuda.mem_get_info()[0] < 12e9:
        pytest.skip("needs 6 GB")
    k, n = 65536, 65536 + 512
    gen = _gen(rows)
    codes = torch.empty(n, k, dtype=torch.int8, device="cuda")
    for lo in range(0, n, 4096):
        codes[lo:lo + 4096] = torch.randint(-127, 128, (min(4096, n - lo), k), generator=gen, device="cuda", dtype=torch.int8)
    w = int8_ops.Int8Weight(codes, torch.rand(n, generator=gen, device="cuda") * 2.0 ** -14)
    held = int8_ops.quantize_rows(_normal(gen, rows, k).bfloat16())
    got = int8_ops.int8_linear(held, w)
    for at in (slice(0, 128), slice(n - 128, n)):
        want = (held.codes.double() @ codes[at].double().t()) * (held.scales.double()[:, None] * w.scales[at].double())
        _close(got[:, at], want)


def test_calls_replay_in_a_graph_and_on_another_stream():
    """Every entry point, captured together and replayed over other inputs, and again on a stream of its own."""
    gen = _gen(10)
    k_pages, v_pages, table = _cache(3, 20, 16, 2, 128)
    lengths = torch.tensor([40, 1, 300], dtype=torch.int32, device="cuda")
    rope = decode_ops.rope_table(320, 128, 1e4, torch.device("cuda"))
    x, r, norm = _normal(gen, 3, 512).bfloat16(), _normal(gen, 3, 512).bfloat16(), torch.ones(512, device="cuda").bfloat16()
    wide = _normal(gen, 200, 512).bfloat16()
    wqkv, wgu, wdown = _weight(gen, 512, 8 * 128), _weight(gen, 512, 2048), _weight(gen, 1024, 512)

    def chain(pools):
        rows, total = int8_ops.add_rms_norm_int8(x, r, norm, 1e-5)
        attn = int8_ops.rope_decode_attention_int8(int8_ops.int8_linear(rows, wqkv), *pools, table, lengths, rope, num_q_heads=4,
                                                   softmax_scale=0.1, splits=16)
        act = int8_ops.swiglu_int8(int8_ops.int8_linear(int8_ops.quantize_rows(attn.flatten(1)), wgu))
        out = int8_ops.int8_linear(act, wdown, out=total, accumulate=True)
        many = int8_ops.int8_linear(wide, wgu)
        k = attn.view(3, 1, 4, 128)[:, :, :2]
        int8_ops.append_int8(k, k, *pools, table, lengths, values=False)
        return out, many, int8_ops.paged_decode_attention_int8(attn, *pools, table, lengths)

    def copies():
        return [int8_ops.Int8Pages(p.codes.clone(), p.tops.clone()) for p in (k_pages, v_pages)]

    want = [t.clone() for t in chain(copies())]
    pools, side = copies(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [t.clone() for t in chain(pools)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    held = copies()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = chain(held)
    for seed in (11, 12):
        for p, o in zip(held, copies()):
            p.codes.copy_(o.codes), p.tops.copy_(o.tops)
        x.copy_(_normal(_gen(seed), 3, 512)), wide.copy_(_normal(_gen(seed), 200, 512))
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, chain(copies())))


def test_products_of_all_kinds_replay_in_graphs_side_by_side():
    gen = _gen(13)
    cases = []
    for rows, k, n in ((1, 2048, 2048), (16, 4096, 1024), (100, 1024, 4096), (300, 1024, 2048)):
        held, w = int8_ops.quantize_rows(_normal(gen, rows, k).bfloat16()), _weight(gen, k, n)
        cases.append((held, w, int8_ops.int8_linear(held, w).clone()))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = [int8_ops.int8_linear(held, w) for held, w, _ in cases]
        graphs.append((graph, out, torch.cuda.Stream()))
    for _ in range(20):
        for graph, _, stream in graphs:
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, out, _ in graphs:
        assert all(torch.equal(y, want) for y, (_, _, want) in zip(out, cases))


def test_attention_of_many_splits_replays_in_graphs_side_by_side():
    lengths = torch.tensor([700, 3000], dtype=torch.int32, device="cuda")
    k_pages, v_pages, table = _cache(2, 3000 // 16 + 1, 16, 2, 128)
    queries = [_normal(_gen(i), 2, 8, 128).bfloat16() for i in range(2)]
    want = [int8_ops.paged_decode_attention_int8(q, k_pages, v_pages, table, lengths, splits=16).clone() for q in queries]
    graphs = []
    for q in queries:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = int8_ops.paged_decode_attention_int8(q, k_pages, v_pages, table, lengths, splits=16)
        graphs.append((graph, out, torch.cuda.Stream()))
    for _ in range(20):
        for graph, _, stream in graphs:
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out, y) for (_, out, _), y in zip(graphs, want))


@pytest.mark.parametrize("splits", [None, 1, 8, 9, 16])
def test_empty_calls(splits):
    k_pages, v_pages, table = _cache(2, 2, 16, 2, 64)
    none, rope = torch.zeros(0, dtype=torch.int32, device="cuda"), decode_ops.rope_table(32, 64, 1e4, torch.device("cuda"))
    empty = torch.zeros(0, 4, 64, device="cuda").bfloat16()
    assert int8_ops.paged_decode_attention_int8(empty, k_pages, v_pages, table[:0], none, splits=splits).shape == (0, 4, 64)
    assert int8_ops.rope_decode_attention_int8(torch.zeros(0, 512, device="cuda").bfloat16(), k_pages, v_pages, table[:0], none, rope,
                                               num_q_heads=4, softmax_scale=0.1, splits=splits).shape == (0, 4, 64)
    zeros = torch.zeros(2, dtype=torch.int32, device="cuda")
    got = int8_ops.paged_decode_attention_int8(torch.ones(2, 4, 64, device="cuda").bfloat16(), k_pages, v_pages, table, zeros, splits=splits)
    assert not got.any()
    no_pages = torch.zeros(2, 0, dtype=torch.int32, device="cuda")
    assert not int8_ops.paged_decode_attention_int8(torch.ones(2, 4, 64, device="cuda").bfloat16(), k_pages, v_pages, no_pages, zeros,
                                                    splits=splits).any()
    for x in (torch.zeros(0, 3, 2, 64, device="cuda").bfloat16(), torch.zeros(2, 0, 2, 64, device="cuda").bfloat16()):
        k, v = int8_ops.append_int8(x, x, k_pages, v_pages, table[:len(x)], zeros[:len(x)], values=True)
        assert k.shape == v.shape == x.shape
    w = _weight(_gen(1), 16, 8)
    assert int8_ops.int8_linear(torch.zeros(0, 16, device="cuda").bfloat16(), w).shape == (0, 8)
    rows, total = int8_ops.add_rms_norm_int8(torch.zeros(0, 16, device="cuda").bfloat16(), None, torch.ones(16, device="cuda"), 1e-5)
    assert rows.codes.shape == (0, 16) and total.shape == (0, 16)


def test_differentiated_operands_are_refused():
    k_pages, v_pages, table = _cache(1, 2, 16, 1, 64)
    w, one = _weight(_gen(1), 16, 8), torch.ones(1, dtype=torch.int32, device="cuda")
    x, q, k = (torch.ones(*s, device="cuda").bfloat16().requires_grad_() for s in ((2, 16), (1, 1, 64), (1, 1, 1, 64)))
    for call in (lambda: int8_ops.quantize_rows(x), lambda: int8_ops.swiglu_int8(x), lambda: int8_ops.int8_linear(x, w),
                 lambda: int8_ops.add_rms_norm_int8(x, None, torch.ones(16, device="cuda"), 1e-5),
                 lambda: int8_ops.append_int8(k, k, k_pages, v_pages, table, one),
                 lambda: int8_ops.paged_decode_attention_int8(q, k_pages, v_pages, table, one)):
        with pytest.raises(ValueError, match="no gradient"):
            call()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_other_types_run_the_plain_statements_on_the_gpu(dtype):
    gen = _gen(14)
    x = _normal(gen, 5, 64).to(dtype)
    w = int8_ops.quantize_weight(_normal(gen, 64, 24))
    cpu = int8_ops.Int8Weight(w.codes.cpu(), w.scales.cpu())
    got = int8_ops.int8_linear(x, w)
    assert got.dtype == dtype and torch.equal(got.cpu(), int8_ops.int8_linear(x.cpu(), cpu))
    k_pages, v_pages, table = _cache(2, 3, 16, 2, 64)
    other = [int8_ops.Int8Pages(p.codes.cpu(), p.tops.cpu()) for p in (k_pages, v_pages)]
    k, start = _normal(gen, 2, 20, 2, 64).to(dtype), torch.tensor([3, 16], dtype=torch.int32, device="cuda")
    a = int8_ops.append_int8(k, k, k_pages, v_pages, table, start, values=True)
    b = int8_ops.append_int8(k.cpu(), k.cpu(), *other, table.cpu(), start.cpu(), values=True)
    assert all(torch.equal(p.codes.cpu(), o.codes) and torch.equal(p.tops.cpu(), o.tops) for p, o in zip((k_pages, v_pages), other))
    assert all((y.cpu().double() - z.double()).abs().max() <= 2 * torch.finfo(dtype).eps * z.abs().max() for y, z in zip(a, b))


# ------------------------------------------------------------------------------------------
# The engine.
# ------------------------------------------------------------------------------------------


def _engine_weights(d, f, vocab, nq, nkv, layers, seed=0):
    from axlearn_b200.inference.decode_engine import FujiDims, LayerWeights

    g = _gen(seed)

    def w(*shape):
        return (_normal(g, *shape) * shape[0] ** -0.5).bfloat16()

    weights = {"layers": [LayerWeights(attn_norm=1 + 0.1 * w(d), wqkv=w(d, (nq + 2 * nkv) * 128), wo=w(nq * 128, d),
                                       ffn_norm=1 + 0.1 * w(d), wgu=w(d, 2 * f), wdown=w(f, d)) for _ in range(layers)],
               "emb": w(vocab, d) * 16, "head": w(vocab, d), "final_norm": 1 + 0.1 * w(d)}
    return weights, FujiDims(num_layers=layers, hidden_dim=d, num_heads=nq, num_kv_heads=nkv, head_dim=128, ffn_dim=f,
                             vocab_size=vocab)


@pytest.mark.parametrize("weight_bits,cache_bits", [(8, 8), (8, 16), (16, 8), (4, 8), (8, 4)])
@pytest.mark.parametrize("b,nq,nkv", [(1, 4, 4), (5, 8, 2)])
def test_engine_in_8_bits_matches_its_plain_statements(weight_bits, cache_bits, b, nq, nkv):
    """Prompts and steps with the kernels against the same engine on the plain statements, the captured step against separate
    launches."""
    from axlearn_b200.inference import decode_engine

    weights, dims = _engine_weights(256, 528, 1000, nq, nkv, 2, seed=b)
    if weight_bits != 16:
        weights = decode_engine.quantize_weights(weights, group=64, bits=weight_bits)
        assert weight_bits == 4 or all(isinstance(lw.wgu, int8_ops.Int8Weight) for lw in weights["layers"])
    ids = torch.randint(0, 1000, (b, 90), device="cuda", generator=_gen(1))
    lengths = torch.randint(1, 71, (b,), device="cuda", generator=_gen(2))
    lengths[0] = 70

    def engine(use_graph):
        return decode_engine.DecodeEngine(weights, dims, batch=b, max_len=96, use_graph=use_graph, cache_bits=cache_bits)

    chained, separate, plain = engine(True), engine(False), engine(False)

    def close():
        # Two layers of some five operations, each of which may round its output the other way (2^-8 of it); norms and
        # residuals pass that on with a gain of about one.  A value that does moves to the next code in 2^-8 |x| / s of the cases, by s:
        # with |x| about 0.8 sigma and A about 3.5 sigma, s = 0.028 sigma, that is sqrt(2 * 2^-8 * 0.8 * 0.028) = 0.013 sigma (rms; both
        # sides may move) of each of the four products' rows and of keys and values, in each layer.  In 4 bits 0.042 of those.
        off = (separate.logits - plain.logits).norm() / plain.logits.norm()
        limit = 10 * 2.0 ** -8 + (2 * 4 * 0.013 if weight_bits == 8 else 0)
        assert off < limit + (2 * 2 * 0.013 if cache_bits == 8 else 2 * 0.042 if cache_bits == 4 else 0), off

    firsts = [e.prefill(ids[:, :70], lengths=lengths) for e in (chained, separate)]
    assert torch.equal(firsts[0], firsts[1])
    _plain(plain.prefill, ids[:, :70], lengths=lengths)
    close()
    for i in range(70, 90):
        x, y = chained.step_logits(ids[:, i]).clone(), separate.step_logits(ids[:, i])
        assert torch.equal(x, y)
        _plain(plain.step_logits, ids[:, i])
        close()
    tokens = chained.generate(ids[:, :33], 5)
    assert tokens.shape == (b, 5) and torch.equal(tokens, separate.generate(ids[:, :33], 5))


@pytest.mark.parametrize("batch", [1, 16])
def test_engine_steps_in_8_bits_at_serving_widths(batch):
    """Kernels that overlap for long: replays of the chained step against separate launches, bit for bit."""
    from axlearn_b200.inference import decode_engine

    weights, dims = _engine_weights(4096, 14336, 8192, 32, 8, 2, seed=3)
    weights = decode_engine.quantize_weights(weights, bits=8)
    engines = [decode_engine.DecodeEngine(weights, dims, batch=batch, max_len=2048, use_graph=use, cache_bits=8) for use in (True, False)]
    ids = torch.randint(0, 8192, (batch, 1500), device="cuda", generator=_gen(4))
    lengths = torch.randint(1, 1501, (batch,), device="cuda", generator=_gen(5))
    for e in engines:
        e.prefill(ids, lengths=lengths)
    for i in range(12):
        x, y = (e.step_logits(ids[:, i]).clone() for e in engines)
        assert torch.equal(x, y), i


@pytest.mark.parametrize("down,fused", [(16, True), (4, True), (8, False)])
def test_prompts_fuse_gate_and_up_wherever_the_down_projection_takes_16_bits(down, fused, monkeypatch):
    import dataclasses

    from axlearn_b200.inference import decode_engine
    from axlearn_b200.ops import int4_ops

    weights, dims = _engine_weights(256, 512, 1000, 4, 4, 2)
    hold = {16: lambda w: w, 8: int8_ops.quantize_weight, 4: int4_ops.quantize_weight}[down]
    weights["layers"] = [dataclasses.replace(lw, wdown=hold(lw.wdown)) for lw in weights["layers"]]
    calls, real = [], cuda_ops.gemm_swiglu
    monkeypatch.setattr(cuda_ops, "gemm_swiglu", lambda *args: (calls.append(args), real(*args))[1])
    engine = decode_engine.DecodeEngine(weights, dims, batch=2, max_len=96, use_graph=False)
    engine.prefill(torch.randint(0, 1000, (2, 64), device="cuda", generator=_gen(1)))
    assert len(calls) == (2 if fused else 0) and engine.logits.isfinite().all()


def test_engine_in_8_bits_is_close_to_16_bits():
    """What both formats lose on a small model: rows, weights and cache are each off by up to half of 1 / 127 of their largest value."""
    from axlearn_b200.inference import decode_engine

    weights, dims = _engine_weights(512, 1024, 1000, 8, 2, 2, seed=9)
    ids = torch.randint(0, 1000, (3, 60), device="cuda", generator=_gen(1))
    logits = []
    for bits in (16, 8):
        w = weights if bits == 16 else decode_engine.quantize_weights(weights, bits=8)
        e = decode_engine.DecodeEngine(w, dims, batch=3, max_len=64, use_graph=False, cache_bits=bits)
        e.prefill(ids[:, :59])
        logits.append(e.step_logits(ids[:, 59]).clone())
    # A uniform rounding of s = 0.03 sigma is 0.03 / sqrt(12) = 0.009 of a value (rms); two for each of four products, two for the
    # cache, in two layers, all passed on with a gain of about one: sqrt(20) * 0.009 = 0.04, and twice that for its spread.
    assert (logits[1] - logits[0]).norm() / logits[0].norm() < 0.08


def test_sample_decode_takes_the_formats_of_the_environment(monkeypatch):
    from axlearn_b200.common import decoding, logit_modifiers, prng
    from axlearn_b200.common.module import functional
    from axlearn_b200.common.utils import tree_map
    from axlearn_b200.inference import decode_engine
    from tests.test_gpu_decode import _tiny_model

    model, params = _tiny_model(1)
    params = tree_map(lambda t: t.cuda().bfloat16() if t.is_floating_point() else t.cuda(), params)
    prefix = torch.randint(2, 512, (2, 24), device="cuda", generator=_gen(6))
    prefix[1, 9:] = 0
    kwargs = dict(input_batch={"prefix": prefix}, num_decodes=2, max_sequence_length=40, logits_modifier=logit_modifiers.top_k_logits(1),
                  stop_decoding_condition=decoding.StopOnSubsequence([[511]]))
    seen = []
    real = decode_engine.DecodeEngine.step_logits
    monkeypatch.setattr(decode_engine.DecodeEngine, "step_logits", lambda self, tokens: (seen.append(self), real(self, tokens))[1])
    monkeypatch.setenv("AXB200_DECODE_INT8", "weights,cache")
    out, _ = functional(model, prng.PRNGKey(5), params, kwargs, is_training=False, method="sample_decode")
    assert out.sequences.shape == (2, 2, 39) and seen[-1].cache_bits == 8
    assert isinstance(seen[-1].w["layers"][0].wo, int8_ops.Int8Weight)
    monkeypatch.setenv("AXB200_DECODE_INT8", "cache")
    functional(model, prng.PRNGKey(5), params, kwargs, is_training=False, method="sample_decode")
    assert seen[-1].cache_bits == 8 and isinstance(seen[-1].w["layers"][0].wo, torch.Tensor)
    for name, value in (("AXB200_DECODE_INT8", "caches"), ("AXB200_DECODE_CACHE_BITS", "4")):
        monkeypatch.setenv("AXB200_DECODE_INT8", "cache")
        monkeypatch.setenv(name, value)
        with pytest.raises(ValueError, match="AXB200_DECODE_INT8"):
            functional(model, prng.PRNGKey(5), params, kwargs, is_training=False, method="sample_decode")
