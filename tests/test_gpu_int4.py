"""Kernels of the 4-bit weights and cache against plain statements in 64 bits."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, *shape):
    return torch.randn(*shape, device="cuda", generator=gen)


def _plain(fn, *args, **kwargs):
    from axlearn_b200.ops.dispatch import use_reference_ops

    with use_reference_ops():
        return fn(*args, **kwargs)


def _cache(b, max_pages, page_size, kv, dim, seed=0, spare=3):
    """Pools of quantised normal values with larger and shifted channels, and a scrambled table."""
    from axlearn_b200.ops import int4_ops

    gen, pools = _gen(seed), []
    for _ in range(2):
        gain, mean = torch.exp(0.5 * _normal(gen, kv, 1, dim)), 0.5 * _normal(gen, kv, 1, dim)
        x = (_normal(gen, b * max_pages + spare, kv, page_size, dim) * gain + mean).bfloat16()
        codes, scales = int4_ops.quantize_groups(x, 32)
        pools.append(int4_ops.Int4Pages(int4_ops._pack_rows(codes), scales))  # pylint: disable=protected-access
    table = torch.randperm(b * max_pages + spare, device="cuda", generator=gen)[:b * max_pages]
    return pools[0], pools[1], table.to(torch.int32).reshape(b, max_pages).contiguous()


def _attention64(q, k_pages, v_pages, table, lengths, scale):
    """``(out, bound)``: attention in 64 bits, and what rounding may add to it."""
    from axlearn_b200.ops import int4_ops

    b, nq, h = q.shape
    kv = k_pages.codes.shape[1]
    out, bound = torch.zeros(b, nq, h, dtype=torch.float64, device="cuda"), torch.zeros(b, nq, h, dtype=torch.float64, device="cuda")
    for i, n in enumerate(lengths.tolist()):
        if not n:
            continue
        pages = table[i, :-(-n // k_pages.codes.shape[2])].long()
        (k, ks), (v, vs) = ((int4_ops.page_values(int4_ops.Int4Pages(x.codes[pages], x.scales[pages]), torch.float64),
                             x.scales[pages].double()) for x in (k_pages, v_pages))
        k, ks, v, vs = (x.transpose(0, 1).flatten(1, 2)[:, :n] for x in (k, ks, v, vs))
        qg = q[i].double().view(kv, -1, h)
        p = torch.softmax(qg @ k.transpose(1, 2) * scale, -1)
        out[i] = (p @ v).flatten(0, 1)
        # A score is a sum of products with 128 + c (tensor cores cut sums off at 2^-23 of their largest term): some 12 steps.
        size = ks.abs() @ torch.tensor([143.0, 1.0], device="cuda", dtype=torch.float64)
        moved = 12 * 2.0 ** -23 * scale * (qg.abs().unflatten(-1, (-1, 32)).sum(-1) @ size.transpose(1, 2)).amax(-1, keepdim=True)
        # A probability is rounded to bf16, its product with s again: p (m + s c) becomes p (1 + a) (m + s c (1 + b)) with a
        # and b up to 2^-8, off by 2^-8 p |v| and (1 + 2^-8) 2^-8 p s c.  Sums in 32 bits; the output's rounding.
        low = vs[..., 1].repeat_interleave(32, -1)
        step = vs[..., 0].repeat_interleave(32, -1)
        bound[i] = (2.0 ** -8 * (p @ v.abs() + 1.004 * (p @ (v - low))) + 8 * 2.0 ** -23 * 143 * (p @ step) + torch.expm1(2 * moved) * (p @ v.abs())
                    + 2.0 ** -20 * (p @ v.abs())).flatten(0, 1)
        bound[i] = 1.01 * bound[i] + 2.0 ** -8 * (out[i].abs() + bound[i])
    return out, bound


@pytest.mark.parametrize("nq,kv,dim", [(4, 4, 128), (8, 4, 64), (3, 1, 128), (8, 2, 128), (16, 2, 64), (12, 1, 128), (40, 2, 128)])
@pytest.mark.parametrize("page_size,splits", [(1, 1), (12, 2), (16, 3), (64, 8), (20, 9), (16, 17)])
def test_attention_at_tile_split_and_page_edges(nq, kv, dim, page_size, splits):
    from axlearn_b200.ops import cuda_ops, int4_ops

    lens = [0, 1, 31, 32, 33, 127, 128, 129, 255, 320]
    k_pages, v_pages, table = _cache(len(lens), -(-320 // page_size), page_size, kv, dim, seed=splits)
    lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = (2 * _normal(_gen(1), len(lens), nq, dim)).bfloat16()
    out = int4_ops.paged_decode_attention_int4(q, k_pages, v_pages, table, lengths, splits=splits)
    want, bound = _attention64(q, k_pages, v_pages, table, lengths, dim ** -0.5)
    cuda_ops.check_status()
    assert not out[0].any() and ((out.double() - want).abs() <= bound).all()
    again = int4_ops.paged_decode_attention_int4(q, k_pages, v_pages, table, lengths, splits=splits)
    assert torch.equal(out, again)


@pytest.mark.parametrize("b,nq,kv,dim,tokens", [(1, 16, 16, 128, 300), (1, 8, 2, 128, 40000), (33, 32, 8, 64, 700), (7, 32, 8, 128, 1)])
def test_attention_with_splits_of_its_own(b, nq, kv, dim, tokens):
    from axlearn_b200.ops import int4_ops

    k_pages, v_pages, table = _cache(b, -(-tokens // 16), 16, kv, dim, seed=b)
    lengths = torch.randint(0, tokens + 1, (b,), dtype=torch.int32, device="cuda", generator=_gen(2))
    lengths[0] = tokens
    q = _normal(_gen(3), b, 2 * nq, dim).bfloat16()[:, ::2]  # not contiguous
    out = torch.full((b, nq, dim), 7.0, device="cuda", dtype=torch.bfloat16)
    assert int4_ops.paged_decode_attention_int4(q, k_pages, v_pages, table, lengths, softmax_scale=0.2, out=out) is out
    want, bound = _attention64(q, k_pages, v_pages, table, lengths, 0.2)
    assert ((out.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dim", [64, 128])
def test_rows_behind_a_sequence_and_other_pages_are_not_read(dim):
    from axlearn_b200.ops import int4_ops

    k_pages, v_pages, table = _cache(3, 4, 16, 2, dim, seed=5)
    lengths = torch.tensor([5, 33, 47], dtype=torch.int32, device="cuda")
    q = _normal(_gen(4), 3, 4, dim).bfloat16()
    before = int4_ops.paged_decode_attention_int4(q, k_pages, v_pages, table, lengths, splits=2)
    for pages in (k_pages, v_pages):
        used = torch.zeros(pages.codes.shape[0], 16, dtype=torch.bool, device="cuda")
        for i, n in enumerate(lengths.tolist()):
            for pos in range(n):
                used[table[i, pos // 16].long(), pos % 16] = True
        pages.scales.transpose(1, 2)[~used] = torch.nan
        pages.codes.transpose(1, 2)[~used] = 255
    table[0, 1:], table[1, 3:] = 10 ** 9, -7  # behind the sequences' last pages
    after = int4_ops.paged_decode_attention_int4(q, k_pages, v_pages, table, lengths, splits=2)
    assert torch.equal(before, after)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q_scale,v_scale", [(2.0 ** 40, 2.0 ** 40), (2.0 ** -40, 2.0 ** -40), (1.0, 2.0 ** -40)])
def test_attention_over_small_and_large_values(dim, q_scale, v_scale):
    """Powers of two that leave the scores as they are leave every digit as it is."""
    from axlearn_b200.ops import int4_ops

    k_pages, v_pages, table = _cache(2, 20, 16, 2, dim, seed=7)
    lengths = torch.tensor([320, 77], dtype=torch.int32, device="cuda")
    q = _normal(_gen(8), 2, 8, dim).bfloat16()
    plain = int4_ops.paged_decode_attention_int4(q, k_pages, v_pages, table, lengths)
    k_pages, v_pages = k_pages._replace(scales=k_pages.scales / q_scale), v_pages._replace(scales=v_pages.scales * v_scale)
    assert torch.equal(int4_ops.paged_decode_attention_int4(q * q_scale, k_pages, v_pages, table, lengths), plain * v_scale)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("tokens", [2, 4, 8, 12, 24, 48, 200])
def test_short_sequences_keep_their_precision(tokens, dim):
    """Two roundings of a probability beside the output's own.  The same roundings simulated in 64 bits add up to 1.22 of the
    output's rounding in the 2-norm; without the shift of the codes by 8 they are 1.4 to 1.8 of it."""
    from axlearn_b200.ops import int4_ops

    k_pages, v_pages, table = _cache(64, -(-tokens // 16), 16, 4, dim, seed=tokens)
    lengths = torch.full((64,), tokens, dtype=torch.int32, device="cuda")
    q = _normal(_gen(4), 64, 8, dim).bfloat16()
    out = int4_ops.paged_decode_attention_int4(q, k_pages, v_pages, table, lengths)
    want, _ = _attention64(q, k_pages, v_pages, table, lengths, dim ** -0.5)
    assert (out.double() - want).norm() <= 1.35 * (want.float().bfloat16().double() - want).norm()


@pytest.mark.parametrize("splits", [1, 8, 16])
def test_scores_far_apart(splits):
    """One key that takes all, early or late, and scores that climb by more than the slack from tile to tile."""
    from axlearn_b200.ops import int4_ops

    k_pages, v_pages, table = _cache(3, 20, 16, 1, 128, seed=9)
    q = torch.zeros(3, 4, 128, device="cuda").bfloat16()
    q[:, :, 0] = 100.0
    k = torch.zeros(3, 320, 1, 128, device="cuda")
    k[0, 5, 0, 0], k[1, 318, 0, 0], k[2, :, 0, 0] = 30.0, 30.0, torch.arange(320, device="cuda") * 0.25 - 40
    start = torch.zeros(3, dtype=torch.int32, device="cuda")
    int4_ops.append_int4(k.bfloat16(), _normal(_gen(10), 3, 320, 1, 128).bfloat16(), k_pages, v_pages, table, start)
    lengths = torch.tensor([320, 319, 320], dtype=torch.int32, device="cuda")
    out = int4_ops.paged_decode_attention_int4(q, k_pages, v_pages, table, lengths, splits=splits)
    want, bound = _attention64(q, k_pages, v_pages, table, lengths, 128 ** -0.5)
    assert ((out.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dim,page_size", [(128, 64), (64, 128)])
def test_pools_beyond_32_bits(dim, page_size):
    """Pages whose codes lie more than 2^32 bytes into the pool: append, step and attention as over a small pool."""
    from axlearn_b200.ops import cuda_ops, decode_ops, int4_ops

    kv, b, used = 8, 2, 6
    pages = 2 ** 32 // (kv * page_size * (dim // 2)) + 40
    if torch.cuda.mem_get_info()[0] < 30 * 2 ** 30:
        pytest.skip("a pool of 12 GB")
    small = _cache(b, used, page_size, kv, dim, seed=11, spare=0)
    high = [int4_ops.int4_pages(pages, page_size, kv, dim, device="cuda") for _ in range(2)]
    for pool, low in zip(high, small):
        pool.codes[-b * used:], pool.scales[-b * used:] = low.codes, low.scales
    table = small[2] + (pages - b * used)
    lengths = torch.tensor([used * page_size - 3, 200], dtype=torch.int32, device="cuda")
    gen = _gen(12)
    q = _normal(gen, b, 16, dim).bfloat16()
    qkv = _normal(gen, b, (16 + 2 * kv) * dim).bfloat16()
    new = [_normal(gen, b, 30, kv, dim).bfloat16() for _ in range(2)]
    rope = decode_ops.rope_table(used * page_size, dim, 1e4, "cuda")

    def run(k_pages, v_pages, table):
        outs = []
        for splits in (1, 4, 16):
            outs.append(int4_ops.paged_decode_attention_int4(q, k_pages, v_pages, table, lengths, splits=splits))
        int4_ops.append_int4(*new, k_pages, v_pages, table, lengths - 40)
        outs.append(int4_ops.rope_decode_attention_int4(qkv, k_pages, v_pages, table, lengths, rope, num_q_heads=16, softmax_scale=0.1))
        return outs

    for got, want in zip(run(*high, table), run(*small)):
        assert torch.equal(got, want)
    cuda_ops.check_status()
    for pool, low in zip(high, small):
        assert torch.equal(pool.codes[-b * used:], low.codes) and torch.equal(pool.scales[-b * used:], low.scales)
        assert not pool.codes[:64].any() and not pool.codes[-b * used - 64:-b * used].any()


def test_values_that_are_not_numbers_stay_where_they_belong():
    from axlearn_b200.ops import int4_ops

    k_pages, v_pages, table = _cache(3, 4, 16, 2, 128, seed=6)
    lengths = torch.tensor([60, 60, 1], dtype=torch.int32, device="cuda")
    v_pages.scales[table[0, 1].long(), 1, 3, 2] = torch.tensor([0.0, torch.nan])
    k_pages.scales[table[1, 0].long(), 0, 5, 0] = torch.tensor([0.0, torch.nan])
    k_pages.scales[table[2, 0].long(), 1, 0, 1] = torch.tensor([0.0, torch.nan])   # the sequence's only key
    q = _normal(_gen(5), 3, 4, 128).bfloat16()
    for splits in (1, 2, 9):
        bad = int4_ops.paged_decode_attention_int4(q, k_pages, v_pages, table, lengths, splits=splits).isnan()
        want = torch.zeros_like(bad)
        want[0, 2:, 64:96] = want[1, :2] = want[2, 2:] = True
        assert torch.equal(bad, want)


def test_bad_places_are_reported_and_not_touched():
    from axlearn_b200.ops import cuda_ops, int4_ops

    k_pages, v_pages, table = _cache(2, 4, 16, 2, 128, seed=7)
    q = _normal(_gen(6), 2, 4, 128).bfloat16()
    k = _normal(_gen(7), 2, 3, 2, 128).bfloat16()
    good = torch.tensor([64, 20], dtype=torch.int32, device="cuda")
    want = int4_ops.paged_decode_attention_int4(q, k_pages, v_pages, table, good)
    cuda_ops.check_status()
    out = int4_ops.paged_decode_attention_int4(q, k_pages, v_pages, table, torch.tensor([65, 20], dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="status 5"):
        cuda_ops.check_status()
    assert torch.equal(out, want)
    before = [x.clone() for x in (*k_pages, *v_pages)]
    for page, start in ((11, 0), (-1, 0), (0, 62), (0, -1)):
        bad = table.clone()
        if page:
            bad[0, 0] = page
        at = torch.tensor([start, 61], dtype=torch.int32, device="cuda")
        live = torch.tensor([3, 0], dtype=torch.int32, device="cuda")
        int4_ops.append_int4(k, k, k_pages, v_pages, bad, at, live=live)
        with pytest.raises(RuntimeError, match="status 5"):
            cuda_ops.check_status()
        if page:
            assert all(torch.equal(x, y) for x, y in zip(before, (*k_pages, *v_pages)))
            int4_ops.paged_decode_attention_int4(q, k_pages, v_pages, bad, good)
            with pytest.raises(RuntimeError, match="status 5"):
                cuda_ops.check_status()


@pytest.mark.parametrize("b,t,kv,dim,page_size,packed", [(1, 1, 1, 128, 16, False), (3, 37, 2, 64, 12, True), (5, 9, 3, 128, 1, True),
                                                       (64, 1, 32, 128, 16, True), (2, 700, 8, 128, 64, True), (4, 700, 7, 128, 12, True),
                                                       (6, 900, 8, 64, 16, False)])
@pytest.mark.parametrize("ragged", [False, True])
def test_append_has_the_bits_of_the_plain_statement(b, t, kv, dim, page_size, packed, ragged):
    from axlearn_b200.ops import cuda_ops, int4_ops

    gen, pages = _gen(b), -(-(t + 40) // page_size)
    k_pages, v_pages, table = _cache(b, pages, page_size, kv, dim, seed=t)
    other = [int4_ops.Int4Pages(*(x.clone() for x in p)) for p in (k_pages, v_pages)]
    x = (_normal(gen, b, t, 2 * kv + 1, dim) * torch.exp(3 * _normal(gen, b, t, 2 * kv + 1, 1))).bfloat16()
    x[0, 0, 1] = 2.5                      # no range
    x[0, -1, 1, 3], x[0, -1, -1, -1] = torch.nan, torch.inf
    x[-1, 0, 2, :32], x[-1, 0, 2, 32:64] = 0.0, x[-1, 0, 2, 32:64] * 2.0 ** -126
    k, v = x[:, :, 1:kv + 1], x[:, :, kv + 1:]
    if not packed:
        k, v = k.contiguous(), v.contiguous()
    start = torch.randint(0, 41, (b,), dtype=torch.int32, device="cuda", generator=gen)
    live = torch.randint(0, t + 1, (b,), dtype=torch.int32, device="cuda", generator=gen) if ragged else None
    got = int4_ops.append_int4(k, v, k_pages, v_pages, table, start, live=live, values=True)
    want = _plain(int4_ops.append_int4, k, v, *other, table, start, live=live, values=True)
    cuda_ops.check_status()
    for x, y in zip((*k_pages, *v_pages, *got), (*other[0], *other[1], *want)):
        assert x.dtype == y.dtype and torch.equal(x.nan_to_num(nan=12345.0) if x.is_floating_point() else x,
                                                  y.nan_to_num(nan=12345.0) if y.is_floating_point() else y)


def _linear64(x, w):
    """``(y, bound)`` in 64 bits."""
    from axlearn_b200.ops import int4_ops

    values = _plain(int4_ops.dequantize_weight, w, torch.float32).double()
    y = x.double() @ values
    terms = x.double().abs() @ values.abs()
    if not int4_ops.multiplies_codes(x.shape[0], w.n):
        bound = 2.0 ** -8 * terms + 2.0 ** -23 * w.k * terms  # weights rounded to bf16; sums of k terms in any order
    else:
        # Products with 128 + c of up to 128 values (tensor cores cut sums off at 2^-23 of their largest term), 8 steps a group
        # and a few in 32 bits for every group and warp.
        tiles, groups = w.scales.shape[:2]
        pairs = w.scales.double().abs().permute(0, 3, 2, 1, 4).reshape(tiles * 16, groups, 2)[:w.n]
        size = (pairs @ torch.tensor([271.0, 2.0], device="cuda", dtype=torch.float64)).t()
        xs = torch.nn.functional.pad(x.double().abs(), (0, groups * w.group - w.k)).unflatten(-1, (groups, w.group)).sum(-1)
        bound = (10 + groups / 8 + 8) * 2.0 ** -23 * (xs @ size)
    return y, 1.01 * bound + 2.0 ** -8 * (y.abs() + bound)


@pytest.mark.parametrize("rows", [1, 2, 7, 8, 9, 16, 17, 31, 33, 64, 65, 200])
@pytest.mark.parametrize("k,n,group", [(8, 8, 64), (72, 24, 128), (200, 40, 64), (1096, 328, 128), (2048, 96, 64)])
def test_linear_of_few_and_many_rows(rows, k, n, group):
    from axlearn_b200.ops import cuda_ops, int4_ops

    gen = _gen(rows + k)
    w = int4_ops.quantize_weight(_normal(gen, k, n) * k ** -0.5 + 0.01, group=group)
    x = (_normal(gen, rows, k) * torch.exp(_normal(gen, k))).bfloat16()
    y, bound = _linear64(x, w)
    got = int4_ops.int4_linear(x, w)
    assert got.dtype == torch.bfloat16 and ((got.double() - y).abs() <= bound).all()
    out = _normal(gen, rows, n).bfloat16()
    want = out.double() + y
    assert int4_ops.int4_linear(x, w, out=out, accumulate=True) is out
    cuda_ops.check_status()
    # The sum is rounded again; behind the GEMM it may be added to an unrounded or a rounded product.
    assert ((out.double() - want).abs() <= bound + 2.0 ** -8 * (want.abs() + y.abs() + bound)).all()


@pytest.mark.parametrize("rows", [17, 33, 128])
@pytest.mark.parametrize("k,n,plan", [(640, 1160, (8, 5)), (1096, 264, (5, 8)), (200, 904, (7, 2)), (2048, 392, (1, 3)),
                                      (72, 2056, (6, 1)), (640, 24, (3, 4)), (1096, 648, (4, 1))])
def test_linear_with_slices_of_k_and_narrow_tiles(rows, k, n, plan, monkeypatch):
    """Slices of one to a dozen stages, tiles of one to eight warps, a last tile of few columns and a last stage of few rows."""
    from axlearn_b200.ops import cuda_ops, int4_ops

    gen = _gen(rows + k)
    w = int4_ops.quantize_weight(_normal(gen, k, n) * k ** -0.5, group=64)
    x = _normal(gen, rows, k).bfloat16()
    y, bound = _linear64(x, w)
    monkeypatch.setattr(int4_ops, "fused_plan", lambda *_: plan)
    got = int4_ops.int4_linear(x, w)
    cuda_ops.check_status()
    assert ((got.double() - y).abs() <= bound).all()
    assert torch.equal(got, int4_ops.int4_linear(x, w))


@pytest.mark.parametrize("rows", [8, 9, 16, 17])
@pytest.mark.parametrize("k,n", [(264, 4096), (264, 4104), (8, 4616)])
def test_linear_where_products_with_codes_end(rows, k, n):
    from axlearn_b200.ops import cuda_ops, int4_ops

    gen = _gen(rows + n)
    w = int4_ops.quantize_weight(_normal(gen, k, n) * k ** -0.5, group=64)
    x = _normal(gen, rows, k).bfloat16()
    y, bound = _linear64(x, w)
    got = int4_ops.int4_linear(x, w)
    cuda_ops.check_status()
    assert ((got.double() - y).abs() <= bound).all()
    alone = torch.cat([int4_ops.int4_linear(row, w) for row in x.split(1)])
    assert ((alone.double() - y).abs() <= bound).all()


@pytest.mark.parametrize("rows", [129, 250, 384, 512, 513, 1500])
@pytest.mark.parametrize("k,n,group", [(1096, 136, 64), (2048, 392, 128), (8, 1160, 64), (264, 4616, 128)])
def test_linear_in_blocks_of_rows(rows, k, n, group):
    """A last block of one row and of most rows, with and without slices of K; the first rows behind the blocks."""
    from axlearn_b200.ops import cuda_ops, int4_ops

    gen = _gen(rows + k)
    w = int4_ops.quantize_weight(_normal(gen, k, n) * k ** -0.5, group=group)
    x = _normal(gen, rows, k + 8).bfloat16()[:, :k]
    y, bound = _linear64(x, w)
    out = _normal(gen, rows + 1, n).bfloat16()
    before = out.clone()
    assert ((int4_ops.int4_linear(x, w, out=out[:rows]).double() - y).abs() <= bound).all()
    assert torch.equal(out[rows], before[rows])
    want = before[:rows].double() + y
    got = int4_ops.int4_linear(x, w, out=before[:rows], accumulate=True)
    cuda_ops.check_status()
    assert ((got.double() - want).abs() <= bound + 2.0 ** -8 * (want.abs() + y.abs() + bound)).all()


@pytest.mark.parametrize("rows", [3, 12, 40, 200, 600])
@pytest.mark.parametrize("accumulate", [False, True])
def test_linear_into_a_place_that_is_not_aligned(rows, accumulate):
    from axlearn_b200.ops import cuda_ops, int4_ops

    gen = _gen(rows)
    w = int4_ops.quantize_weight(_normal(gen, 264, 4104) * 264 ** -0.5)
    x = _normal(gen, rows, 264).bfloat16()
    flat = torch.ones(rows * 4104 + 2, dtype=torch.bfloat16, device="cuda")
    out = flat[1:-1].view(rows, 4104)
    want = int4_ops.int4_linear(x, w, out=torch.ones_like(out), accumulate=accumulate)
    assert torch.equal(int4_ops.int4_linear(x, w, out=out, accumulate=accumulate), want)
    cuda_ops.check_status()
    assert flat[0] == 1 and flat[-1] == 1


@pytest.mark.parametrize("rows", [5, 12, 40, 200])
@pytest.mark.parametrize("x_scale,w_scale", [(2.0 ** 40, 2.0 ** 20), (2.0 ** -40, 2.0 ** -40), (2.0 ** 50, 2.0 ** -50)])
def test_linear_of_small_and_large_values(rows, x_scale, w_scale):
    """Powers of two leave every digit as it is."""
    from axlearn_b200.ops import int4_ops

    gen = _gen(rows)
    weights, x = _normal(gen, 520, 4104), _normal(gen, rows, 520).bfloat16()
    plain = int4_ops.int4_linear(x, int4_ops.quantize_weight(weights))
    scaled = int4_ops.int4_linear(x * x_scale, int4_ops.quantize_weight(weights * w_scale))
    assert torch.equal(scaled, plain * (x_scale * w_scale))


def test_products_of_all_kinds_replay_in_graphs_side_by_side():
    """Two graphs of the same weights on two streams at once, each with the bits of separate calls."""
    from axlearn_b200.ops import cuda_ops, int4_ops

    gen = _gen(31)
    w = int4_ops.quantize_weight(_normal(gen, 1032, 4616) * 1032 ** -0.5)
    v = int4_ops.quantize_weight(_normal(gen, 4616, 264) * 4616 ** -0.5, group=64)
    kinds = (1, 12, 40, 128, 300, 600)
    inputs = [[torch.empty(rows, 1032, dtype=torch.bfloat16, device="cuda") for rows in kinds] for _ in range(2)]

    def run(xs):
        return [int4_ops.int4_linear(int4_ops.int4_linear(x, w), v) for x in xs]

    streams, graphs, outs = [torch.cuda.Stream() for _ in range(2)], [], []
    run(inputs[0])
    for xs in inputs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]), cuda_ops.chained_launches():
            outs.append(run(xs))
    for seed in (32, 33, 34):
        for i, xs in enumerate(inputs):
            for x in xs:
                x.copy_(_normal(_gen(2 * seed + i), *x.shape))
        torch.cuda.synchronize()
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for xs, got in zip(inputs, outs):
            assert all(torch.equal(a, b) for a, b in zip(got, run(xs)))
    cuda_ops.check_status()


@pytest.mark.parametrize("rows", [1, 12, 40])
def test_linear_of_codes_beyond_32_bits(rows):
    from axlearn_b200.ops import cuda_ops, int4_ops

    k, n = 16384, 2 ** 33 // 16384 + 128
    if torch.cuda.mem_get_info()[0] < 30 * 2 ** 30:
        pytest.skip("codes of 4.3 GB")
    part = int4_ops.quantize_weight(_normal(_gen(20), k, 64) * k ** -0.5)
    codes = torch.zeros(n // 16, k // 64, 512, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(n // 16, k // 128, 8, 2, 2, dtype=torch.bfloat16, device="cuda")
    codes[-4:], scales[-4:] = part.codes, part.scales
    x = _normal(_gen(rows), rows, k).bfloat16()
    got = int4_ops.int4_linear(x, int4_ops.Int4Weight(codes, scales, k=k, n=n, group=128))
    cuda_ops.check_status()
    values = _plain(int4_ops.dequantize_weight, part, torch.float32).double()
    y, terms = x.double() @ values, x.double().abs() @ values.abs()
    # Weights may be rounded to bf16, the output is, sums of k terms in any order.
    bound = 2.0 ** -8 * terms + 2.0 ** -23 * k * terms
    assert ((got[:, -64:].double() - y).abs() <= bound + 2.0 ** -8 * (y.abs() + bound)).all()
    assert not got[:, :-64].any()


@pytest.mark.parametrize("rows", [3, 40, 90])
def test_linear_takes_strided_rows_and_keeps_rows_apart(rows):
    from axlearn_b200.ops import int4_ops

    gen = _gen(11)
    w = int4_ops.quantize_weight(_normal(gen, 256, 48))
    wide = _normal(gen, 2, rows, 300).bfloat16()
    for x in (wide[0, :, 16:272], wide[0, :, 1:257], wide[:, :, :256], wide[0, :, 44:], wide[0, :256 // rows * 0 + rows, 8:264]):
        assert torch.equal(int4_ops.int4_linear(x, w), int4_ops.int4_linear(x.clone(memory_format=torch.contiguous_format), w))
    x = wide[0, :, :256].clone()
    before = int4_ops.int4_linear(x, w)
    x[rows // 2, 5], x[0, 0] = torch.nan, torch.inf
    after = int4_ops.int4_linear(x, w)
    hit = torch.zeros(rows, dtype=torch.bool, device="cuda")
    hit[0] = hit[rows // 2] = True
    assert torch.equal(before[~hit], after[~hit]) and not after[hit].isfinite().any()
    assert int4_ops.int4_linear(x[:0], w).shape == (0, 48)


@pytest.mark.parametrize("k,n,group", [(8, 8, 128), (200, 40, 64), (1096, 328, 128)])
def test_expanded_weights_have_the_bits_of_the_plain_statement(k, n, group):
    from axlearn_b200.ops import int4_ops

    w = int4_ops.quantize_weight(_normal(_gen(k), k, n), group=group)
    assert torch.equal(int4_ops.dequantize_weight(w), _plain(int4_ops.dequantize_weight, w))


@pytest.mark.parametrize("nq,kv,dim,splits", [(4, 4, 128, 1), (8, 2, 64, 3), (20, 2, 128, 9), (32, 8, 128, None)])
def test_a_step_is_rotation_append_and_attention(nq, kv, dim, splits):
    from axlearn_b200.ops import cuda_ops, decode_ops, int4_ops

    lens = [0, 1, 16, 17, 32, 33, 95, 96]
    b, page_size = len(lens), 16
    k_pages, v_pages, table = _cache(b, 6, page_size, kv, dim, seed=8)
    other = [int4_ops.Int4Pages(*(x.clone() for x in p)) for p in (k_pages, v_pages)]
    rope = decode_ops.rope_table(96, dim, 1e4, "cuda")
    lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")
    qkv = _normal(_gen(9), b, (nq + 2 * kv) * dim).bfloat16()
    given = qkv.clone()
    out = int4_ops.rope_decode_attention_int4(qkv, k_pages, v_pages, table, lengths, rope, num_q_heads=nq, softmax_scale=dim ** -0.5,
                                              splits=splits)
    _plain(int4_ops.rope_decode_attention_int4, qkv, *other, table, lengths, rope, num_q_heads=nq, softmax_scale=dim ** -0.5)
    cuda_ops.check_status()
    assert torch.equal(qkv, given)
    q = qkv.view(b, -1, dim)[:, :nq]
    q = int4_ops._rotate(q[:, None], rope, lengths[:, None].long() - 1)[:, 0]  # pylint: disable=protected-access
    want, bound = _attention64(q, k_pages, v_pages, table, lengths, dim ** -0.5)
    # The rotated query may round the other way where products are fused: 2^-8 of it, as a score's move.
    scale = 2.0 ** -8 * dim ** -0.5 * dim * q.abs().max() * int4_ops.page_values(k_pages).abs().max()
    slack = torch.expm1(2 * scale * 2.0 ** -8) * int4_ops.page_values(v_pages).abs().max()
    assert ((out.double() - want).abs() <= bound + slack).all() and not out[0].any()
    # The new rows: a rotated key may round the other way, which moves a level by one step at most.
    for mine, plain in zip((k_pages, v_pages), other):
        a, c = int4_ops.page_values(mine), int4_ops.page_values(plain)
        step = plain.scales[..., 0].float().repeat_interleave(32, -1)
        assert ((a - c).abs() <= 1.1 * step + 2.0 ** -6 * c.abs()).all()
        assert (a != c).float().mean() < 1e-3
    assert torch.equal(v_pages.codes, other[1].codes) and torch.equal(v_pages.scales, other[1].scales)


def test_scratch_that_does_not_fit_is_refused():
    from axlearn_b200.ops import int4_ops

    k_pages, v_pages, table = _cache(2, 20, 16, 2, 128, seed=7)
    lengths = torch.tensor([320, 77], dtype=torch.int32, device="cuda")
    q = _normal(_gen(8), 2, 8, 128).bfloat16()
    floats = int4_ops.attention_scratch_floats(2, 8, 128, 16)
    whole = torch.empty(floats + 1, device="cuda")
    for scratch in (whole[:-2], whole[1:], whole[:-1].double(), torch.empty(floats)):
        with pytest.raises(ValueError):
            int4_ops.paged_decode_attention_int4(q, k_pages, v_pages, table, lengths, splits=16, scratch=scratch)
    out = int4_ops.paged_decode_attention_int4(q, k_pages, v_pages, table, lengths, splits=16, scratch=whole)
    assert torch.equal(out, int4_ops.paged_decode_attention_int4(q, k_pages, v_pages, table, lengths, splits=16))


def test_a_step_without_a_place_appends_nothing():
    from axlearn_b200.ops import cuda_ops, decode_ops, int4_ops

    k_pages, v_pages, table = _cache(3, 2, 16, 2, 128, seed=20)
    rope = decode_ops.rope_table(40, 128, 1e4, "cuda")
    qkv = _normal(_gen(21), 3, 8 * 128).bfloat16()
    before = [x.clone() for x in (*k_pages, *v_pages)]
    lengths = torch.tensor([33, 0, 20], dtype=torch.int32, device="cuda")
    table[2, 1] = 99                                            # the third sequence's new page is none of the pool's
    out = int4_ops.rope_decode_attention_int4(qkv, k_pages, v_pages, table, lengths, rope, num_q_heads=4, softmax_scale=0.1)
    with pytest.raises(RuntimeError, match="status 5"):
        cuda_ops.check_status()
    assert not out[:2].any() and all(torch.equal(x, y) for x, y in zip(before, (*k_pages, *v_pages)))
    # A position that the rotation table does not have is reported, too.
    table[2, 1] = table[1, 1]
    int4_ops.rope_decode_attention_int4(qkv, k_pages, v_pages, table, torch.tensor([0, 0, 20], dtype=torch.int32, device="cuda"),
                                        rope[:19].contiguous(), num_q_heads=4, softmax_scale=0.1)
    with pytest.raises(RuntimeError, match="status 5"):
        cuda_ops.check_status()


@pytest.mark.parametrize("b,t,nq,kv,dim", [(2, 300, 8, 2, 128), (1, 1, 4, 4, 64), (3, 130, 12, 4, 64), (3, 1300, 6, 2, 128)])
def test_prompts_attend_to_what_the_cache_stands_for(b, t, nq, kv, dim):
    from axlearn_b200.ops import cuda_ops, decode_ops, int4_ops

    k_pages, v_pages, table = _cache(b, -(-t // 16), 16, kv, dim, seed=10)
    rope = decode_ops.rope_table(t, dim, 1e4, "cuda")
    qkv = _normal(_gen(12), b, t, (nq + 2 * kv) * dim).bfloat16()
    given = qkv.clone()
    out = int4_ops.prompt_attention_int4(qkv, k_pages, v_pages, table, rope, num_q_heads=nq, softmax_scale=dim ** -0.5)
    cuda_ops.check_status()
    q, k, v = qkv.view(b, t, -1, dim).split((nq, kv, kv), 2)
    pos = torch.arange(t, device="cuda")
    for x, pages in ((k, k_pages), (v, v_pages)):  # what attention read is what the cache holds
        held = int4_ops.page_values(pages, torch.bfloat16)[table.long()].transpose(2, 3).flatten(1, 2)[:, :t]
        assert torch.equal(x, held)
    g = given.view(b, t, -1, dim)
    turned = int4_ops._rotate(g, rope, pos.expand(b, t))  # pylint: disable=protected-access
    assert ((q.float() - turned[:, :, :nq].float()).abs() <= 2.0 ** -7 * turned[:, :, :nq].float().abs() + 2.0 ** -20).all()
    qq, kk, vv = (x.double().transpose(1, 2) for x in (q, k.repeat_interleave(nq // kv, 2), v.repeat_interleave(nq // kv, 2)))
    seen = pos[:, None] >= pos
    p = torch.softmax((qq @ kk.transpose(2, 3) * dim ** -0.5).masked_fill(~seen, -torch.inf), -1)
    want, size = ((p @ x).transpose(1, 2).flatten(2) for x in (vv, vv.abs()))
    # Probabilities in bf16 and the output's rounding; scores and sums in 32 bits.
    assert ((out.double() - want).abs() <= 2.0 ** -8 * (want.abs() + 1.02 * size) + 2.0 ** -12 * size).all()


def test_calls_replay_in_a_graph_and_on_another_stream():
    """Captured append, step and product: replays see new inputs, and have the bits of separate calls."""
    from axlearn_b200.ops import cuda_ops, decode_ops, int4_ops

    b, nq, kv, dim = 2, 8, 2, 128
    k_pages, v_pages, table = _cache(b, 80, 16, kv, dim, seed=13)
    rope = decode_ops.rope_table(1280, dim, 1e4, "cuda")
    lengths = torch.tensor([700, 9], dtype=torch.int32, device="cuda")
    w = int4_ops.quantize_weight(_normal(_gen(14), 512, (nq + 2 * kv) * dim))
    x = _normal(_gen(15), b, 512).bfloat16()

    def step(cache):
        qkv = int4_ops.int4_linear(x, w)
        return int4_ops.rope_decode_attention_int4(qkv, *cache, table, lengths, rope, num_q_heads=nq, softmax_scale=0.05, splits=9)

    mine = [int4_ops.Int4Pages(*(t.clone() for t in p)) for p in (k_pages, v_pages)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = step(mine)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(warm, step((k_pages, v_pages)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph), cuda_ops.chained_launches():
        out = step(mine)
    for seed in (16, 17, 18):
        lengths.add_(1)
        x.copy_(_normal(_gen(seed), b, 512))
        graph.replay()
        assert torch.equal(out, step((k_pages, v_pages)))
    for p, o in zip(mine, (k_pages, v_pages)):
        row = (table.long().gather(1, (lengths[:, None].long() - 1) // 16)[:, 0], (lengths.long() - 1) % 16)
        assert torch.equal(p.codes[row[0], :, row[1]], o.codes[row[0], :, row[1]])
    cuda_ops.check_status()


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


@pytest.mark.parametrize("weight_bits,cache_bits", [(4, 4), (4, 16), (16, 4)])
@pytest.mark.parametrize("b,nq,nkv", [(1, 4, 4), (5, 8, 2)])
def test_engine_in_4_bits_matches_its_plain_statements(weight_bits, cache_bits, b, nq, nkv):
    """Prompts and steps with the kernels against the same engine on the plain 4-bit statements, the captured step against
    separate launches."""
    from axlearn_b200.inference import decode_engine
    from axlearn_b200.ops import int4_ops

    weights, dims = _engine_weights(256, 520, 1000, nq, nkv, 2, seed=b)
    if weight_bits == 4:
        weights = decode_engine.quantize_weights(weights, group=64)
        assert all(isinstance(lw.wgu, int4_ops.Int4Weight) for lw in weights["layers"])
    ids = torch.randint(0, 1000, (b, 90), device="cuda", generator=_gen(1))
    lengths = torch.randint(1, 71, (b,), device="cuda", generator=_gen(2))
    lengths[0] = 70

    def engine(use_graph):
        return decode_engine.DecodeEngine(weights, dims, batch=b, max_len=96, use_graph=use_graph, cache_bits=cache_bits)

    chained, separate, plain = engine(True), engine(False), engine(False)

    def close():
        # Two layers of some five operations, each of which may round its output the other way (2^-8 of it); norms and
        # residuals pass that on with a gain of about one.  A key or value x that does moves to the next level of its group in
        # 2^-8 |x| / s of the cases, by s: with |x| about 0.8 sigma and s a fifteenth of 4.2 sigma that is sqrt(2 * 2^-8 * 0.8
        # * 0.28) = 0.042 sigma (rms; both sides may move) of keys and values alike, in each layer's attention.
        off = (separate.logits - plain.logits).norm() / plain.logits.norm()
        assert off < 10 * 2.0 ** -8 + (2 * 0.042 if cache_bits == 4 else 0), off

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
def test_engine_steps_in_4_bits_at_serving_widths(batch):
    """Kernels that overlap for long: replays of the chained step against separate launches, bit for bit."""
    from axlearn_b200.inference import decode_engine

    weights, dims = _engine_weights(4096, 14336, 8192, 32, 8, 2, seed=3)
    weights = decode_engine.quantize_weights(weights)
    engines = [decode_engine.DecodeEngine(weights, dims, batch=batch, max_len=2048, use_graph=use, cache_bits=4) for use in (True, False)]
    ids = torch.randint(0, 8192, (batch, 1500), device="cuda", generator=_gen(4))
    lengths = torch.randint(1, 1501, (batch,), device="cuda", generator=_gen(5))
    for e in engines:
        e.prefill(ids, lengths=lengths)
    for i in range(12):
        x, y = (e.step_logits(ids[:, i]).clone() for e in engines)
        assert torch.equal(x, y), i


def test_sample_decode_takes_the_bits_of_the_environment(monkeypatch):
    from axlearn_b200.common import decoding, logit_modifiers, prng
    from axlearn_b200.common.module import functional
    from axlearn_b200.common.utils import tree_map
    from axlearn_b200.inference import decode_engine
    from axlearn_b200.ops import int4_ops
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
    monkeypatch.setenv("AXB200_DECODE_WEIGHT_BITS", "4")
    monkeypatch.setenv("AXB200_DECODE_CACHE_BITS", "4")
    out, _ = functional(model, prng.PRNGKey(5), params, kwargs, is_training=False, method="sample_decode")
    assert out.sequences.shape == (2, 2, 39) and seen[-1].cache_bits == 4
    assert isinstance(seen[-1].w["layers"][0].wo, int4_ops.Int4Weight)
    monkeypatch.delenv("AXB200_DECODE_WEIGHT_BITS")
    functional(model, prng.PRNGKey(5), params, kwargs, is_training=False, method="sample_decode")
    assert seen[-1].cache_bits == 4 and isinstance(seen[-1].w["layers"][0].wo, torch.Tensor)
    monkeypatch.setenv("AXB200_DECODE_CACHE_BITS", "8")
    with pytest.raises(ValueError, match="4 or 16"):
        functional(model, prng.PRNGKey(5), params, kwargs, is_training=False, method="sample_decode")


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_the_plain_attention_on_the_gpu_reads_the_sequences_pages_alone(dtype):
    """Types without a kernel, and the plain statement asked for: tables with anything behind a sequence, bad places reported."""
    from axlearn_b200.ops import cuda_ops, int4_ops

    k_pages, v_pages, table = _cache(3, 4, 16, 2, 64, seed=31)
    lengths = torch.tensor([5, 33, 0], dtype=torch.int32, device="cuda")
    q = _normal(_gen(32), 3, 4, 64)
    want = int4_ops.paged_decode_attention_int4(q.to(dtype), k_pages, v_pages, table, lengths)
    reference = _plain(int4_ops.paged_decode_attention_int4, q.bfloat16(), k_pages, v_pages, table, lengths)
    table[0, 1:], table[1, 3:], table[2] = 10 ** 9, -7, 99
    assert torch.equal(int4_ops.paged_decode_attention_int4(q.to(dtype), k_pages, v_pages, table, lengths), want)
    assert torch.equal(_plain(int4_ops.paged_decode_attention_int4, q.bfloat16(), k_pages, v_pages, table, lengths), reference)
    assert not want[2].any()
    cuda_ops.check_status()
    table[0, 0] = 99
    out = int4_ops.paged_decode_attention_int4(q.to(dtype), k_pages, v_pages, table, lengths)
    with pytest.raises(RuntimeError, match="status 5"):
        cuda_ops.check_status()
    assert torch.equal(out[1:], want[1:]) and not out[0].any()


def test_the_plain_append_on_the_gpu_reports_places_that_are_not_there():
    from axlearn_b200.ops import cuda_ops, int4_ops

    k_pages, v_pages, table = _cache(2, 4, 16, 2, 128, seed=33)
    k = _normal(_gen(34), 2, 3, 2, 128)
    before = [x.clone() for x in (*k_pages, *v_pages)]
    live = torch.tensor([3, 0], dtype=torch.int32, device="cuda")
    for page, start in ((11, 0), (-1, 0), (0, 64), (0, -3)):
        bad = table.clone()
        if page:
            bad[0, 0] = page
        int4_ops.append_int4(k, k, k_pages, v_pages, bad, torch.tensor([start, 70], dtype=torch.int32, device="cuda"), live=live)
        with pytest.raises(RuntimeError, match="status 5"):
            cuda_ops.check_status()
        assert all(torch.equal(x, y) for x, y in zip(before, (*k_pages, *v_pages)))
    int4_ops.append_int4(k, k, k_pages, v_pages, table[:, :0].contiguous(), torch.zeros_like(live), live=live)
    with pytest.raises(RuntimeError, match="status 5"):
        cuda_ops.check_status()
    int4_ops.append_int4(k, k, k_pages, v_pages, table, torch.zeros_like(live), live=live)
    cuda_ops.check_status()


@pytest.mark.parametrize("dim,splits", [(128, 1), (64, 3), (128, 16)])
@pytest.mark.parametrize("plain", [False, True])
def test_a_step_behind_the_rotation_table_appends_nothing(dim, splits, plain):
    from axlearn_b200.ops import cuda_ops, decode_ops, int4_ops

    k_pages, v_pages, table = _cache(3, 8, 16, 2, dim, seed=35)
    rope = decode_ops.rope_table(128, dim, 1e4, "cuda")
    qkv = _normal(_gen(36), 3, 8 * dim).bfloat16()

    def step(cache, positions, lengths):
        call = _plain if plain else (lambda fn, *args, **kwargs: fn(*args, **kwargs))
        return call(int4_ops.rope_decode_attention_int4, qkv, *cache, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                    rope[:positions].contiguous(), num_q_heads=4, softmax_scale=0.1, splits=splits)

    caches = [[int4_ops.Int4Pages(*(x.clone() for x in p)) for p in (k_pages, v_pages)] for _ in range(2)]
    out = step(caches[0], 70, [100, 70, 71])          # the last position of the table is 69
    with pytest.raises(RuntimeError, match="status 5"):
        cuda_ops.check_status()
    want = step(caches[1], 128, [0, 70, 0])
    cuda_ops.check_status()
    assert torch.equal(out, want) and not out[0].any() and out[1].any() and not out[2].any()
    for x, y in zip(caches[0], caches[1]):
        assert torch.equal(x.codes, y.codes) and torch.equal(x.scales, y.scales)


@pytest.mark.parametrize("splits", [None, 1, 8, 9, 16])
def test_empty_calls(splits):
    from axlearn_b200.ops import cuda_ops, decode_ops, int4_ops

    k_pages, v_pages, _ = _cache(2, 3, 16, 2, 128, seed=37)
    before = [x.clone() for x in (*k_pages, *v_pages)]
    table, none = (torch.zeros(0, *shape, dtype=torch.int32, device="cuda") for shape in ((200,), ()))
    rope = decode_ops.rope_table(3200, 128, 1e4, "cuda")
    q, qkv = (torch.empty(0, *shape, dtype=torch.bfloat16, device="cuda") for shape in ((4, 128), (1024,)))
    assert int4_ops.paged_decode_attention_int4(q, k_pages, v_pages, table, none, splits=splits).shape == (0, 4, 128)
    assert int4_ops.rope_decode_attention_int4(qkv, k_pages, v_pages, table, none, rope, num_q_heads=4, softmax_scale=0.1,
                                               splits=splits).shape == (0, 4, 128)
    for b, t in ((0, 5), (2, 0)):
        table, start = (torch.zeros(b, *shape, dtype=torch.int32, device="cuda") for shape in ((200,), ()))
        rows = torch.empty(b, t, 2, 128, dtype=torch.bfloat16, device="cuda")
        assert int4_ops.append_int4(rows, rows, k_pages, v_pages, table, start, values=True)[0].shape == rows.shape
        prompt = torch.empty(b, t, 1024, dtype=torch.bfloat16, device="cuda")
        assert int4_ops.prompt_attention_int4(prompt, k_pages, v_pages, table, rope, num_q_heads=4, softmax_scale=0.1).shape == (b, t, 512)
    cuda_ops.check_status()
    assert all(torch.equal(x, y) for x, y in zip(before, (*k_pages, *v_pages)))


def test_differentiated_operands_are_refused():
    from axlearn_b200.ops import int4_ops

    k_pages, v_pages, table = _cache(2, 3, 16, 2, 128, seed=38)
    lengths = torch.tensor([3, 40], dtype=torch.int32, device="cuda")
    q, w = _normal(_gen(39), 2, 4, 128).bfloat16(), int4_ops.quantize_weight(_normal(_gen(40), 512, 64))
    calls = [(q, lambda x: int4_ops.paged_decode_attention_int4(x, k_pages, v_pages, table, lengths)),
             (q.view(2, 512), lambda x: int4_ops.int4_linear(x, w)),
             (q.view(2, 2, 2, 128), lambda x: int4_ops.append_int4(x, q.view(2, 2, 2, 128), k_pages, v_pages, table, lengths))]
    for x, fn in calls:
        fn(x)
        with pytest.raises(ValueError, match="no gradient"):
            fn(x.clone().requires_grad_())
        with torch.no_grad():
            fn(x.clone().requires_grad_())
        with torch.autograd.forward_ad.dual_level(), pytest.raises(ValueError, match="no gradient"):
            fn(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)))


@pytest.mark.parametrize("rows", [3, 16, 40, 200, 600])
@pytest.mark.parametrize("k", [264, 2048, 4104])
@pytest.mark.parametrize("accumulate", [False, True])
def test_linear_in_place(rows, k, accumulate):
    """``out`` is x, or begins a row before or behind it."""
    from axlearn_b200.ops import cuda_ops, int4_ops

    gen = _gen(rows + k)
    w = int4_ops.quantize_weight(_normal(gen, k, k) * k ** -0.5)
    flat = _normal(gen, rows + 2, k).bfloat16()
    for start in (0, 1, 2):
        buffer = flat.clone()
        x, out = buffer[1:rows + 1], buffer[start:start + rows]
        want = int4_ops.int4_linear(x.clone(), w, out=out.clone(), accumulate=accumulate)
        assert torch.equal(int4_ops.int4_linear(x, w, out=out, accumulate=accumulate), want)
    cuda_ops.check_status()


@pytest.mark.parametrize("nq,kv,dim,splits", [(8, 2, 128, 1), (8, 8, 64, 8), (40, 2, 128, 3), (4, 1, 128, 16)])
def test_attention_in_place(nq, kv, dim, splits):
    from axlearn_b200.ops import int4_ops

    k_pages, v_pages, table = _cache(9, 40, 16, kv, dim, seed=41)
    lengths = torch.arange(0, 9, dtype=torch.int32, device="cuda") * 80
    flat = _normal(_gen(42), 9 * nq * dim + 64).bfloat16()
    for start in (0, 16, 64):
        buffer = flat.clone()
        q, out = buffer[:-64].view(9, nq, dim), buffer[start:start + 9 * nq * dim].view(9, nq, dim)
        want = int4_ops.paged_decode_attention_int4(q.clone(), k_pages, v_pages, table, lengths, splits=splits)
        assert torch.equal(int4_ops.paged_decode_attention_int4(q, k_pages, v_pages, table, lengths, splits=splits, out=out), want)


@pytest.mark.parametrize("nq,kv,dim,splits", [(4, 4, 128, 1), (8, 2, 64, 3), (20, 2, 128, 9), (24, 3, 64, 8), (32, 8, 128, None)])
@pytest.mark.parametrize("page_size", [16, 12])
def test_a_step_with_exact_rotations(nq, kv, dim, splits, page_size):
    """Quarter turns: products with 0 and 1 are exact, so what is appended has the plain statement's bits and the output keeps to
    the bound of attention alone.  The new key is like its first head's query and takes most of that head's weight."""
    from axlearn_b200.ops import cuda_ops, int4_ops

    lens = [1, 2, 16, 17, 32, 33, 95, 96, 97, 127, 128, 129, 300]
    b = len(lens)
    k_pages, v_pages, table = _cache(b, -(-300 // page_size), page_size, kv, dim, seed=43)
    other = [int4_ops.Int4Pages(*(x.clone() for x in p)) for p in (k_pages, v_pages)]
    lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")
    turns = (torch.arange(300, device="cuda")[:, None] + torch.arange(dim // 2, device="cuda")) % 4
    rope = torch.tensor([[0.0, 1.0], [1.0, 0.0], [0.0, -1.0], [-1.0, 0.0]], device="cuda")[turns].contiguous()
    qkv = _normal(_gen(44), b, nq + 2 * kv, dim).bfloat16()
    qkv[:, nq:nq + kv] = 2 * qkv[:, :nq:nq // kv]
    args = dict(num_q_heads=nq, softmax_scale=dim ** -0.5)
    out = int4_ops.rope_decode_attention_int4(qkv.flatten(1), k_pages, v_pages, table, lengths, rope, splits=splits, **args)
    _plain(int4_ops.rope_decode_attention_int4, qkv.flatten(1), *other, table, lengths, rope, **args)
    cuda_ops.check_status()
    for mine, plain in zip((k_pages, v_pages), other):
        assert torch.equal(mine.codes, plain.codes) and torch.equal(mine.scales, plain.scales)
    q = int4_ops._rotate(qkv[:, None, :nq], rope, lengths[:, None].long() - 1)[:, 0]  # pylint: disable=protected-access
    want, bound = _attention64(q, k_pages, v_pages, table, lengths, dim ** -0.5)
    assert ((out.double() - want).abs() <= bound).all()
    without, _ = _attention64(q, k_pages, v_pages, table, lengths - 1, dim ** -0.5)
    first = slice(None, None, nq // kv)
    assert (((want - without).abs() > 8 * bound)[:, first].float().mean((1, 2)) > 0.8).all()


@pytest.mark.parametrize("dim", [64, 128])
def test_attention_up_to_the_ranges_of_its_documentation(dim):
    """Queries up to 2^63, steps and smallest values up to 2^55 over the number of tokens: powers of two leave every digit."""
    from axlearn_b200.ops import int4_ops

    k_pages, v_pages, table = _cache(2, 20, 16, 2, dim, seed=45)
    lengths = torch.tensor([320, 77], dtype=torch.int32, device="cuda")
    q = _normal(_gen(46), 2, 8, dim).bfloat16()
    q_scale = 2.0 ** (62 - math.ceil(math.log2(q.abs().max().item())))
    v_scale = 2.0 ** (54 - math.ceil(math.log2(320 * v_pages.scales.abs().max().item())))
    plain = int4_ops.paged_decode_attention_int4(q, k_pages, v_pages, table, lengths)
    k_pages, v_pages = k_pages._replace(scales=k_pages.scales / q_scale), v_pages._replace(scales=v_pages.scales * v_scale)
    for splits in (1, 4, 16):
        out = int4_ops.paged_decode_attention_int4(q * q_scale, k_pages, v_pages, table, lengths, splits=splits)
        assert out.isfinite().all()
    assert torch.equal(int4_ops.paged_decode_attention_int4(q * q_scale, k_pages, v_pages, table, lengths), plain * v_scale)
