"""bchip_attention_paged against the formula in 64 bits: sequences of pieces of prompts, verify passes and
single tokens over shuffled pages whose unused slots hold NaN, both cache types."""
import numpy as np
import pytest

import bchip
import q4_plain as Q
from paged_plain import Batch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    with bchip.Ctx(0) as c:
        yield c


def call(ctx, b, q, nh, scale, out=None):
    kb, vb, qb = ctx.upload(b.k), ctx.upload(b.v), ctx.upload(q)
    ob = ctx.upload(np.full(q.shape, 7.0, np.float32) if out is None else out)
    starts, lens, table, *rest = b.args(ctx)
    ctx.attention_paged(qb, kb, vb, b.kv_type, ob, starts, lens, table, *rest, nh, b.nkv, b.hd, scale)
    got = ctx.read(ob, q.shape)
    for x in (kb, vb, qb, ob, table):
        x.free()
    return got


def expect(b, q, nh, scale, only=None):
    """Per sequence: rows' results, and how far an f32-grade one may lie. (The bound's terms hold for f32 caches too. By
    f32 products: hd of them, each sum's rounding 2^-24. In three bf16 parts: what is left out of a product, twice
    2^-7 2^-16 of it, is 2^-22, as with two f16; the first parts' sums round 16 times an MFMA, hd / 32 of
    them, and the five others', 5 hd / 2 times, at 2^-7 of that: less than hd in all.)"""
    for i, (n, m) in enumerate(zip(b.rows, b.lens)):
        if n == 0 or (only is not None and i not in only):
            continue
        a = int(b.starts[i])
        k, v = (b.of(p, i).astype(np.float64) for p in (b.k, b.v))
        visible = np.arange(m)[None] <= (m - n + np.arange(n))[:, None]
        want, mass, top = Q.attention(q[a:a + n], k, v, b.nkv, visible, scale)
        yield i, slice(a, a + n), want, Q.bound(mass, top, b.hd)


def check(ctx, b, q, nh, scale):
    got = call(ctx, b, q, nh, scale)
    for i, at, want, most in expect(b, q, nh, scale):
        off = np.abs(got[at] - want)
        assert np.isfinite(got[at]).all(), f"sequence {i}: not finite"
        assert (off <= most).all(), f"sequence {i}: off by {off.max()} ({(off / most).max()} of the bound)"
    assert (got[int(b.starts[-1]):] == 7.0).all(), "a padded row was written"
    return got


SHAPES = [(14, 2, 64), (32, 8, 128), (28, 4, 128), (8, 8, 32), (6, 2, 80), (12, 4, 96), (16, 4, 256), (16, 1, 128), (4, 2, 8),
          (5, 1, 160), (6, 3, 72), (2, 2, 200)]


@pytest.mark.parametrize("kv_type", [bchip.F16, bchip.F32])
@pytest.mark.parametrize("shape", SHAPES)
def test_steps_of_ragged_lists(ctx, shape, kv_type):
    nh, nkv, hd = shape
    rng = np.random.default_rng(nh * hd + kv_type)
    lens = [1, 2, 15, 16, 17, 31, 33, 64, 127, 300, 641, 1000]
    b = Batch(rng, [1] * len(lens), lens, nkv, hd, kv_type, pad=2)
    q = (2 * rng.standard_normal((b.total, nh, hd))).astype(np.float32)
    check(ctx, b, q, nh, hd ** -0.5)


@pytest.mark.parametrize("kv_type", [bchip.F16, bchip.F32])
@pytest.mark.parametrize("shape", SHAPES)
def test_one_short_list(ctx, shape, kv_type):
    nh, nkv, hd = shape
    rng = np.random.default_rng(nh * hd + 7 + kv_type)
    for n in (1, 16, 40, 333):
        b = Batch(rng, [1], [n], nkv, hd, kv_type)
        q = (2 * rng.standard_normal((1, nh, hd))).astype(np.float32)
        check(ctx, b, q, nh, hd ** -0.5)


@pytest.mark.parametrize("kv_type", [bchip.F16, bchip.F32])
@pytest.mark.parametrize("shape", SHAPES)
def test_verify_passes(ctx, shape, kv_type):
    nh, nkv, hd = shape
    rng = np.random.default_rng(nh * hd + 1 + kv_type)
    b = Batch(rng, [2, 3, 5, 1, 8], [2, 50, 600, 1, 1500], nkv, hd, kv_type, page_slots=32, pad=1)
    q = (2 * rng.standard_normal((b.total, nh, hd))).astype(np.float32)
    check(ctx, b, q, nh, hd ** -0.5)


@pytest.mark.parametrize("kv_type", [bchip.F16, bchip.F32])
@pytest.mark.parametrize("shape", SHAPES)
def test_pieces_of_prompts_and_steps_in_one_batch(ctx, shape, kv_type):
    nh, nkv, hd = shape
    rng = np.random.default_rng(nh * hd + 2 + kv_type)
    rows, lens = [33, 0, 1, 70, 1, 17, 0], [33, 5, 90, 200, 1, 300, 64]
    b = Batch(rng, rows, lens, nkv, hd, kv_type, page_slots=64, pad=5, stride=9)
    q = (2 * rng.standard_normal((b.total, nh, hd))).astype(np.float32)
    check(ctx, b, q, nh, hd ** -0.5)


@pytest.mark.parametrize("kv_type", [bchip.F16, bchip.F32])
@pytest.mark.parametrize("shape,rows,before", [((32, 8, 128), 300, 700), ((14, 2, 64), 501, 300), ((8, 8, 32), 257, 0), ((2, 2, 256), 200, 100),
                                               ((4, 1, 96), 400, 1200)])
def test_longer_pieces(ctx, shape, rows, before, kv_type):
    nh, nkv, hd = shape
    rng = np.random.default_rng(rows + kv_type)
    b = Batch(rng, [rows], [rows + before], nkv, hd, kv_type)
    q = (2 * rng.standard_normal((b.total, nh, hd))).astype(np.float32)
    check(ctx, b, q, nh, hd ** -0.5)


@pytest.mark.parametrize("kv_type", [bchip.F16, bchip.F32])
def test_a_wide_pass(ctx, kv_type):
    """Enough query rows for 32 of them a wave (f16)."""
    rng = np.random.default_rng(3)
    b = Batch(rng, [700, 650], [700, 800], 16, 64, kv_type)
    q = (2 * rng.standard_normal((b.total, 32, 64))).astype(np.float32)
    check(ctx, b, q, 32, 0.125)


@pytest.mark.parametrize("kv_type", [bchip.F16, bchip.F32])
@pytest.mark.parametrize("page_slots", [16, 32, 128, 1024])
def test_page_sizes(ctx, page_slots, kv_type):
    rng = np.random.default_rng(page_slots)
    b = Batch(rng, [1, 40, 3], [777, 100, 1025], 2, 64, kv_type, page_slots=page_slots)
    q = rng.standard_normal((b.total, 8, 64)).astype(np.float32)
    check(ctx, b, q, 8, 0.125)


@pytest.mark.parametrize("kv_type", [bchip.F16, bchip.F32])
def test_more_sequences_than_a_launch_takes(ctx, kv_type):
    rng = np.random.default_rng(11)
    lens = rng.integers(1, 90, 256).tolist()
    rows = [min(n, 1 if i % 3 else 20) for i, n in enumerate(lens)]
    b = Batch(rng, rows, lens, 1, 32, kv_type)
    q = rng.standard_normal((b.total, 4, 32)).astype(np.float32)
    check(ctx, b, q, 4, 32 ** -0.5)


@pytest.mark.parametrize("kv_type", [bchip.F16, bchip.F32])
def test_a_long_list(ctx, kv_type):
    rng = np.random.default_rng(12)
    b = Batch(rng, [1, 1], [40000, 9], 2, 64, kv_type, page_slots=16)
    q = (2 * rng.standard_normal((2, 14, 64))).astype(np.float32)
    check(ctx, b, q, 14, 0.125)


@pytest.mark.parametrize("kv_type", [bchip.F16, bchip.F32])
def test_sizes_of_queries(ctx, kv_type):
    """Queries of 0, tiny and large ones: every row has its own power of two; scales of either sign."""
    rng = np.random.default_rng(13)
    b = Batch(rng, [1, 24, 4], [200, 150, 90], 2, 64, kv_type)
    q = rng.standard_normal((b.total, 8, 64)).astype(np.float32)
    q[::5] *= 1e-20
    q[1::5] *= 300.0
    q[2::5] = 0.0
    check(ctx, b, q, 8, 0.125)
    check(ctx, b, q, 8, -0.03)


@pytest.mark.parametrize("kv_type", [bchip.F16, bchip.F32])
def test_reruns_and_neighbours(ctx, kv_type):
    """The same call gives the same bits; a sequence alone agrees with itself in a batch to f32 rounding."""
    rng = np.random.default_rng(14)
    b = Batch(rng, [1, 90, 6, 1], [3000, 400, 2000, 7], 4, 128, kv_type)
    q = (2 * rng.standard_normal((b.total, 16, 128))).astype(np.float32)
    got = check(ctx, b, q, 16, 128 ** -0.5)
    np.testing.assert_array_equal(got.view(np.uint32), call(ctx, b, q, 16, 128 ** -0.5).view(np.uint32))
    for i, at, want, most in expect(b, q, 16, 128 ** -0.5):
        alone = Batch.__new__(Batch)
        alone.__dict__ |= {**b.__dict__, "rows": [b.rows[i]], "lens": [b.lens[i]], "starts": np.array([0, b.rows[i]], np.uint32),
                           "table": b.table[i:i + 1]}
        assert (np.abs(call(ctx, alone, q[at], 16, 128 ** -0.5) - want) <= most).all()


@pytest.mark.parametrize("kv_type", [bchip.F16, bchip.F32])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("rows,n", [(6, 40), (6, 900), (60, 200), (130, 130)])
def test_values_that_are_not_finite_reach_only_rows_that_see_them(ctx, rows, n, bad, kv_type):
    """Such a K or V in a slot that some rows of a pass see and some do not, in K and V apart."""
    rng = np.random.default_rng(15)
    for which in ("k", "v"):
        b = Batch(rng, [rows, 1], [n, 50], 2, 64, kv_type)
        q = rng.standard_normal((b.total, 4, 64)).astype(np.float32)
        p, o = b.places(0)
        slot = n - rows // 2  # the rows from here on see it
        good = [x.copy() for x in (b.k, b.v)]
        getattr(b, which)[p[slot], o[slot], 1, 3] = bad
        got = call(ctx, b, q, 4, 0.125)
        first = slot - (n - rows)
        b.k, b.v = good
        for i, at, want, most in expect(b, q, 4, 0.125):
            ok = np.abs(got[at] - want) <= most
            if i == 0:
                ok[first:, 2:] = True  # unspecified: rows that see the slot, heads of that KV head
            assert ok.all(), f"{which} {bad}: sequence {i}, rows {np.flatnonzero(~ok.all((1, 2)))}"


@pytest.mark.parametrize("kv_type", [bchip.F16, bchip.F32])
def test_queries_that_are_not_finite(ctx, kv_type):
    rng = np.random.default_rng(16)
    for rows in (1, 4, 40):
        b = Batch(rng, [rows, 1], [100, 50], 2, 64, kv_type)
        q = rng.standard_normal((b.total, 4, 64)).astype(np.float32)
        clean = q.copy()
        q[rows // 2, 1, 5] = np.nan
        q[rows // 2, 2, 5] = np.inf
        got = call(ctx, b, q, 4, 0.125)
        assert np.isnan(got[rows // 2, 1]).all()
        for i, at, want, most in expect(b, clean, 4, 0.125):
            ok = np.abs(got[at] - want) <= most
            if i == 0:
                ok[rows // 2, 1:3] = True
            assert ok.all()


@pytest.mark.parametrize("kv_type", [bchip.F16, bchip.F32])
@pytest.mark.parametrize("rows,n", [(1, 40), (1, 2000), (5, 300), (50, 300)])
def test_a_page_past_the_pool_gives_nan_and_nothing_else(ctx, rows, n, kv_type):
    """The rows that see a slot of it; the other sequences, and rows before it, as ever."""
    rng = np.random.default_rng(17)
    for number in (0xFFFFFFFF, None):
        b = Batch(rng, [rows, 1], [n, 70], 2, 64, kv_type)
        q = rng.standard_normal((b.total, 4, 64)).astype(np.float32)
        at_page = (n - 1) // 16  # the last page: rows that end before it do not see it
        kept = b.table[0, at_page]
        b.table[0, at_page] = b.npages if number is None else number
        got = call(ctx, b, q, 4, 0.125)
        b.table[0, at_page] = kept
        for i, at, want, most in expect(b, q, 4, 0.125):
            sees = (n - rows + np.arange(at.stop - at.start) >= 16 * at_page) if i == 0 else np.zeros(1, bool)
            assert np.isnan(got[at][sees]).all()
            assert (np.abs(got[at] - want) <= most)[~sees].all()


@pytest.mark.parametrize("kv_type", [bchip.F16, bchip.F32])
def test_pages_past_4_gb(ctx, kv_type):
    """A pool of 4.5 GB a buffer whose sequences' pages lie around and past 2^32 bytes: append, attention and
    copies as over a small pool."""
    nh, nkv, hd, es = 16, 8, 128, 2 if kv_type == bchip.F16 else 4
    page_bytes = 16 * nkv * hd * es
    npages = int(4.5 * 2 ** 30) // page_bytes
    edge = 2 ** 32 // page_bytes
    rng = np.random.default_rng(18)
    b = Batch(rng, [1, 40], [70, 100], nkv, hd, kv_type)
    high = np.concatenate([[edge - 1, edge, npages - 1, 3], edge + 1 + np.arange(b.npages - 4)]).astype(np.uint32)  # a page's place in the large pool
    big = [ctx.zeros(npages * page_bytes) for _ in range(2)]
    for pool, buf in zip((b.k, b.v), big):
        for page, at in zip(pool, high):
            ctx.upload(page, buf, int(at) * page_bytes)
    table = np.where(b.table < b.npages, high[np.minimum(b.table, b.npages - 1)], 0xFFFFFFFF).astype(np.uint32)
    q = rng.standard_normal((b.total, nh, hd)).astype(np.float32)
    kn, vn = (rng.standard_normal((b.total, nkv, hd)).astype(np.float32) for _ in range(2))
    positions = np.concatenate([np.arange(m - n, m) for n, m in zip(b.rows, b.lens)]).astype(np.uint32)
    inv = ctx.upload(np.ones(hd // 2, np.float32))
    outs = []
    for (kc, vc), tab, pages in ((big, table, npages), ([ctx.upload(b.k), ctx.upload(b.v)], b.table, b.npages)):
        qb, kb, vb, pb, tb, ob = (ctx.upload(x) for x in (q, kn, vn, positions, tab, np.zeros_like(q)))
        ctx.rope_append_paged(qb, kb, vb, kc, vc, kv_type, inv, pb, b.starts, b.lens, tb, b.stride, 16, pages, nh, nkv, hd, hd, True)
        ctx.attention_paged(qb, kc, vc, kv_type, ob, b.starts, b.lens, tb, b.stride, 16, pages, nh, nkv, hd, 0.1)
        last = int(tab[1, 6])
        free = 1 if pages == npages else [p for p in range(b.npages) if p not in b.table][0]
        ctx.copy_pages([kc, vc], kv_type, 16 * nkv * hd, pages, [last], [free])
        bits = np.uint16 if es == 2 else np.uint32
        outs.append([ctx.read(ob, q.size, np.uint32)] + [ctx.read(x, 16 * nkv * hd, bits, at * page_bytes) for x in (kc, vc) for at in (last, free)])
    for x, y in zip(*outs):
        np.testing.assert_array_equal(x, y)
    assert np.isfinite(outs[0][0].view(np.float32)).all()
    for buf in big:
        buf.free()


def test_two_contexts_at_once(ctx):
    """Calls queued on two contexts beside each other, each with scratch of its own."""
    rng = np.random.default_rng(19)
    with bchip.Ctx(0) as other:
        work = []
        for c, (rows, lens) in ((ctx, ([1, 1, 30], [9000, 4000, 700])), (other, ([1, 64], [12000, 3000]))):
            b = Batch(rng, rows, lens, 4, 128, bchip.F16)
            q = rng.standard_normal((b.total, 16, 128)).astype(np.float32)
            want = call(c, b, q, 16, 0.1)
            kb, vb, qb, ob = (c.upload(x) for x in (b.k, b.v, q, np.zeros_like(q)))
            starts, ln, table, *rest = b.args(c)
            work.append((c, lambda c=c, a=(qb, kb, vb, bchip.F16, ob, starts, ln, table, *rest, 16, 4, 128, 0.1): c.attention_paged(*a), ob, want))
        for _ in range(10):
            for _, go, _, _ in work:
                go()
        for c, _, ob, want in work:
            np.testing.assert_array_equal(c.read(ob, want.shape).view(np.uint32), want.view(np.uint32))


@pytest.mark.parametrize("rows", [1, 6, 40, 200])
@pytest.mark.parametrize("hd", [64, 128])
def test_f32_values_of_any_size(ctx, rows, hd):
    """An f32 cache keeps f32's range: dims of K and of V, and slots of V, 2^60 apart, as near as others."""
    rng = np.random.default_rng(20 + rows)
    b = Batch(rng, [rows, 1], [rows + 300, 50], 2, hd, bchip.F32)
    size = 2.0 ** rng.integers(-30, 31, hd)
    b.k *= size.astype(np.float32)
    b.v *= (2.0 ** rng.integers(-30, 31, hd)).astype(np.float32)
    b.v *= (2.0 ** rng.integers(-30, 31, (b.npages, 16, 1, 1))).astype(np.float32)
    q = (rng.standard_normal((b.total, 4, hd)) / size).astype(np.float32)
    check(ctx, b, q, 4, hd ** -0.5)


@pytest.mark.parametrize("kv_type", [bchip.F16, bchip.F32])
@pytest.mark.parametrize("shape", [(16, 4, 128), (14, 2, 64)])
@pytest.mark.parametrize("rows,lens", [([1] * 40 + [100], [2000] * 40 + [100]), ([1, 1, 2, 200], [3000, 900, 1500, 200]),
                                       ([3, 3, 200, 90], [3000, 800, 200, 400]), ([1, 1, 1, 20, 12], [2500] * 5), ([600], [1500]),
                                       ([3, 60, 60, 60], [4000, 60, 60, 90]), ([300, 1], [300, 6000])])
def test_batches_that_are_cut_in_different_ways(ctx, rows, lens, shape, kv_type):
    """Many long steps beside a piece of a prompt, few beside a large one, prompts alone, from their start and
    before many slots: blocks of 64 and of 128 query rows, steps of 8 query rows and of 16, whole lists and chunks."""
    nh, nkv, hd = shape
    rng = np.random.default_rng(len(rows) * hd)
    b = Batch(rng, rows, lens, nkv, hd, kv_type, pad=2)
    q = (2 * rng.standard_normal((b.total, nh, hd))).astype(np.float32)
    check(ctx, b, q, nh, hd ** -0.5)
