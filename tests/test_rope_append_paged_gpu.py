"""bchip_rope_append_paged against bchip_rope_append, bit for bit, and what it leaves alone; bchip_copy_pages."""
import numpy as np
import pytest

import bchip
import oracle as O
from paged_plain import DTYPE, Batch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    with bchip.Ctx(0) as c:
        yield c


def appended(ctx, b, q, k, v, positions, nh, rope_dim, neox):
    """q and the pools after the call."""
    inv = ctx.upload(O.inv_freq(rope_dim, 1e4) if rope_dim else np.zeros(1, np.float32))
    bufs = [ctx.upload(x) for x in (q, k, v, b.k, b.v)]
    pb = ctx.upload(positions)
    starts, lens, table, *rest = b.args(ctx)
    ctx.rope_append_paged(*bufs, b.kv_type, inv, pb, starts, lens, table, *rest, nh, b.nkv, b.hd, rope_dim, neox)
    got = ctx.read(bufs[0], q.shape), ctx.read(bufs[3], b.k.shape, b.k.dtype), ctx.read(bufs[4], b.v.shape, b.v.dtype)
    for x in (*bufs, inv, pb, table):
        x.free()
    return got


def bits(x):
    return np.ascontiguousarray(x).view(np.uint16 if x.dtype == np.float16 else np.uint32)


def check(ctx, b, nh, rope_dim, neox, rng, far=0):
    n = int(b.starts[-1])
    q = rng.standard_normal((b.total, nh, b.hd)).astype(np.float32)
    k, v = (rng.standard_normal((b.total, b.nkv, b.hd)).astype(np.float32) for _ in range(2))
    positions = np.zeros(b.total, np.uint32)
    for i, (r, m) in enumerate(zip(b.rows, b.lens)):
        positions[b.starts[i]:b.starts[i + 1]] = np.arange(m - r, m) + far
    got_q, got_k, got_v = appended(ctx, b, q, k, v, positions, nh, rope_dim, neox)
    # The same rows by the call over a contiguous cache.
    inv = ctx.upload(O.inv_freq(rope_dim, 1e4) if rope_dim else np.zeros(1, np.float32))
    bufs = [ctx.upload(x) for x in (q[:n], k[:n], v[:n])]
    kc, vc, pb = (ctx.zeros(n * b.nkv * b.hd * b.k.itemsize) for _ in range(3))
    pb = ctx.upload(positions)
    ctx.rope_append(*bufs, kc, vc, b.kv_type, inv, pb, n, nh, b.nkv, b.hd, rope_dim, neox, 0)
    want_q = ctx.read(bufs[0], (n, nh, b.hd))
    rk, rv = (ctx.read(x, (n, b.nkv, b.hd), DTYPE[b.kv_type]) for x in (kc, vc))
    np.testing.assert_array_equal(bits(got_q[:n]), bits(want_q))
    np.testing.assert_array_equal(bits(got_q[n:]), bits(q[n:]))
    want_k, want_v = b.k.copy(), b.v.copy()
    for i, (r, m) in enumerate(zip(b.rows, b.lens)):
        p, o = (x[m - r:] for x in b.places(i))
        want_k[p, o], want_v[p, o] = rk[b.starts[i]:b.starts[i + 1]], rv[b.starts[i]:b.starts[i + 1]]
    np.testing.assert_array_equal(bits(got_k), bits(want_k))
    np.testing.assert_array_equal(bits(got_v), bits(want_v))


@pytest.mark.parametrize("kv_type", [bchip.F16, bchip.F32])
@pytest.mark.parametrize("neox", [False, True])
@pytest.mark.parametrize("nh,nkv,hd,rope_dim", [(14, 2, 64, 64), (32, 8, 128, 128), (6, 3, 72, 72), (4, 2, 80, 40), (4, 4, 8, 8), (8, 2, 256, 64),
                                                (6, 2, 64, 20), (4, 1, 96, 2), (4, 2, 64, 0)])
def test_rows_go_to_their_slots_with_the_bits_of_the_call_over_one_cache(ctx, nh, nkv, hd, rope_dim, neox, kv_type):
    rng = np.random.default_rng(hd + rope_dim)
    b = Batch(rng, [1, 0, 20, 1, 5, 0], [1, 3, 37, 300, 64, 9], nkv, hd, kv_type, pad=2)
    check(ctx, b, nh, rope_dim, neox, rng)


@pytest.mark.parametrize("kv_type", [bchip.F16, bchip.F32])
@pytest.mark.parametrize("rows,lens,page_slots", [([1], [1], 16), ([1], [5000], 16), ([700, 400, 1], [700, 2000, 17], 256), ([1] * 256, list(range(1, 257)), 32)])
def test_batches(ctx, rows, lens, page_slots, kv_type):
    rng = np.random.default_rng(len(rows))
    check(ctx, Batch(rng, rows, lens, 2, 64, kv_type, page_slots=page_slots), 8, 64, True, rng)


def test_far_positions(ctx):
    rng = np.random.default_rng(5)
    check(ctx, Batch(rng, [3, 1], [40, 900], 2, 128, bchip.F16), 8, 128, False, rng, far=1 << 20)


@pytest.mark.parametrize("kv_type", [bchip.F16, bchip.F32])
def test_a_page_past_the_pool_stores_nothing(ctx, kv_type):
    rng = np.random.default_rng(6)
    b = Batch(rng, [2, 1], [18, 5], 2, 64, kv_type)
    q, k, v = (rng.standard_normal((3, h, 64)).astype(np.float32) for h in (4, 2, 2))
    positions = np.array([16, 17, 4], np.uint32)
    _, want_k, want_v = appended(ctx, b, q, k, v, positions, 4, 64, False)
    page, kept = b.table[0, 1], (b.k, b.v)
    for number in (0xFFFFFFFF, b.npages):
        b.table[0, 1] = number
        got_q, got_k, got_v = appended(ctx, b, q, k, v, positions, 4, 64, False)
        for got, want, old in ((got_k, want_k, kept[0]), (got_v, want_v, kept[1])):
            want = want.copy()
            want[page] = old[page]
            np.testing.assert_array_equal(bits(got), bits(want))
        assert not np.array_equal(got_q, q)  # q turns all the same


@pytest.mark.parametrize("kv_type", [bchip.F16, bchip.F32])
@pytest.mark.parametrize("nbufs,npages,elems,n", [(1, 2, 16 * 64, 1), (4, 9, 16 * 72, 4), (64, 40, 16 * 256, 20), (200, 5, 16 * 8, 2), (2, 700, 16 * 64, 300),
                                                  (3, 4, 32 * 1024, 2), (2, 3, 12, 1)])
def test_copied_pages(ctx, nbufs, npages, elems, n, kv_type):
    rng = np.random.default_rng(npages)
    if elems * DTYPE[kv_type]().itemsize % 16:
        pytest.skip("not whole 16-byte pieces: refused")
    pools = [rng.standard_normal((npages, elems)).astype(DTYPE[kv_type]) for _ in range(nbufs)]
    order = rng.permutation(npages).astype(np.uint32)
    dst, src = order[:n], rng.choice(order[n:], n)  # a page may be copied more than once
    bufs = [ctx.upload(x) for x in pools]
    ctx.copy_pages(bufs, kv_type, elems, npages, src, dst)
    for x, buf in zip(pools, bufs):
        want = x.copy()
        want[dst] = x[src]
        np.testing.assert_array_equal(bits(ctx.read(buf, x.shape, x.dtype)), bits(want))
        buf.free()
