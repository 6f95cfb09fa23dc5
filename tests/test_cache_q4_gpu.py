"""A KV cache in 4 bits beside attention: conversion, the append of rotated rows, moves, keep and
growth, against the format's restatement (q4_plain.py). Codes and scales are equal bit for bit:
every step that decides them is an exactly rounded f32 operation, and the rotation is the
library's own (bchip_rope), whose bits the f16 and f32 appends share."""
import numpy as np
import pytest

import bchip
import oracle as O
import q4_plain as P

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = bchip.Ctx(0)
    yield c
    c.close()


def awkward(n, seed):
    """Blocks of ordinary values, ties of both signs, zeros, tiny, huge and half-way values."""
    r = np.random.default_rng(seed)
    x = (r.standard_normal((n // 32, 32)) * np.exp(r.uniform(-12, 9, (n // 32, 1)))).astype(np.float32)
    kinds = r.integers(0, 8, n // 32)
    x[kinds == 0] = 0.0
    for i in np.flatnonzero(kinds == 1):  # two largest magnitudes of opposite sign
        m = np.abs(x[i]).max()
        x[i, 3], x[i, 20] = -m, m
    x[kinds == 2] = (r.integers(-16, 17, ((kinds == 2).sum(), 32)) / 2.0).astype(np.float32)  # ties of codes
    x[kinds == 3] *= np.float32(1e-30)
    x[kinds == 4] *= np.float32(1e4)
    return x.reshape(-1)


def raw(ctx, buf, n):
    return ctx.read(buf, bchip.nbytes_of(bchip.Q4, n), np.uint8)


def assert_same_bits(got, want):
    np.testing.assert_array_equal(got, want)


@pytest.mark.parametrize("n,off", [(32, 0), (96, 32), (256, 0), (4096, 224), (100000 // 32 * 32, 7 * 32)])
@pytest.mark.parametrize("src", ["f32", "f16"])
def test_copy_to_and_from_4_bits(ctx, n, off, src):
    x = awkward(n, n + off)
    if src == "f16":
        x = np.clip(x, -60000, 60000).astype(np.float16)
    sb = ctx.upload(x)
    db = ctx.upload(np.full(bchip.nbytes_of(bchip.Q4, off + n), 0xA5, np.uint8))
    ctx.copy(sb, bchip.F32 if src == "f32" else bchip.F16, db, bchip.Q4, off, n)
    codes, d = P.quantise(x.astype(np.float32))
    want = np.full(off + n, 0, np.uint8), np.zeros((off + n) // 32, np.float16)
    want[0][off:], want[1][off // 32:] = codes, d
    got = raw(ctx, db, off + n).reshape(-1, 144)
    w = P.pack(*want).reshape(-1, 144)
    # What the copy did not name keeps its bytes.
    mask = P.pack(np.where(np.arange(off + n) >= off, 15, 0).astype(np.uint8),
                  np.where(np.arange((off + n) // 32) >= off // 32, np.uint16(0xFFFF), np.uint16(0)).view(np.float16)).reshape(-1, 144)
    assert_same_bits(got & mask, w & mask)
    assert_same_bits(got & ~mask, np.full_like(got, 0xA5) & ~mask)
    for t, dt in ((bchip.F32, np.float32), (bchip.F16, np.float16)):
        if off % 256 == 0:
            ob = ctx.zeros((n + 8) * 4)
            ctx.copy(db, bchip.Q4, ob, t, 8, n)
            back = ctx.read(ob, n, dt, off=8 * dt().itemsize)
            np.testing.assert_array_equal(back.astype(np.float64), P.unpack(P.pack(codes, d), n))
            ob.free()
    for b in (sb, db):
        b.free()


def test_values_that_are_not_finite_make_their_block_nan(ctx):
    x = np.random.default_rng(1).standard_normal((6, 32)).astype(np.float32)
    x[1, 5], x[3, 0], x[4, 31] = np.nan, np.inf, -np.inf
    sb, db, ob = ctx.upload(x), ctx.zeros(144), ctx.zeros(6 * 32 * 4)
    ctx.copy(sb, bchip.F32, db, bchip.Q4, 0, x.size)
    ctx.copy(db, bchip.Q4, ob, bchip.F32, 0, x.size)
    got = ctx.read(ob, x.shape)
    assert np.isnan(got[[1, 3, 4]]).all() and np.isfinite(got[[0, 2, 5]]).all()
    np.testing.assert_array_equal(got[[0, 2, 5]], P.stored(x[[0, 2, 5]]))
    # 4 bits to 4 bits: the blocks as they are.
    eb = ctx.zeros(144 * 2)
    ctx.copy(db, bchip.Q4, eb, bchip.Q4, 224, x.size)
    ctx.copy(eb, bchip.Q4, ob, bchip.F32, 0, 32)
    cb = ctx.zeros(144 * 2)
    ctx.copy(eb, bchip.Q4, cb, bchip.Q4, 0, 224 + x.size)
    ctx.move(cb, bchip.Q4, 224, 0, x.size)
    ctx.copy(cb, bchip.Q4, ob, bchip.F32, 0, x.size)
    np.testing.assert_array_equal(ctx.read(ob, x.shape), got)
    for b in (sb, db, ob, eb, cb):
        b.free()


SHAPES = [(4, 2, 32, 32, False), (14, 2, 64, 64, True), (12, 4, 96, 96, True), (32, 8, 128, 128, False), (28, 4, 128, 64, True),
          (8, 1, 160, 40, False), (6, 3, 224, 100, True), (16, 4, 256, 256, True)]


@pytest.mark.parametrize("nh,nkv,hd,rd,neox", SHAPES)
@pytest.mark.parametrize("rows,slot0", [(1, 0), (1, 7), (5, 3), (67, 130)])
def test_append_is_the_rotated_row_in_4_bits(ctx, nh, nkv, hd, rd, neox, rows, slot0):
    r = np.random.default_rng(hd * rows + slot0)
    kvd = nkv * hd
    q, k, v = (r.standard_normal((rows, n * hd)).astype(np.float32) for n in (nh, nkv, nkv))
    pos = (slot0 * 37 + np.arange(rows)).astype(np.uint32)
    n = (slot0 + rows) * kvd
    was = np.random.default_rng(3).integers(0, 256, bchip.nbytes_of(bchip.Q4, n)).astype(np.uint8)
    qb, kb, vb, q2, k2 = (ctx.upload(x) for x in (q, k, v, q, k))
    kc, vc, ib, pb = ctx.upload(was), ctx.upload(was), ctx.upload(O.inv_freq(rd, 1e4)), ctx.upload(pos)
    ctx.rope_append(qb, kb, vb, kc, vc, bchip.Q4, ib, pb, rows, nh, nkv, hd, rd, neox, slot0)
    ctx.rope(q2, ib, pb, rows, nh, hd, rd, neox)
    ctx.rope(k2, ib, pb, rows, nkv, hd, rd, neox)
    np.testing.assert_array_equal(ctx.read(qb, q.shape), ctx.read(q2, q.shape))
    np.testing.assert_array_equal(ctx.read(kb, k.shape), k)
    for buf, x in ((kc, ctx.read(k2, k.shape)), (vc, v)):
        codes, d = np.zeros(n, np.uint8), np.zeros(n // 32, np.float16)
        c, s = P.quantise(x)
        codes[slot0 * kvd:], d[slot0 * kvd // 32:] = c.reshape(-1), s.reshape(-1)
        mask = P.pack(np.where(np.arange(n) >= slot0 * kvd, 15, 0).astype(np.uint8),
                      np.where(np.arange(n // 32) >= slot0 * kvd // 32, np.uint16(0xFFFF), np.uint16(0)).view(np.float16))
        got, want = raw(ctx, buf, n), P.pack(codes, d)
        assert_same_bits(got & mask, want & mask)
        assert_same_bits(got & ~mask, was & ~mask)  # earlier slots, and the unit's end
    for b in (qb, kb, vb, q2, k2, kc, vc, ib, pb):
        b.free()


@pytest.mark.parametrize("nh,nkv,hd,rd,neox,rows", [(32, 8, 128, 128, False, 517), (14, 2, 64, 64, True, 2333), (13, 1, 128, 64, True, 1401),
                                                    (9, 3, 96, 40, False, 1900), (6, 6, 32, 32, True, 4600)])
def test_an_append_of_many_rows(ctx, nh, nkv, hd, rd, neox, rows):
    """Rows from which a thread takes several heads: the bits of appends of a few rows each."""
    r = np.random.default_rng(rows)
    kvd, n = nkv * hd, rows * nkv * hd
    q, k, v = (r.standard_normal((rows, x * hd)).astype(np.float32) for x in (nh, nkv, nkv))
    pos = (np.arange(rows) * 31 + 5).astype(np.uint32)
    ib, pb, kb, vb = ctx.upload(O.inv_freq(rd, 1e4)), ctx.upload(pos), ctx.upload(k), ctx.upload(v)
    got = []
    for step in (rows, 100):
        qb, kc, vc = ctx.upload(q), ctx.zeros(bchip.nbytes_of(bchip.Q4, n)), ctx.zeros(bchip.nbytes_of(bchip.Q4, n))
        for i in range(0, rows, step):
            ctx.rope_append(qb.offset(i * nh * hd * 4), kb.offset(i * kvd * 4), vb.offset(i * kvd * 4), kc, vc, bchip.Q4, ib,
                            pb.offset(i * 4), min(step, rows - i), nh, nkv, hd, rd, neox, i)
        got.append([ctx.read(qb, q.shape), raw(ctx, kc, n), raw(ctx, vc, n)])
        for b in (qb, kc, vc):
            b.free()
    for x, y in zip(*got):
        np.testing.assert_array_equal(x, y)
    for b in (ib, pb, kb, vb):
        b.free()


def test_ragged_append_is_each_rows_own(ctx):
    nh, nkv, hd, n = 8, 2, 64, 70
    kvd = nkv * hd
    r = np.random.default_rng(5)
    q, k, v = (r.standard_normal((n, h * hd)).astype(np.float32) for h in (nh, nkv, nkv))
    lens = r.integers(1, 9, n).astype(np.uint32)
    offs = np.concatenate([[0], np.cumsum(lens)])[:-1].astype(np.uint64)
    total = int(lens.sum()) * kvd
    pos = r.integers(0, 4000, n).astype(np.uint32)
    qb, kb, vb = ctx.upload(q), ctx.upload(k), ctx.upload(v)
    q1 = ctx.upload(q)
    ib, pb = ctx.upload(O.inv_freq(hd, 1e4)), ctx.upload(pos)
    bufs = [ctx.zeros(bchip.nbytes_of(bchip.Q4, total)) for _ in range(4)]
    ctx.rope_append_ragged(qb, kb, vb, bufs[0], bufs[1], bchip.Q4, ib, pb, lens, offs, nh, nkv, hd, hd, True)
    for i in range(n):
        ctx.rope_append(q1.offset(i * nh * hd * 4), kb.offset(i * kvd * 4), vb.offset(i * kvd * 4), bufs[2], bufs[3], bchip.Q4,
                        ib, pb.offset(4 * i), 1, nh, nkv, hd, hd, True, int(offs[i] + lens[i] - 1))
    assert_same_bits(ctx.read(qb, q.shape), ctx.read(q1, q.shape))
    for a, b in ((0, 2), (1, 3)):
        assert_same_bits(raw(ctx, bufs[a], total), raw(ctx, bufs[b], total))
    for b in [qb, kb, vb, q1, ib, pb] + bufs:
        b.free()


@pytest.mark.parametrize("kvd,base,rows", [(32, 0, [1]), (32, 5, [0, 2, 3, 9]), (128, 3, [1, 2, 3]), (96, 11, [0, 1, 5, 40]), (1024, 2, [7])])
def test_keep_moves_rows_of_blocks(ctx, kvd, base, rows):
    slots = base + max(rows) + 2
    x = np.random.default_rng(kvd).standard_normal((3, slots, kvd)).astype(np.float32)
    bufs = [ctx.upload(P.pack(*P.quantise(a))) for a in x]
    ctx.keep(bufs, bchip.Q4, kvd, base, rows)
    for a, b in zip(x, bufs):
        want = P.stored(a)
        for i, r in enumerate(rows):
            want[base + i] = want[base + r]
        np.testing.assert_array_equal(P.unpack(raw(ctx, b, slots * kvd), slots * kvd).reshape(slots, kvd), want)
        b.free()


@pytest.mark.parametrize("frm,to,n", [(64, 32, 320), (512, 0, 512), (96, 64, 32), (4096, 32, 5000 // 32 * 32)])
def test_move_of_overlapping_blocks(ctx, frm, to, n):
    x = np.random.default_rng(n).standard_normal(frm + n).astype(np.float32)
    b = ctx.upload(P.pack(*P.quantise(x)))
    ctx.move(b, bchip.Q4, frm, to, n)
    want = P.stored(x)
    want[to:to + n] = P.stored(x)[frm:frm + n]
    np.testing.assert_array_equal(P.unpack(raw(ctx, b, x.size), x.size), want)
    b.free()


@pytest.mark.parametrize("keep,total", [(0, 320), (32, 32), (96, 288), (256, 1024), (1024 * 5, 1024 * 300), (128 * 7, 128 * 301)])
def test_growth_keeps_the_prefix_and_zeroes_the_rest(ctx, keep, total):
    x = np.random.default_rng(keep).standard_normal(max(keep, 32)).astype(np.float32)
    sb = [ctx.upload(P.pack(*P.quantise(x))) for _ in range(2)]
    db = [ctx.upload(np.full(bchip.nbytes_of(bchip.Q4, total), 0x77, np.uint8)) for _ in range(2)]
    ctx.cache_grow(sb, db, bchip.Q4, keep, total)
    want = np.zeros(total)
    want[:keep] = P.stored(x)[:keep]
    for b in db:
        np.testing.assert_array_equal(P.unpack(raw(ctx, b, total), total), want)
    for b in sb + db:
        b.free()


def test_a_kv_cache_of_4_bits_grows_and_keeps(ctx):
    kvd, layers = 128, 3
    cache = bchip.KvCache(ctx, layers, kvd, bchip.Q4)
    cache.reserve(10, 0, 4096)
    assert cache.cap == 256 and cache.bytes() == 2 * layers * 256 * kvd // 256 * 144
    x = np.random.default_rng(2).standard_normal((2 * layers, 256, kvd)).astype(np.float32)
    for a, b in zip(x, cache.k + cache.v):
        t = ctx.upload(a)
        ctx.copy(t, bchip.F32, b, bchip.Q4, 0, a.size)
        t.free()
    cache.reserve(300, 255, 4096)
    cache.keep(200, [3, 5, 6])
    for a, b in zip(x, cache.k + cache.v):
        want = np.zeros((cache.cap, kvd))
        want[:255] = P.stored(a)[:255]
        for i, r in enumerate([3, 5, 6]):
            want[200 + i] = want[200 + r]
        np.testing.assert_array_equal(P.unpack(raw(ctx, b, want.size), want.size).reshape(want.shape), want)
    cache.free()


def test_bad_arguments_are_refused(ctx):
    a, b = ctx.zeros(144 * 8), ctx.zeros(144 * 8)
    f = ctx.zeros(4 * 2048)
    pb, ib = ctx.zeros(64), ctx.zeros(1024)

    def refused(code, fn):
        with pytest.raises(bchip.BchipError) as e:
            fn()
        assert e.value.code == code, bchip.last_error()

    arg = lambda fn: refused(bchip.E_ARG, fn)
    arg(lambda: ctx.copy(f, bchip.F32, a, bchip.Q4, 0, 33))
    arg(lambda: ctx.copy(f, bchip.F32, a, bchip.Q4, 16, 32))
    arg(lambda: ctx.copy(a, bchip.Q4, f, bchip.F32, 0, 40))
    arg(lambda: ctx.copy(f, bchip.F32, a, bchip.Q4, 8 * 256, 32))          # past the buffer
    arg(lambda: ctx.copy(f, bchip.F32, a, bchip.Q4, (1 << 64) - 32, 32))
    arg(lambda: ctx.copy(a.ptr + 8, bchip.Q4, f, bchip.F32, 0, 32))        # not aligned
    arg(lambda: ctx.copy(f, bchip.F32, a, 3, 0, 32))
    arg(lambda: ctx.move(a, bchip.Q4, 48, 0, 32))
    arg(lambda: ctx.move(a, bchip.Q4, 64, 0, 8 * 256))
    arg(lambda: ctx.keep([a], bchip.Q4, 48, 0, [1]))
    arg(lambda: ctx.keep([a], bchip.Q4, 256, 0, [8]))
    arg(lambda: ctx.cache_grow([a], [b], bchip.Q4, 48, 64))
    arg(lambda: ctx.cache_grow([a], [b], bchip.Q4, 32, 9 * 256))
    arg(lambda: ctx.cache_grow([a], [a], bchip.Q4, 32, 64))
    arg(lambda: ctx.fill_normal(a, bchip.Q4, 32, 1))
    arg(lambda: ctx.rope_append(f, f, f, a, b, bchip.Q4, ib, pb, 1, 4, 2, 64, 64, True, 16))  # past the cache
    arg(lambda: ctx.rope_append(f, f, f, a.ptr + 4, b, bchip.Q4, ib, pb, 1, 4, 2, 64, 64, True, 0))
    refused(bchip.E_UNSUPPORTED, lambda: ctx.rope_append(f, f, f, a, b, bchip.Q4, ib, pb, 1, 4, 2, 80, 80, True, 0))
    refused(bchip.E_UNSUPPORTED, lambda: ctx.rope_append_ragged(f, f, f, a, b, bchip.Q4, ib, pb, [1], [0], 4, 2, 16, 16, True))
    for x in (a, b):
        assert not ctx.read(x, 144 * 8, np.uint8).any()
        x.free()
    for x in (f, pb, ib):
        x.free()
