"""Attention over caches in 4 bits, against its formula in 64 bits over the values the codes stand
for (q4_plain.py): decode steps, short and long line passes, trees, ragged pools. Two bounds a
case: every output within what its roundings can add up to (q4_plain.bound), and the whole within
8e-6 of the result's norm: the roundings of a score's 2 hd / 32 MFMAs and of its weight, 2^-24
each and independent, leave about 1e-6, while q or a weight without its low part would leave
2^-12 / 3 of a typical product, 8e-5."""
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


def cache(n, kvd, seed, scale=1.0):
    """A buffer of n slots and its values [n, kvd]."""
    x = (np.random.default_rng(seed).standard_normal((n, kvd)) * scale).astype(np.float32)
    buf = P.pack(*P.quantise(x))
    return buf, P.unpack(buf, n * kvd).reshape(n, kvd)


def gate(got, want, mass, top, hd, what, norm=True):
    got = got.astype(np.float64)
    err = np.abs(got - want)
    lim = P.bound(mass, top, hd)
    size = np.linalg.norm(want)
    rel = np.linalg.norm(got - want) / size if size else 0.0
    print(f"{what}: rel {rel:.2e}, worst {np.max(err / lim):.3f} of the bound", flush=True)
    assert (err <= lim).all(), f"{what}: {np.max(err / lim)} of the bound"
    assert not norm or rel <= 8e-6, f"{what}: rel {rel}"


def run(ctx, q, kbuf, vbuf, nkv, pos, scale, masks=None, fill=np.nan):
    rows, nh, hd = q.shape
    qb, kb, vb = ctx.upload(q), ctx.upload(kbuf), ctx.upload(vbuf)
    ob = ctx.upload(np.full((rows + 1, nh, hd), fill, np.float32))
    mb = ctx.upload(bchip.masks_words(masks)) if masks is not None else None
    ctx.attention(qb, kb, vb, bchip.Q4, ob, mb, masks is not None, rows, nh, nkv, hd, pos, scale)
    got = ctx.read(ob, (rows + 1, nh, hd))
    for b in (qb, kb, vb, ob) + ((mb,) if mb else ()):
        b.free()
    assert np.isnan(got[rows]).all()  # the row behind the last stays as it was
    return got[:rows]


def line(rows, pos):
    return np.arange(pos + rows)[None] <= (pos + np.arange(rows))[:, None]


# Every number of 32-dim blocks a head can have, groups of 1 to 16 heads.
SHAPES = [(2, 2, 32), (14, 2, 64), (12, 4, 96), (32, 8, 128), (7, 1, 160), (16, 1, 192), (6, 2, 224), (16, 4, 256), (8, 1, 32), (9, 3, 64)]


@pytest.mark.parametrize("nh,nkv,hd", SHAPES)
@pytest.mark.parametrize("rows,pos", [(1, 0), (1, 31), (1, 32), (1, 300), (1, 5000), (2, 0), (3, 126), (5, 700), (17, 0), (33, 62), (70, 500)])
def test_lines(ctx, nh, nkv, hd, rows, pos):
    r = np.random.default_rng(rows * 7 + pos + hd)
    q = (r.standard_normal((rows, nh, hd)) * 2).astype(np.float32)
    n, kvd, scale = pos + rows, nkv * hd, hd ** -0.5
    kbuf, k = cache(n, kvd, 1)
    vbuf, v = cache(n, kvd, 2)
    got = run(ctx, q, kbuf, vbuf, nkv, pos, scale)
    want, mass, top = P.attention(q, k.reshape(n, nkv, hd), v.reshape(n, nkv, hd), nkv, line(rows, pos), scale)
    gate(got, want, mass, top, hd, f"{nh}/{nkv} x {hd}, {rows} at {pos}")
    np.testing.assert_array_equal(got, run(ctx, q, kbuf, vbuf, nkv, pos, scale))  # the same bits again


# Passes whose workgroups take 32 query rows a wave, and long lists.
@pytest.mark.parametrize("nh,nkv,hd,rows,pos", [(32, 8, 128, 1100, 0), (32, 8, 128, 1037, 333), (14, 2, 64, 2345, 77), (12, 4, 96, 2801, 0),
                                                (2, 2, 32, 9000, 5), (16, 4, 256, 700, 301), (64, 8, 128, 8, 20000), (32, 8, 128, 1, 60001),
                                                (28, 4, 128, 1, 131071), (8, 8, 256, 2, 9999)])
def test_long_passes(ctx, nh, nkv, hd, rows, pos):
    r = np.random.default_rng(rows)
    q = (r.standard_normal((rows, nh, hd)) * 2).astype(np.float32)
    n, kvd = pos + rows, nkv * hd
    kbuf, k = cache(n, kvd, 3)
    vbuf, v = cache(n, kvd, 4)
    got = run(ctx, q, kbuf, vbuf, nkv, pos, hd ** -0.5)
    some = np.unique(np.concatenate([[0, rows - 1, min(rows - 1, 63), rows // 2], r.integers(0, rows, 20)]))
    see = np.arange(n)[None] <= (pos + some)[:, None]
    want, mass, top = P.attention(q[some], k.reshape(n, nkv, hd), v.reshape(n, nkv, hd), nkv, see, hd ** -0.5)
    gate(got[some], want, mass, top, hd, f"{nh}/{nkv} x {hd}, {rows} at {pos}")
    assert np.isfinite(got).all()


@pytest.mark.parametrize("nh,nkv,hd", [(14, 2, 64), (64, 8, 128), (12, 4, 96), (16, 4, 256), (2, 2, 32)])
@pytest.mark.parametrize("rows,pos", [(1, 0), (2, 0), (5, 33), (64, 0), (33, 700), (16, 3000)])
def test_trees(ctx, nh, nkv, hd, rows, pos):
    r = np.random.default_rng(rows + pos)
    q = (r.standard_normal((rows, nh, hd)) * 2).astype(np.float32)
    masks = r.integers(0, 1 << 63, rows, dtype=np.uint64) * np.uint64(2) + r.integers(0, 2, rows, dtype=np.uint64)
    masks[0] = 0                     # sees the slots below pos alone (nothing at pos 0)
    masks[-1] = np.uint64(1) << np.uint64(63) if rows > 1 else np.uint64(0)
    n, kvd, scale = pos + 64, nkv * hd, hd ** -0.5
    kbuf, k = cache(n, kvd, 5)
    vbuf, v = cache(n, kvd, 6)
    bits = (masks[:, None] >> np.arange(64, dtype=np.uint64)[None]) & np.uint64(1)
    see = np.concatenate([np.ones((rows, pos), bool), bits.astype(bool)], 1)
    want, mass, top = P.attention(q, k.reshape(n, nkv, hd), v.reshape(n, nkv, hd), nkv, see, scale)
    gate(run(ctx, q, kbuf, vbuf, nkv, pos, scale, masks), want, mass, top, hd, f"tree {nh}/{nkv} x {hd}, {rows} at {pos}")
    # Rows of no deeper node than the pass's own: no slot past the highest named one is read.
    low = masks & ((np.uint64(1) << np.uint64(min(rows, 63))) - np.uint64(1))
    held = pos + rows
    see = np.concatenate([np.ones((rows, pos), bool), ((low[:, None] >> np.arange(rows, dtype=np.uint64)[None]) & np.uint64(1)).astype(bool)], 1)
    want, mass, top = P.attention(q, k.reshape(n, nkv, hd)[:held], v.reshape(n, nkv, hd)[:held], nkv, see, scale)
    cut = bchip.nbytes_of(bchip.Q4, held * kvd)
    gate(run(ctx, q, kbuf[:cut], vbuf[:cut], nkv, pos, scale, low), want, mass, top, hd, "the same, masks of its own rows")


def ragged_row(q, k, v, nkv, hd, scale, i, off, length, got):
    kk, vv = (t[int(off):int(off + length)].reshape(-1, nkv, hd) for t in (k, v))
    want, mass, top = P.attention(q[i:i + 1], kk, vv, nkv, np.ones((1, int(length)), bool), scale)
    assert (np.abs(got[i:i + 1] - want) <= P.bound(mass, top, hd)).all(), f"sequence {i} of {length}"
    return want


@pytest.mark.parametrize("nh,nkv,hd", [(28, 4, 128), (14, 2, 64), (2, 1, 32), (12, 4, 96), (16, 1, 128)])
@pytest.mark.parametrize("seqs,longest", [(1, 1), (3, 40), (16, 900), (70, 300)])
def test_ragged(ctx, nh, nkv, hd, seqs, longest):
    r = np.random.default_rng(seqs)
    lens = r.integers(1, longest + 1, seqs).astype(np.uint32)
    gaps = r.integers(0, 3, seqs)
    offs = (np.concatenate([[0], np.cumsum(lens + gaps)])[:-1] + 1).astype(np.uint64)
    n, kvd, scale = int(offs[-1] + lens[-1]), nkv * hd, hd ** -0.5
    q = (r.standard_normal((seqs, nh, hd)) * 2).astype(np.float32)
    kbuf, k = cache(n, kvd, 7)
    vbuf, v = cache(n, kvd, 8)
    qb, kb, vb, ob = ctx.upload(q), ctx.upload(kbuf), ctx.upload(vbuf), ctx.zeros(q.nbytes)
    ctx.attention_ragged(qb, kb, vb, bchip.Q4, ob, lens, offs, nh, nkv, hd, scale)
    got = ctx.read(ob, q.shape)
    whole = np.linalg.norm(got - np.concatenate([ragged_row(q, k, v, nkv, hd, scale, i, o, l, got) for i, (o, l) in enumerate(zip(offs, lens))]))
    assert whole <= 8e-6 * np.linalg.norm(got)
    for b in (qb, kb, vb, ob):
        b.free()


@pytest.mark.parametrize("lens", [[20000] + [100] * 63, [33, 6000] + [100] * 15, [1300] * 3 + [640] * 9, [2561] * 65])
def test_ragged_lists_of_unlike_lengths(ctx, lens):
    """One long list among brief ones is cut, whatever their average; more lists than a launch takes."""
    nh, nkv, hd = 14, 2, 64
    lens = np.array(lens, np.uint32)
    offs = np.concatenate([[0], np.cumsum(lens)[:-1]]).astype(np.uint64)
    n, kvd, scale, r = int(lens.sum()), nkv * hd, hd ** -0.5, np.random.default_rng(len(lens))
    q = (r.standard_normal((len(lens), nh, hd)) * 2).astype(np.float32)
    kbuf, k = cache(n, kvd, 17)
    vbuf, v = cache(n, kvd, 18)
    qb, kb, vb, ob = ctx.upload(q), ctx.upload(kbuf), ctx.upload(vbuf), ctx.zeros(q.nbytes)
    ctx.attention_ragged(qb, kb, vb, bchip.Q4, ob, lens, offs, nh, nkv, hd, scale)
    got = ctx.read(ob, q.shape)
    whole = np.linalg.norm(got - np.concatenate([ragged_row(q, k, v, nkv, hd, scale, i, o, l, got) for i, (o, l) in enumerate(zip(offs, lens))]))
    assert whole <= 8e-6 * np.linalg.norm(got)
    for b in (qb, kb, vb, ob):
        b.free()


def test_more_rows_than_a_grid_holds(ctx):
    """65535 units of 64 query rows a KV head are a grid's most: a longer pass runs in parts."""
    nh, nkv, hd, rows = 16, 1, 32, 65535 * 4 + 70
    r = np.random.default_rng(2)
    q = np.resize((r.standard_normal((1000, nh, hd)) * 2).astype(np.float32), (rows, nh, hd))
    kbuf, k = cache(rows, hd, 19)
    vbuf, v = cache(rows, hd, 20)
    got = run(ctx, q, kbuf, vbuf, nkv, 0, hd ** -0.5)
    some = np.array([0, 65535 * 4 - 1, 65535 * 4, rows - 1])
    see = np.arange(rows)[None] <= some[:, None]
    want, mass, top = P.attention(q[some], k.reshape(rows, nkv, hd), v.reshape(rows, nkv, hd), nkv, see, hd ** -0.5)
    gate(got[some], want, mass, top, hd, "rows in parts")
    assert np.isfinite(got).all()


# Enough rows that a wave takes 32 of them.
@pytest.mark.parametrize("nh,nkv,hd,rows,pos", [(32, 8, 128, 1500, 0), (28, 4, 128, 1701, 333), (14, 2, 64, 7100, 77), (12, 4, 96, 3800, 0),
                                                (16, 8, 32, 6200, 5)])
def test_passes_of_32_rows_a_wave(ctx, nh, nkv, hd, rows, pos):
    """Against the formula in some rows; a V block that is not finite reaches the rows that see its
    slot, and no other."""
    r = np.random.default_rng(rows)
    q = (r.standard_normal((rows, nh, hd)) * 2).astype(np.float32)
    n, kvd, odd = pos + rows, nkv * hd, pos + rows - 41
    kbuf, k = cache(n, kvd, 21)
    x = np.random.default_rng(22).standard_normal((n, nkv, hd)).astype(np.float32)
    x[odd, nkv - 1, hd - 1] = np.inf  # the last block of the last head
    vbuf = P.pack(*P.quantise(x.reshape(n, kvd)))
    v = P.unpack(vbuf, n * kvd).reshape(n, nkv, hd)
    got = run(ctx, q, kbuf, vbuf, nkv, pos, hd ** -0.5)
    some = np.unique(np.concatenate([[0, rows - 1, 31, 32, rows - 41, rows - 42], r.integers(0, rows, 16)]))
    see = np.arange(n)[None] <= (pos + some)[:, None]
    want, mass, top = P.attention(q[some], k.reshape(n, nkv, hd), v, nkv, see, hd ** -0.5)
    bad = np.zeros(got.shape, bool)
    bad[rows - 41:, nh - nh // nkv:, hd - 32:] = True
    np.testing.assert_array_equal(np.isnan(got), bad)
    fine = ~bad[some]
    assert (np.abs(got[some] - want)[fine] <= P.bound(mass, top, hd)[fine]).all()
    assert np.linalg.norm((got[some] - want)[fine]) <= 8e-6 * np.linalg.norm(want[fine])


@pytest.mark.parametrize("nh,nkv,hd,rows,pos", [(32, 8, 128, 200, 4000), (32, 8, 128, 340, 9001), (14, 2, 64, 777, 3999), (12, 4, 96, 600, 7000),
                                                (16, 4, 256, 400, 3500)])
def test_pieces_of_a_prompt_behind_a_long_history(ctx, nh, nkv, hd, rows, pos):
    """Passes of many workgroups whose lists are cut all the same."""
    r = np.random.default_rng(rows)
    q = (r.standard_normal((rows, nh, hd)) * 2).astype(np.float32)
    n, kvd = pos + rows, nkv * hd
    kbuf, k = cache(n, kvd, 25)
    vbuf, v = cache(n, kvd, 26)
    got = run(ctx, q, kbuf, vbuf, nkv, pos, hd ** -0.5)
    some = np.unique(np.concatenate([[0, rows - 1, rows // 2], r.integers(0, rows, 12)]))
    see = np.arange(n)[None] <= (pos + some)[:, None]
    want, mass, top = P.attention(q[some], k.reshape(n, nkv, hd), v.reshape(n, nkv, hd), nkv, see, hd ** -0.5)
    gate(got[some], want, mass, top, hd, f"{nh}/{nkv} x {hd}, {rows} at {pos}")
    assert np.isfinite(got).all()


def test_a_tree_of_many_heads(ctx):
    """A tree whose KV heads alone make enough workgroups for 32 rows a wave."""
    nh, nkv, hd, rows, pos = 768, 48, 96, 64, 70
    r = np.random.default_rng(5)
    q = (r.standard_normal((rows, nh, hd)) * 2).astype(np.float32)
    masks = r.integers(0, 1 << 63, rows, dtype=np.uint64) * np.uint64(2)
    n, kvd = pos + 64, nkv * hd
    kbuf, k = cache(n, kvd, 23)
    vbuf, v = cache(n, kvd, 24)
    got = run(ctx, q, kbuf, vbuf, nkv, pos, hd ** -0.5, masks)
    some = np.array([0, 1, 17, 31, 32, 63])
    bits = (masks[some][:, None] >> np.arange(64, dtype=np.uint64)[None]) & np.uint64(1)
    see = np.concatenate([np.ones((len(some), pos), bool), bits.astype(bool)], 1)
    want, mass, top = P.attention(q[some], k.reshape(n, nkv, hd), v.reshape(n, nkv, hd), nkv, see, hd ** -0.5)
    gate(got[some], want, mass, top, hd, "a tree of 768 heads")
    assert np.isfinite(got).all()


def test_a_pool_past_4_gib(ctx):
    """Slots whose bytes lie past 2^32."""
    nh, nkv, hd, length = 8, 8, 128, 700
    kvd, off = nkv * hd, 8_000_003
    r = np.random.default_rng(9)
    q = (r.standard_normal((2, nh, hd)) * 2).astype(np.float32)
    size = bchip.nbytes_of(bchip.Q4, (off + length) * kvd)
    assert off * kvd * 9 // 16 > 1 << 32
    kb, vb = ctx.zeros(size), ctx.zeros(size)
    kbuf, k = cache(length, kvd, 10)
    vbuf, v = cache(length, kvd, 11)
    at = off * kvd // 256 * 144
    ctx.upload(kbuf, kb, at)
    ctx.upload(vbuf, vb, at)
    qb, ob = ctx.upload(q), ctx.zeros(q.nbytes)
    ctx.attention_ragged(qb, kb, vb, bchip.Q4, ob, [length - 1, length], [off, off], nh, nkv, hd, hd ** -0.5)
    got = ctx.read(ob, q.shape)
    see = np.arange(length)[None] < np.array([[length - 1], [length]])
    want, mass, top = P.attention(q, k.reshape(-1, nkv, hd), v.reshape(-1, nkv, hd), nkv, see, hd ** -0.5)
    gate(got, want, mass, top, hd, "past 4 GiB")
    for b in (qb, kb, vb, ob):
        b.free()


@pytest.mark.parametrize("rows,G", [(1, 4), (5, 4), (3, 2), (40, 8)])
def test_what_a_row_does_not_see_does_not_reach_it(ctx, rows, G):
    """Blocks that are not finite in slots past a row's list, in holes of a tree, and in the slots
    of some rows: a row's outputs are NaN where it sees one, and the plain result elsewhere."""
    nkv, hd, pos = 2, 128, 45
    nh, n, kvd, scale = nkv * G, pos + 64, nkv * 128, 128 ** -0.5
    r = np.random.default_rng(rows)
    q = r.standard_normal((rows, nh, hd)).astype(np.float32)
    kx, vx = (r.standard_normal((n, nkv, hd)).astype(np.float32) for _ in range(2))
    vx[pos, 0, 40] = np.inf             # row 0's last slot: V block 1 of head 0
    vx[pos + rows - 1, 1, 127] = np.nan  # the last row's: V block 3 of head 1
    kx[pos + rows // 2, 1, 0] = np.nan  # K: every output of head 1's rows that see it
    kx[pos + rows:], vx[pos + rows:] = np.nan, np.inf
    kbuf, vbuf = P.pack(*P.quantise(kx.reshape(n, kvd))), P.pack(*P.quantise(vx.reshape(n, kvd)))
    k, v = (P.unpack(b, n * kvd).reshape(n, nkv, hd) for b in (kbuf, vbuf))

    def check(got, see, what):
        want, mass, top = P.attention(q, k, v, nkv, see, scale)
        np.testing.assert_array_equal(np.isnan(got), np.isnan(want), err_msg=what)
        fine = ~np.isnan(want)
        assert (np.abs(got - want)[fine] <= P.bound(mass, np.nan_to_num(top), hd)[fine]).all(), what
        assert fine.any() and not fine.all(), what

    check(run(ctx, q, kbuf, vbuf, nkv, pos, scale), np.pad(line(rows, pos), ((0, 0), (0, n - pos - rows))), "line")
    masks = (np.uint64(1) << np.arange(rows, dtype=np.uint64))  # row i sees slot pos + i alone of the tree's
    see = np.arange(n)[None] < pos
    see = see | (np.arange(n)[None] == pos + np.arange(rows)[:, None])
    check(run(ctx, q, kbuf, vbuf, nkv, pos, scale, masks), see, "tree")


def test_odd_values(ctx):
    """q rows that are zero, tiny, huge, infinite or NaN beside ordinary ones, and caches of tiny
    and of large values."""
    nh, nkv, hd, n = 8, 2, 64, 100
    r = np.random.default_rng(4)
    q = r.standard_normal((7, nh, hd)).astype(np.float32)
    q[1], q[2], q[3] = 0, q[2] * 1e-30, q[3] * 1e5
    q[4, 0, 3], q[5, 1, 60] = np.inf, np.nan
    for ks, vs in ((1.0, 1.0), (1e-3, 1e-4), (300.0, 2000.0)):
        kbuf, k = cache(n, nkv * hd, 12, ks)
        vbuf, v = cache(n, nkv * hd, 13, vs)
        got = run(ctx, q, kbuf, vbuf, nkv, n - 7, hd ** -0.5)
        bad = np.zeros((7, nh), bool)
        bad[4, 0] = bad[5, 1] = True
        assert np.isnan(got[bad]).all() and np.isfinite(got[~bad]).all()
        qq = np.where(bad[..., None], np.float32(0), q)
        want, mass, top = P.attention(qq, k.reshape(n, nkv, hd), v.reshape(n, nkv, hd), nkv, line(7, n - 7), hd ** -0.5)
        err, lim = np.abs(got - want), P.bound(mass, top, hd)
        worst = (err / lim).max(-1)
        print(ks, vs, np.where(bad, 0, worst).max(1))
        assert (err <= lim)[~bad].all()


@pytest.mark.parametrize("rows,nh,nkv,hd,rd,neox,pos", [(1, 32, 8, 128, 128, False, 777), (1, 14, 2, 64, 64, True, 0), (4, 14, 2, 64, 32, True, 130),
                                                        (9, 16, 4, 256, 256, False, 300)])
def test_a_step_is_its_two_calls(ctx, rows, nh, nkv, hd, rd, neox, pos):
    kvd, scale = nkv * hd, hd ** -0.5
    r = np.random.default_rng(pos)
    q, k, v = (r.standard_normal((rows, n * hd)).astype(np.float32) for n in (nh, nkv, nkv))
    was, _ = cache(pos + rows, kvd, 14)
    ib, pb = ctx.upload(O.inv_freq(rd, 1e4)), ctx.upload((pos + np.arange(rows)).astype(np.uint32))
    kb, vb = ctx.upload(k), ctx.upload(v)
    res = []
    calls = ["two", "rows"] + (["one", "noalloc"] if rows == 1 else [])
    for how in calls:
        qb, kc, vc, ob = ctx.upload(q), ctx.upload(was), ctx.upload(was), ctx.zeros(q.nbytes)
        a = (qb, kb, vb, kc, vc, bchip.Q4, ib, pb)
        if how == "two":
            ctx.rope_append(*a, rows, nh, nkv, hd, rd, neox, pos)
            ctx.attention(qb, kc, vc, bchip.Q4, ob, None, False, rows, nh, nkv, hd, pos, scale)
        elif how == "rows":
            ctx.rope_append_attention_rows(*a, rows, nh, nkv, hd, rd, neox, pos, scale, ob)
        else:
            (ctx.rope_append_attention if how == "one" else ctx.rope_append_attention_noalloc)(*a, nh, nkv, hd, rd, neox, pos, scale, ob)
        res.append([ctx.read(ob, q.shape), ctx.read(qb, q.shape)] + [ctx.read(c, was.size, np.uint8) for c in (kc, vc)])
        for b in (qb, kc, vc, ob):
            b.free()
    for how, x in zip(calls[1:], res[1:]):
        for name, a, b in zip(("out", "q", "K", "V"), x, res[0]):
            np.testing.assert_array_equal(a, b, err_msg=f"{how}: {name}")
    for b in (ib, pb, kb, vb):
        b.free()


def test_bad_arguments_are_refused(ctx):
    kc, q, out = ctx.zeros(144 * 40), ctx.zeros(4 * 4096), ctx.zeros(4 * 4096)  # 10 slots of 8 x 128

    def refused(code, fn):
        with pytest.raises(bchip.BchipError) as e:
            fn()
        assert e.value.code == code, bchip.last_error()

    refused(bchip.E_ARG, lambda: ctx.attention(q, kc, kc, bchip.Q4, out, None, False, 1, 32, 8, 128, 10, 0.1))
    refused(bchip.E_ARG, lambda: ctx.attention(q, kc.ptr + 8, kc, bchip.Q4, out, None, False, 1, 32, 8, 128, 1, 0.1))
    refused(bchip.E_ARG, lambda: ctx.attention(q, kc, kc, bchip.Q4, out, None, True, 1, 32, 8, 128, 1, 0.1))
    refused(bchip.E_ARG, lambda: ctx.attention(q, kc, kc, 3, out, None, False, 1, 32, 8, 128, 1, 0.1))
    refused(bchip.E_UNSUPPORTED, lambda: ctx.attention(q, kc, kc, bchip.Q4, out, None, False, 1, 32, 8, 80, 1, 0.1))
    refused(bchip.E_UNSUPPORTED, lambda: ctx.attention(q, kc, kc, bchip.Q4, out, None, False, 1, 34, 2, 32, 1, 0.1))
    refused(bchip.E_ARG, lambda: ctx.attention_ragged(q, kc, kc, bchip.Q4, out, [3], [8], 32, 8, 128, 0.1))
    refused(bchip.E_ARG, lambda: ctx.attention_ragged(q, kc, kc, bchip.Q4, out, [0], [1], 32, 8, 128, 0.1))
    refused(bchip.E_ARG, lambda: ctx.attention_ragged(q, kc, kc, bchip.Q4, out, [3], [(1 << 64) // 1024], 32, 8, 128, 0.1))
    refused(bchip.E_UNSUPPORTED, lambda: ctx.attention_ragged(q, kc, kc, bchip.Q4, out, [3], [0], 32, 8, 48, 0.1))
    # Lists whose last tile would end past 2^32.
    refused(bchip.E_UNSUPPORTED, lambda: ctx.attention(q, kc, kc, bchip.Q4, out, None, False, 1, 1, 1, 32, (1 << 32) - 256, 0.1))
    refused(bchip.E_UNSUPPORTED, lambda: ctx.attention_ragged(q, kc, kc, bchip.Q4, out, [(1 << 32) - 255], [0], 1, 1, 32, 0.1))
    for b in (kc, q, out):
        b.free()
