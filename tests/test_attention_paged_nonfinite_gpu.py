"""bchip_attention_paged where a K or V is not finite or a page is missing, over head dims of every kernel and at
every part of a tile: what a row does not see leaves it as it is. Each kernel looks through the tiles that some
of its rows see a part of, by a share of the tile's bytes a thread, which not every head dim divides."""
import numpy as np
import pytest

import bchip
from paged_plain import Batch
from test_attention_paged_gpu import call, expect

pytestmark = pytest.mark.gpu

DIMS = [8, 32, 64, 72, 80, 96, 128, 160, 192, 200, 256]
G, NKV = 2, 2
# New rows and slots: up to 16 query rows a KV head, 17 to 64, and more, the new slots at the start, in the
# middle and at the end of a tile of 64.
ROWS = [(6, 64), (6, 40), (8, 200), (30, 192), (32, 128), (20, 200), (31, 150), (130, 130), (100, 192), (90, 250)]


@pytest.fixture(scope="module")
def ctx():
    with bchip.Ctx(0) as c:
        yield c


def batches(rng, rows, n, hd, kv_type, beside):
    """The pass alone, and beside a step of another sequence (both kinds of blocks in one launch)."""
    return Batch(rng, [rows] + [1] * beside, [n] + [50] * beside, NKV, hd, kv_type)


@pytest.mark.parametrize("kv_type", [bchip.F16, bchip.F32])
@pytest.mark.parametrize("hd", DIMS)
@pytest.mark.parametrize("beside", [0, 1])
def test_values_in_any_place_of_a_tile(ctx, beside, hd, kv_type):
    rng = np.random.default_rng(hd + beside)
    nh, scale = G * NKV, hd ** -0.5
    for rows, n in ROWS:
        b = batches(rng, rows, n, hd, kv_type, beside)
        q = rng.standard_normal((b.total, nh, hd)).astype(np.float32)
        clean = list(expect(b, q, nh, scale))
        p, o = b.places(0)
        for slot in sorted({n - 1, n - rows + 1, *rng.integers(n - rows + 1, n, 3).tolist()}):
            for which, bad, dim in (("v", np.inf, hd - 1), ("v", np.nan, 3), ("k", -np.inf, 1)):
                pool = getattr(b, which)
                kept = pool[p[slot], o[slot], 1, dim]
                pool[p[slot], o[slot], 1, dim] = bad
                got = call(ctx, b, q, nh, scale)
                pool[p[slot], o[slot], 1, dim] = kept
                for i, at, want, most in clean:
                    ok = np.abs(got[at] - want) <= most
                    if i == 0:
                        ok[slot - (n - rows):, G:] = True  # unspecified: rows that see the slot, heads of that KV head
                    assert ok.all(), f"{rows} rows at {n}, {which} {bad} in slot {slot}: sequence {i}, rows {np.flatnonzero(~ok.all((1, 2)))}"


@pytest.mark.parametrize("kv_type", [bchip.F16, bchip.F32])
@pytest.mark.parametrize("hd", DIMS)
def test_a_full_slot_of_values(ctx, hd, kv_type):
    """Every V of a slot, in every slot that some rows of a pass of 60 query rows see and some do not."""
    rng = np.random.default_rng(hd)
    nh, scale, rows, n = G * NKV, hd ** -0.5, 30, 128
    b = batches(rng, rows, n, hd, kv_type, 0)
    q = rng.standard_normal((b.total, nh, hd)).astype(np.float32)
    _, at, want, most = next(expect(b, q, nh, scale))
    p, o = b.places(0)
    for slot in range(n - rows + 1, n):
        kept = b.v[p[slot], o[slot]].copy()
        b.v[p[slot], o[slot]] = np.nan
        got = call(ctx, b, q, nh, scale)
        b.v[p[slot], o[slot]] = kept
        first = slot - (n - rows)
        ok = (np.abs(got - want) <= most)[:first]
        assert ok.all(), f"slot {slot}: rows {np.flatnonzero(~ok.all((1, 2)))} of the {first} before it"


@pytest.mark.parametrize("kv_type", [bchip.F16, bchip.F32])
@pytest.mark.parametrize("hd", DIMS)
def test_pages_past_the_pool(ctx, hd, kv_type):
    rng = np.random.default_rng(hd + 1)
    nh, scale = G * NKV, hd ** -0.5
    for rows, n in ((1, 333), (6, 40), (20, 200), (30, 192), (130, 130)):
        b = batches(rng, rows, n, hd, kv_type, 1)
        q = rng.standard_normal((b.total, nh, hd)).astype(np.float32)
        clean = list(expect(b, q, nh, scale))
        for page in {(n - 1) // 16, (n - rows // 2) // 16}:
            kept = b.table[0, page]
            b.table[0, page] = b.npages
            got = call(ctx, b, q, nh, scale)
            b.table[0, page] = kept
            for i, at, want, most in clean:
                sees = (n - rows + np.arange(rows) >= 16 * page) if i == 0 else np.zeros(1, bool)
                assert np.isnan(got[at][sees]).all(), (rows, n, page, i)
                assert (np.abs(got[at] - want) <= most)[~sees].all(), (rows, n, page, i)


@pytest.mark.parametrize("kv_type", [bchip.F16, bchip.F32])
@pytest.mark.parametrize("hd", DIMS)
def test_queries_that_are_not_finite(ctx, hd, kv_type):
    rng = np.random.default_rng(hd + 2)
    nh, scale = G * NKV, hd ** -0.5
    for rows, n in ((1, 100), (6, 100), (30, 100), (90, 100)):
        b = batches(rng, rows, n, hd, kv_type, 1)
        clean = rng.standard_normal((b.total, nh, hd)).astype(np.float32)
        q = clean.copy()
        q[rows // 2, 1, hd - 1] = np.nan
        q[rows // 2, 2, 0] = np.inf
        got = call(ctx, b, q, nh, scale)
        assert np.isnan(got[rows // 2, 1]).all()
        for i, at, want, most in expect(b, clean, nh, scale):
            ok = np.abs(got[at] - want) <= most
            if i == 0:
                ok[rows // 2, 1:3] = True
            assert ok.all(), (rows, i)
