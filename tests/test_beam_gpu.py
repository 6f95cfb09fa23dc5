"""bchip_beam_select against the definition in 64 bits."""
import numpy as np
import pytest

import bchip

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    with bchip.Ctx(0) as c:
        yield c


def select(ctx, scores, sums, k):
    n, beams = sums.shape
    sb, mb = ctx.upload(scores), ctx.upload(sums)
    best, beam, token = (ctx.zeros(n * k * 4) for _ in range(3))
    ctx.beam_select(sb, mb, n, beams, scores.shape[1], k, best, beam, token)
    got = ctx.read(best, (n, k)), ctx.read(beam, (n, k), np.uint32), ctx.read(token, (n, k), np.uint32)
    for x in (sb, mb, best, beam, token):
        x.free()
    return got


def formula(scores, sums):
    """Every continuation's score [searches, beams, vocab] in 64 bits."""
    n, beams = sums.shape
    x = scores.astype(np.float64)
    with np.errstate(invalid="ignore", divide="ignore"):
        m = x.max(1, keepdims=True)
        x = x - m - np.log(np.exp(x - m).sum(1, keepdims=True))
        return x.reshape(n, beams, -1) + sums.astype(np.float64)[:, :, None]


def check(ctx, scores, sums, k):
    """The continuations that come back have the scores of the k best, in order, and are named once; which of
    two it is is settled where their scores lie further apart than a row's sum may be off. Its terms are
    2^x, x = (s - m) log2 e in two roundings, 2^-23 |x| off, so 2^-23 ln 2 |x| of the term; the terms'
    average |x| by their weights is at most log2 of the vocabulary, 20: 2^-19. The instruction's 2^-23, and
    a thread's sum of up to 64 terms one by one, 2^-18, a wave's and the rest in a tree or 64 bits: 2^-17
    holds all. Rounding the result adds 2^-24 of it."""
    n, beams = sums.shape
    vocab = scores.shape[1]
    best, beam, token = select(ctx, scores, sums, k)
    full = formula(scores, sums)
    for i in range(n):
        flat = full[i].reshape(-1)
        order = np.lexsort((np.arange(flat.size), -flat))[:k]
        want = flat[order]
        at = beam[i].astype(np.int64) * vocab + token[i]
        assert (beam[i] < beams).all() and (token[i] < vocab).all()
        assert len(set(at.tolist())) == k
        for j in range(k):
            if want[j] == -np.inf:
                assert best[i, j] == -np.inf and flat[at[j]] == -np.inf
                continue
            tol = 2.0 ** -17 + 2.0 ** -24 * abs(want[j])
            assert abs(best[i, j] - want[j]) <= tol, (i, j, best[i, j], want[j])
            assert abs(flat[at[j]] - want[j]) <= 2 * tol, (i, j, at[j], order[j])
            near = np.abs(flat - want[j]) <= 2 * tol
            if near.sum() == 1:
                assert at[j] == order[j], (i, j, at[j], order[j])


def drawn(rng, n, beams, vocab):
    scores = (2 * rng.standard_normal((n * beams, vocab))).astype(np.float32)
    hot = rng.integers(0, vocab, (n * beams, min(16, vocab)))
    np.put_along_axis(scores, hot, (8 + 6 * rng.random(hot.shape)).astype(np.float32), 1)
    return scores, (-20 - 3 * rng.random((n, beams))).astype(np.float32)


@pytest.mark.parametrize("n,beams,vocab,k", [(1, 1, 1, 1), (1, 1, 5, 5), (3, 2, 7, 14), (1, 4, 1000, 8), (5, 3, 8191, 6), (2, 4, 8193, 64), (1, 64, 500, 64),
                                             (2, 8, 40000, 16), (1, 4, 151936, 8), (1, 2, 600000, 4), (40, 5, 3000, 10), (700, 4, 300, 8), (1, 64, 70000, 64), (5, 1, 256, 6),
                                             (6, 1, 1000, 20), (4, 1, 1025, 64), (2, 3, 2048, 33), (1, 1, 1048576, 64), (1, 5, 900000, 64)])
def test_the_best_continuations(ctx, n, beams, vocab, k):
    rng = np.random.default_rng(vocab + k)
    check(ctx, *drawn(rng, n, beams, vocab), k)


@pytest.mark.parametrize("vocab", [300, 20000])
def test_a_search_that_starts_has_one_beam(ctx, vocab):
    rng = np.random.default_rng(1)
    scores, sums = drawn(rng, 3, 4, vocab)
    sums[:, 1:] = -np.inf
    sums[:, 0] = 0.0
    check(ctx, scores, sums, 8)
    _, beam, _ = select(ctx, scores, sums, 8)
    assert (beam == 0).all()


def test_masked_tokens_and_few_that_are_left(ctx):
    """All but three tokens of each row at -inf: what is left comes first, -inf behind it."""
    rng = np.random.default_rng(2)
    scores, sums = drawn(rng, 2, 3, 9000)
    keep = rng.permutation(9000)[:3]
    masked = np.full_like(scores, -np.inf)
    masked[:, keep] = scores[:, keep]
    check(ctx, masked, sums, 16)
    best, _, token = select(ctx, masked, sums, 16)
    assert np.isin(token[:, :9], keep).all() and (best[:, 9:] == -np.inf).all()
    low = masked.copy()
    low[np.isneginf(low)] = np.finfo(np.float32).min  # a mask of the type's lowest value
    _, _, token = select(ctx, low, sums, 16)
    assert np.isin(token[:, :9], keep).all()


@pytest.mark.parametrize("vocab,k", [(50, 64), (5000, 64), (20000, 7)])
def test_equal_scores_go_by_beam_then_token(ctx, vocab, k):
    scores, sums = np.zeros((6, vocab), np.float32), np.full((2, 3), -1.0, np.float32)
    _, beam, token = select(ctx, scores, sums, k)
    at = np.arange(k)
    assert (beam == at // vocab).all() and (token == at % vocab).all()
    sums[:, 0] = -2.0  # then the first beam last
    _, beam, token = select(ctx, scores, sums, k)
    order = np.concatenate([np.arange(vocab, 3 * vocab), np.arange(vocab)])[:k]
    assert (beam == order // vocab).all() and (token == order % vocab).all()


def test_rows_without_a_distribution_come_last(ctx):
    rng = np.random.default_rng(3)
    scores, sums = drawn(rng, 1, 4, 3000)
    scores[1, 17] = np.nan
    scores[2] = -np.inf
    best, beam, token = select(ctx, scores, sums, 8)
    assert np.isfinite(best).all() and not np.isin(beam, (1, 2)).any()
    scores[0, 5] = np.inf
    scores[3, 5] = np.nan
    best, beam, token = select(ctx, scores, sums, 8)
    assert np.isnan(best).all()
    at = beam[0].astype(np.int64) * 3000 + token[0]
    assert len(set(at.tolist())) == 8 and (token < 3000).all()


def test_reruns(ctx):
    rng = np.random.default_rng(4)
    scores, sums = drawn(rng, 3, 8, 50000)
    a, b = select(ctx, scores, sums, 16), select(ctx, scores, sums, 16)
    for x, y in zip(a, b):
        np.testing.assert_array_equal(x.view(np.uint32), y.view(np.uint32))


@pytest.mark.parametrize("beams,vocab", [(8, 200000), (30, 151936)])
@pytest.mark.parametrize("form", ["equal", "slope", "plateau", "masked"])
def test_many_groups_at_once(ctx, beams, vocab, form):
    """Searches of more groups than one round holds a thread's few of: scores all equal (first beams, first tokens),
    falling slowly along the vocabulary (the best side by side), a few levels, and all but one token masked."""
    rng = np.random.default_rng(vocab)
    sums = np.zeros((1, beams), np.float32)
    if form == "equal":
        scores = np.zeros((beams, vocab), np.float32)
    elif form == "slope":
        scores = np.tile(np.linspace(8, -8, vocab).astype(np.float32), (beams, 1))
        sums[0] = -0.001 * np.arange(beams)
    elif form == "plateau":
        scores = rng.integers(0, 3, (beams, vocab)).astype(np.float32)
        sums[0] = -np.arange(beams)
    else:
        scores = np.full((beams, vocab), -np.inf, np.float32)
        scores[np.arange(beams), rng.integers(0, vocab, beams)] = 1.0
        sums[0] = -rng.random(beams)
    for k in (1, 33, 64):
        check(ctx, scores, sums, k)
        if form in ("equal", "masked"):
            best, beam, token = select(ctx, scores, sums, k)
            got = list(zip(beam[0].tolist(), token[0].tolist()))
            if form == "equal":
                assert got == [(0, t) for t in range(k)]
            else:
                assert got[:beams] == [(b, int(scores[b].argmax())) for b in np.argsort(-sums[0])][:k]
