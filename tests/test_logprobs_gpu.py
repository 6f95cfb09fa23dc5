"""bchip_logprobs against log_softmax in 64 bits: every form of row (odd vocabularies whose rows
start anywhere, one workgroup a row and many), ties, masks of -inf, NaN and infinities, peaked
rows whose log probabilities are tiny, temperatures, and what may be left out.

Bounds: x = (s - m) / T rounds three times and e^x twice more, 2^-24 each, the exponent's by |x|; a
thread sums at most 32 terms a block of 8192 scores, then come ten sums of pairs. Terms count by
e^x, and so weighted |x| averages at most the entropy, under 12 here: log L is off by at most 2^-24
(4 x 12 + 32 x 2 + 20) < 2^-17 of the terms' share, an entropy, of two such sums, by twice that. In
a peaked row the share is log L itself: a value of size a is within 2^-17 a, or 2^-22 |x| from x."""
import numpy as np
import pytest

import bchip

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = bchip.Ctx(0)
    yield c
    c.close()


def plain(s, T, tokens, top):
    s = s.astype(np.float64)
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        x = (s - np.where(np.isnan(s), -np.inf, s).max(1, keepdims=True)) / np.float64(np.float32(T))
        e = np.exp(x)
        big = e == 1
        rest = np.where(big, 0, e).sum(1)
        n = big.sum(1)
        log_l = np.where(n == 1, np.log1p(rest), np.log(n + rest))
        lp = x - log_l[:, None]
        p = e / (n + rest)[:, None]
        ent = log_l - np.where(e > 0, p * x, np.where(np.isnan(e), np.nan, 0)).sum(1)
    # Descending, ties by id, NaN last.
    ids = np.stack([np.lexsort((np.arange(s.shape[1]), -np.where(np.isnan(r), -np.inf, r), np.isnan(r)))[:top] for r in s]) \
        if top else np.zeros((len(s), 0), int)
    tok = np.array([lp[r, t] if t < s.shape[1] else np.nan for r, t in enumerate(tokens)])
    return tok, ent, ids.astype(np.uint32), np.take_along_axis(lp, ids, 1), log_l


def call(ctx, s, T, tokens, top, offset=0):
    """The call's results, its scores at an address `offset` floats into their buffer."""
    rows, vocab = s.shape
    sb = ctx.zeros((s.size + offset) * 4)
    ctx.upload(s, sb, offset * 4)
    tb = ctx.upload(np.asarray(tokens, np.uint32))
    lb, eb, ib, pb = (ctx.upload(np.full(n + 1, 7, np.float32)) for n in (rows, rows, rows * top, rows * top))
    ctx.logprobs(sb.offset(offset * 4), rows, vocab, T, tb, lb, eb, top, ib if top else None, pb if top else None)
    got = ctx.read(lb, rows + 1), ctx.read(eb, rows + 1), ctx.read(ib, rows * top + 1, np.uint32), ctx.read(pb, rows * top + 1)
    for b in (sb, tb, lb, eb, ib, pb):
        b.free()
    assert got[0][-1] == got[1][-1] == got[3][-1] == 7 and got[2][-1:].view(np.float32) == 7  # nothing behind the results
    return got[0][:-1], got[1][:-1], got[2][:-1].reshape(rows, top), got[3][:-1].reshape(rows, top)


def check(got, want, what):
    tok, ent, ids, tops = got
    np.testing.assert_array_equal(ids, want[2], err_msg=what)
    size = np.abs(want[4])
    for name, g, w, lim in (("logprob", tok, want[0], size), ("entropy", ent, want[1], None), ("top", tops, want[3], size[:, None])):
        np.testing.assert_array_equal(np.isnan(g), np.isnan(w), err_msg=f"{what}: {name}")
        np.testing.assert_array_equal(np.isneginf(g), np.isneginf(w), err_msg=f"{what}: {name}")
        fine = np.isfinite(w)
        with np.errstate(invalid="ignore"):
            err = np.abs(g - w)
        scale = np.minimum(lim, 1) * 2.0 ** -17 + np.abs(w) * 2.0 ** -22 if lim is not None else 2.0 ** -16 * np.minimum(w + 2.0 ** -8, 1)
        scale = np.broadcast_to(scale, w.shape)
        assert (err[fine] <= scale[fine] + 1e-38).all(), f"{what}: {name} off by {np.max(err[fine] / scale[fine])} of the bound"


def rows_of(rows, vocab, seed, peak=True):
    r = np.random.default_rng(seed)
    s = (r.standard_normal((rows, vocab)) * 2).astype(np.float32)
    if peak:
        for i in range(rows):
            at = r.integers(0, vocab, 32)
            s[i, at] += (4 + 8 * r.random(32)).astype(np.float32)
    return s


@pytest.mark.parametrize("vocab", [1, 2, 37, 255, 1000, 8191, 8192, 8193, 32000, 128256, 151936])
@pytest.mark.parametrize("rows,top,T", [(1, 1, 1.0), (3, 5, 0.7), (5, 20, 1.0), (2, 64, 1.3), (4, 0, 0.3), (3, 33, 1.0), (2, 8, 1.0), (2, 9, 2.0)])
def test_rows_of_scores(ctx, vocab, rows, top, T):
    top = min(top, vocab)
    s = rows_of(rows, vocab, vocab + rows)
    tokens = np.random.default_rng(rows).integers(0, vocab, rows)
    tokens[0] = s[0].argmax()
    check(call(ctx, s, T, tokens, top, offset=rows % 4), plain(s, T, tokens, top), f"{rows} x {vocab}, top {top}, T {T}")


@pytest.mark.parametrize("vocab", [5000, 20000, 600001])
@pytest.mark.parametrize("top", [1, 20, 64])
def test_orders_that_are_not_random(ctx, vocab, top):
    """Ascending and descending scores, all equal, two values, masks that leave few, one or no
    token, blocks of -inf, NaN and infinities."""
    r = np.random.default_rng(top)
    s = np.tile((r.standard_normal(vocab) * 2).astype(np.float32), (14, 1))
    s[0].sort()
    s[1] = s[0][::-1]
    s[2] = 3.25
    s[3] = np.where(r.random(vocab) < 0.5, 1.0, 2.0)
    s[4][r.random(vocab) > 30 / vocab] = -np.inf
    s[5] = -np.inf
    s[5, vocab // 2] = 1.5
    s[6] = -np.inf
    s[7, : vocab * 3 // 4] = -np.inf
    s[8, 17] = np.nan
    s[9] = np.nan
    s[10, [3, vocab - 1]] = np.inf
    s[11] = np.where(r.random(vocab) < 0.5, 0.0, -0.0)
    s[12] = np.finfo(np.float32).min
    s[12, 9] = 0
    s[13, 100:] = np.nan
    tokens = np.array([0, 0, 5, 7, 11, vocab // 2, 3, 2, 3, 4, 3, 2, 9, 50])
    check(call(ctx, s, 1.0, tokens, top), plain(s, 1.0, tokens, top), f"{vocab}, top {top}")


def test_peaked_rows_keep_their_digits(ctx):
    """The likeliest token's log probability down to 1e-30."""
    vocab = 40000
    s = rows_of(8, vocab, 3, peak=False)
    best = np.arange(8) * 4999 + 1
    for i in range(8):
        s[i, best[i]] = s[i].max() + 10 * i
    got, want = call(ctx, s, 1.0, best, 3), plain(s, 1.0, best, 3)
    check(got, want, "peaked")
    np.testing.assert_allclose(got[0], want[0], rtol=2e-5)
    np.testing.assert_allclose(got[1], want[1], rtol=2e-5)


def test_what_is_left_out_is_left_alone_and_ids_past_the_vocabulary_are_nan(ctx):
    s = rows_of(3, 30000, 5)
    sb, tb = ctx.upload(s), ctx.upload(np.array([5, 30000, 0xFFFFFFFF], np.uint32))
    lb, eb, ib, pb = ctx.zeros(12), ctx.zeros(12), ctx.zeros(3 * 7 * 4), ctx.zeros(3 * 7 * 4)
    tok, ent, ids, tops, _ = plain(s, 1.0, [5, 30000, 30000], 7)
    ctx.logprobs(sb, 3, 30000, 1.0, tb, lb, None, 0, None, None)
    got = ctx.read(lb, 3)
    assert abs(got[0] - tok[0]) < 1e-4 and np.isnan(got[1:]).all()
    ctx.logprobs(sb, 3, 30000, 1.0, None, None, eb, 0, None, None)
    np.testing.assert_allclose(ctx.read(eb, 3), ent, rtol=2e-5)
    ctx.logprobs(sb, 3, 30000, 1.0, None, None, None, 7, ib, pb)
    np.testing.assert_array_equal(ctx.read(ib, (3, 7), np.uint32), ids)
    ctx.logprobs(sb, 3, 30000, 1.0, None, None, None, 0, None, None)
    ctx.logprobs(sb, 0, 30000, 1.0, None, None, None, 0, None, None)
    for b in (sb, tb, lb, eb, ib, pb):
        b.free()


def test_many_rows(ctx):
    """Rows past what one launch's scratch holds, each the bits of its own call."""
    rows, vocab, top = 8000, 9001, 64
    s = np.tile(rows_of(40, vocab, 6), (rows // 40, 1))
    tokens = np.arange(rows) % vocab
    got = call(ctx, s, 1.0, tokens, top)
    one = call(ctx, s[:40], 1.0, tokens[:40], top)
    for a, b in zip(got[1:], one[1:]):
        np.testing.assert_array_equal(a, np.tile(b, (rows // 40,) + (1,) * (b.ndim - 1)))
    np.testing.assert_array_equal(got[0][:40], one[0])


def test_rows_of_several_blocks_a_workgroup(ctx):
    """More rows than workgroups: each takes a row's blocks in turn and keeps the best of them. Rows whose
    best come in order, equal ones, masks that leave few numbers, and NaNs beside -inf alone."""
    rows, vocab, top = 1030, 20001, 20
    r = np.random.default_rng(11)
    x = (r.standard_normal((rows, vocab)) * 3).astype(np.float32)
    x[1] = np.linspace(-5, 5, vocab)
    x[2] = x[1][::-1]
    x[3] = 0.5
    x[4, :19000] = -np.inf
    x[5] = -np.inf
    x[5, [3, 8200, 16500]] = 1.0, 3.0, 2.0
    x[6, :17000] = 1.0
    x[7] = np.floor(x[7])
    x[8] = np.nan                        # -inf and one number among NaNs
    x[8, 9000:9030], x[8, 20000] = -np.inf, 7.0
    x[9, 10000] = np.nan
    tokens = r.integers(0, vocab, rows).astype(np.uint32)
    tokens[3:8] = 5, 19500, 8200, 17500, 1
    check(call(ctx, x, 1.0, tokens, top), plain(x, 1.0, tokens, top), "several blocks")
    few = call(ctx, x[:40], 1.0, tokens[:40], top)
    for a, b in zip(call(ctx, x, 1.0, tokens, top), few):
        np.testing.assert_array_equal(a[:40], b)  # the bits do not depend on the rows beside


def test_a_captured_call(ctx):
    """Under capture a fresh context has no scratch: a workgroup takes each row. The same ids; values
    within rounding; and once scratch is there, a graph that took it survives a larger call."""
    from test_matmul_scratch_gpu import captured, hip
    s = rows_of(3, 70000, 8)
    want = plain(s, 1.0, [1, 2, 3], 20)
    with bchip.Ctx(0) as c:
        sb, tb = c.upload(s), c.upload(np.array([1, 2, 3], np.uint32))
        lb, eb, ib, pb = c.zeros(12), c.zeros(12), c.zeros(240), c.zeros(240)
        step = lambda: c.logprobs(sb, 3, 70000, 1.0, tb, lb, eb, 20, ib, pb)
        graphs = [captured(c, step)]
        step()
        graphs.append(captured(c, step))
        big = c.zeros(600 * 70000 * 4)
        bi, bp = c.zeros(600 * 64 * 4), c.zeros(600 * 64 * 4)
        for _ in range(3):
            c.logprobs(big, 600, 70000, 1.0, None, None, None, 64, bi, bp)
            for stream, graph in graphs:
                for b in (lb, eb, ib, pb):
                    c.upload(np.zeros(b.nbytes, np.uint8), b)
                hip("hipGraphLaunch", graph, stream)
                check((c.read(lb, 3), c.read(eb, 3), c.read(ib, (3, 20), np.uint32), c.read(pb, (3, 20))), want, "replayed")
        for _, graph in graphs:
            hip("hipGraphExecDestroy", graph)


def test_a_row_without_scratch_gives_the_same_bits(ctx):
    from test_matmul_scratch_gpu import captured, hip
    s, tokens = rows_of(3, 70000, 9), [69999, 0, 35000]
    want = call(ctx, s, 0.7, tokens, 20)
    with bchip.Ctx(0) as c:  # nothing has run here: under capture no scratch can be had
        sb, tb = c.upload(s), c.upload(np.array(tokens, np.uint32))
        lb, eb, ib, pb = c.zeros(12), c.zeros(12), c.zeros(240), c.zeros(240)
        stream, graph = captured(c, lambda: c.logprobs(sb, 3, 70000, 0.7, tb, lb, eb, 20, ib, pb))
        hip("hipGraphLaunch", graph, stream)
        got = c.read(lb, 3), c.read(eb, 3), c.read(ib, (3, 20), np.uint32), c.read(pb, (3, 20))
        hip("hipGraphExecDestroy", graph)
    for a, b in zip(got, want):
        np.testing.assert_array_equal(a, b)


def test_bad_arguments_are_refused(ctx):
    s, o, w = ctx.zeros(4 * 2000), ctx.zeros(4 * 100), ctx.zeros(4 * 1)

    def refused(fn):
        with pytest.raises(bchip.BchipError) as e:
            fn()
        assert e.value.code == bchip.E_ARG, bchip.last_error()

    for T in (0.0, -1.0, float("nan"), float("inf"), 1e-7):
        refused(lambda: ctx.logprobs(s, 2, 1000, T, o, o, o, 0, None, None))
    refused(lambda: ctx.logprobs(None, 2, 1000, 1.0, o, o, o, 0, None, None))
    refused(lambda: ctx.logprobs(s, 2, 1000, 1.0, o, None, o, 0, None, None))
    refused(lambda: ctx.logprobs(s, 2, 1000, 1.0, None, o, o, 0, None, None))
    refused(lambda: ctx.logprobs(s, 2, 1000, 1.0, o, o, o, 5, None, o))
    refused(lambda: ctx.logprobs(s, 2, 1000, 1.0, o, o, o, 65, o, o))
    refused(lambda: ctx.logprobs(s, 2, 3, 1.0, o, o, o, 4, o, o))
    refused(lambda: ctx.logprobs(s, 2, 0, 1.0, o, o, o, 0, o, o))
    refused(lambda: ctx.logprobs(s, 3, 1000, 1.0, o, o, o, 0, None, None))      # past the scores
    refused(lambda: ctx.logprobs(s, 2, 1000, 1.0, w, o, o, 0, None, None))      # past the tokens
    refused(lambda: ctx.logprobs(s, 2, 1000, 1.0, o, o, w, 0, None, None))
    refused(lambda: ctx.logprobs(s, 2, 1000, 1.0, o, o, o, 60, o, o))           # past the ids
    refused(lambda: ctx.logprobs(s, 70000, 1, 1.0, None, None, None, 0, None, None))
    for b in (s, o, w):
        b.free()
