"""bchip_logprobs over every number of workgroups a row can have: from a workgroup for each block of a
row, which few rows take, to one for whole rows, which thousands take. A row's results are the same
bits in all of them, and with or without scratch."""
import numpy as np
import pytest

import bchip

pytestmark = pytest.mark.gpu

VOCAB, TOP, KINDS = 40001, 7, 50  # five blocks a row


@pytest.fixture(scope="module")
def rows_and_results():
    """A context, score rows on the device (KINDS of them, again and again), and each kind's results alone."""
    r = np.random.default_rng(21)
    s = (r.standard_normal((KINDS, VOCAB)) * 3).astype(np.float32)
    s[3] = np.floor(s[3])           # ties
    s[4, 100:39000] = -np.inf
    s[5, 17], s[6, 40000] = np.nan, np.inf
    s[7] = np.sort(s[7])
    tokens = r.integers(0, VOCAB, KINDS).astype(np.uint32)
    tokens[8] = VOCAB
    with bchip.Ctx(0) as c:
        most = 2200
        scores, tk = c.zeros(most * VOCAB * 4), c.upload(np.resize(tokens, most))
        c.upload(s, scores)
        for at in range(KINDS, most, KINDS):
            n = min(KINDS, most - at)
            c.copy(scores, bchip.F32, scores, bchip.F32, at * VOCAB, n * VOCAB)
        alone = [results(c, scores, tk, i, 1) for i in range(KINDS)]
        yield c, scores, tk, [np.concatenate([a[k] for a in alone]) for k in range(4)], s


def outs(c, rows):
    return [c.zeros(rows * 4), c.zeros(rows * 4), c.zeros(rows * TOP * 4), c.zeros(rows * TOP * 4)]


def run(c, scores, tk, first, rows, o):
    c.logprobs(scores.offset(first * VOCAB * 4), rows, VOCAB, 0.9, tk.offset(first * 4), o[0], o[1], TOP, o[2], o[3])


def read(c, rows, o):
    return [c.read(o[0], rows, np.uint32), c.read(o[1], rows, np.uint32), c.read(o[2], (rows, TOP), np.uint32), c.read(o[3], (rows, TOP), np.uint32)]


def results(c, scores, tk, first, rows):
    o = outs(c, rows)
    run(c, scores, tk, first, rows, o)
    got = read(c, rows, o)
    for b in o:
        b.free()
    return got


def test_the_rows_are_what_they_should_be(rows_and_results):
    """Against log softmax in 64 bits. x = (s - m) / T rounds three times and e^x twice more, 2^-24 each,
    the exponent's by |x|, whose weighted mean is at most the entropy, under 12; a thread sums 32 terms a
    block and ten sums of pairs follow: log L is off by at most 2^-24 (4 x 12 + 32 + 20) < 2^-17, and x by
    2^-22 of itself."""
    _, _, _, alone, s = rows_and_results
    for i in (0, 7, 20):
        x = s[i].astype(np.float64) / np.float64(np.float32(0.9))
        lp = x - x.max() - np.log(np.exp(x - x.max()).sum())
        best = np.lexsort((np.arange(VOCAB), -s[i]))[:TOP]
        np.testing.assert_array_equal(alone[2][i], best)
        np.testing.assert_allclose(alone[3][i].view(np.float32), lp[best], rtol=2.0 ** -22, atol=2.0 ** -17)
    assert np.isnan(alone[0].view(np.float32)[[5, 6, 8]]).all()


# Workgroups a row: 5, 3, 2, 2, 1, 1.
@pytest.mark.parametrize("rows", [50, 700, 1024, 2047, 2048, 2200])
def test_a_rows_bits_are_those_of_its_own_call(rows_and_results, rows):
    c, scores, tk, alone, _ = rows_and_results
    for got, want in zip(results(c, scores, tk, 0, rows), alone):
        np.testing.assert_array_equal(got, np.resize(want, (rows,) + want.shape[1:]))


def test_a_captured_call_gives_the_same_bits(rows_and_results):
    """On a context without scratch, and once there is some, on every replay."""
    from test_matmul_scratch_gpu import captured, hip
    _, _, _, alone, s = rows_and_results
    with bchip.Ctx(0) as c:
        scores, tk, o = c.upload(s[9:14]), c.zeros(20), outs(c, 5)
        call = lambda: run(c, scores, tk, 0, 5, o)
        graphs = [captured(c, call)]
        call()
        want = read(c, 5, o)
        for k in (1, 2, 3):
            np.testing.assert_array_equal(want[k], alone[k][9:14])
        graphs.append(captured(c, call))
        for _ in range(3):
            for stream, graph in graphs:
                for b in o:
                    c.upload(np.zeros(b.nbytes, np.uint8), b)
                hip("hipGraphLaunch", graph, stream)
                for got, w in zip(read(c, 5, o), want):
                    np.testing.assert_array_equal(got, w)
        for _, graph in graphs:
            hip("hipGraphExecDestroy", graph)
