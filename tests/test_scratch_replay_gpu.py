"""Graphs captured over calls that took scratch, replayed after larger calls of the same context have
outgrown it: the eager call's bits, on every replay."""
import numpy as np
import pytest

import bchip
import oracle as O
from test_matmul_scratch_gpu import captured, hip

pytestmark = pytest.mark.gpu


def matmul(c, r):
    rows, cols, n = 1000, 4096, 12
    w, x, out = c.upload(np.asarray(O.random_tensor(O.Q8_0, rows, cols, 3), np.uint8)), c.upload(r.standard_normal((n, cols)).astype(np.float32)), c.zeros(n * rows * 4)
    return lambda: c.matmul(w, O.Q8_0, x, out, rows, cols, n), [(out, n * rows)]


def sample(c, r):
    rows, vocab = 2, 30000
    s, ids = c.upload(r.standard_normal((rows, vocab)).astype(np.float32)), c.zeros(rows * 4)
    return lambda: c.sample(s, rows, vocab, 0.8, 0.95, 5, 0, ids), [(ids, rows)]


def attention(t, rows, n):
    def make(c, r):
        nh, nkv, hd = 16, 4, 128
        x = c.upload(r.standard_normal(n * nkv * hd).astype(np.float32))
        q, out = c.upload(r.standard_normal(rows * nh * hd).astype(np.float32)), c.zeros(rows * nh * hd * 4)
        kv = c.zeros(bchip.nbytes_of(t, n * nkv * hd))
        c.copy(x, bchip.F32, kv, t, 0, n * nkv * hd)
        return lambda: c.attention(q, kv, kv, t, out, None, False, rows, nh, nkv, hd, n - rows, 0.09), [(out, rows * nh * hd)]
    return make


def fused_step(c, r):
    nh, nkv, hd, n = 16, 4, 128, 1500
    kvd = nkv * hd
    was = c.upload(r.standard_normal(n * kvd).astype(np.float16))
    q0, k = c.upload(r.standard_normal(nh * hd).astype(np.float32)), c.upload(r.standard_normal(kvd).astype(np.float32))
    q, out, kv = c.zeros(nh * hd * 4), c.zeros(nh * hd * 4), c.zeros(n * kvd * 2)
    c.copy(was, bchip.F16, kv, bchip.F16, 0, n * kvd)
    freq, pos = c.upload(O.inv_freq(hd, 1e4)), c.upload(np.array([n - 1], np.uint32))

    def call():
        c.copy(q0, bchip.F32, q, bchip.F32, 0, nh * hd)  # (the step rotates q in place)
        c.rope_append_attention(q, k, k, kv, kv, bchip.F16, freq, pos, nh, nkv, hd, hd, False, n - 1, 0.09, out)
    return call, [(out, nh * hd), (q, nh * hd)]


CALLS = {"matmul": matmul, "sample": sample, "f16 step": attention(bchip.F16, 1, 3000), "f16 verify": attention(bchip.F16, 12, 3000),
         "f32 verify": attention(bchip.F32, 12, 3000), "4-bit step": attention(bchip.Q4, 1, 5000), "4-bit verify": attention(bchip.Q4, 12, 3000),
         "f16 fused step": fused_step}


@pytest.mark.parametrize("name", CALLS)
def test_a_graph_replayed_after_larger_calls(name):
    r = np.random.default_rng(7)
    with bchip.Ctx(0) as c:
        call, outs = CALLS[name](c, r)
        call()
        want = [c.read(b, n, np.uint32) for b, n in outs]
        assert all(w.any() for w in want)
        s, ex = captured(c, call)
        # Larger calls: keys, states of a long f16 list and of a 4-bit pass.
        vocab, rows = 60000, 300
        scores, ids, lp = c.zeros(rows * vocab * 4), c.zeros(rows * 64 * 4), c.zeros(rows * 64 * 4)
        big16, big4 = attention(bchip.F16, 8, 30000)(c, r)[0], attention(bchip.Q4, 600, 9000)(c, r)[0]
        for _ in range(3):
            c.sample(scores, rows, vocab, 1.0, 0.9, 1, 0, ids)
            c.logprobs(scores, rows, vocab, 1.0, None, None, None, 64, ids, lp)
            big16()
            big4()
            for b, n in outs:
                c.upload(np.zeros(n, np.uint32), b)
            hip("hipGraphLaunch", ex, s)
            for (b, n), w in zip(outs, want):
                np.testing.assert_array_equal(c.read(b, n, np.uint32), w)
        hip("hipGraphExecDestroy", ex)
