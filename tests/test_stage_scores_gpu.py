"""GpuLayers.logprobs and GpuLayers.sample in pieces of rows: the results of the rows at once, bit for
bit, and those of the scores that GpuLayers.logits gives."""
import numpy as np
import pytest

import bchip
import oracle as O
from layers import Config, GpuLayers, Matrix

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = bchip.Ctx(0)
    yield c
    c.close()


@pytest.mark.parametrize("ty", [O.Q8_0, O.Q4K, O.F16], ids=lambda t: O.TYPE_NAMES[t])
@pytest.mark.parametrize("rows,vocab,upto", [(1, 4000, None), (3, 4000, 3999), (70, 4000, None), (301, 1003, None), (301, 20000, 17000)])
def test_pieces_do_not_change_a_result(ctx, ty, rows, vocab, upto):
    e = 512
    r = np.random.default_rng(rows + vocab)
    cfg = Config(n_embd=e, n_layer=0, n_head=4, n_head_kv=4, head_dim=128, rope_dim=128, vocab=vocab)
    some = np.asarray(O.random_tensor(ty, 301, e, 5), np.uint8).reshape(301, -1)
    data = np.resize(some, (vocab, some.shape[1])).tobytes()
    g = GpuLayers(ctx, cfg, [], head=(np.ones(e, np.float32), Matrix(ty, data, vocab, e)))
    x = (r.standard_normal((rows, e)) * 2).astype(np.float32)
    n = upto or vocab
    tokens = r.integers(0, n, rows)

    def results():
        return [*g.logprobs(x, rows, tokens, top=5, temperature=0.8, upto=upto), *g.logprobs(x, rows, upto=upto)[1:2],
                g.sample(x, rows, 0.7, 0.9, 11, 3, upto=upto), g.sample(x, rows, 0.0, 1.0, 11, 3, upto=upto)]

    want = results()
    scores = g.logits(x, rows, upto).astype(np.float64)
    np.testing.assert_array_equal(want[-1], scores.argmax(1))
    np.testing.assert_array_equal(want[2], np.argsort(-scores, 1, kind="stable")[:, :5])
    for most in (7 * n * 4, 2 * n * 4, 1):
        g.SCORE_BYTES = most
        for a, b in zip(results(), want):
            np.testing.assert_array_equal(np.asarray(a).view(np.uint32), np.asarray(b).view(np.uint32))
    g.free()
