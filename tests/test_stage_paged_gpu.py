"""A stage over a cache in pages, as it is used: pieces of prompts and tokens of several conversations in
one pass, forks, conversations that end and give their pages back, and beam search over forks
(GpuLayers.forward_paged, GpuLayers.beams, bchip.PagePool), against the same layers in f64
(tiny_model.RefModel); and the calls captured into graphs."""
import numpy as np
import pytest

import bchip
import oracle as O
from layers import GpuLayers
from paged_plain import Batch
from test_matmul_scratch_gpu import captured, hip
from tiny_model import RefModel, embed, tiny_model, wide_model

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    with bchip.Ctx(0) as c:
        yield c


# f32 layers are held to the reference's own bound of a batch row (model.rs:641-642); a cache in f16 rounds
# K and V by 2^-11 of themselves, to the bound that the f16 layers are held to elsewhere.
BARS = {bchip.F32: 1e-4, bchip.F16: 5e-3}


class Texts:
    """Conversations of one pool beside their texts; every pass is checked against the f64 layers over the texts."""

    def __init__(self, ctx, model, kv_type, npages, page_slots=16):
        cfg, layers, head, self.embd = model
        self.cfg, self.kv_type = cfg, kv_type
        self.g, self.ref = GpuLayers(ctx, cfg, layers, head, kv_type), RefModel(cfg, layers, head)
        self.pool = self.g.new_pool(npages, page_slots)
        self.text = {}

    def start(self):
        s = self.pool.new()
        self.text[s] = []
        return s

    def fork(self, s):
        f = self.pool.fork(s)
        self.text[f] = list(self.text[s])
        return f

    def drop(self, s):
        self.pool.drop(s)
        del self.text[s]

    def want(self, s):
        """The f64 states of a whole text."""
        return self.ref.forward(embed(self.embd, self.text[s]), 0, None, self.ref.new_cache())

    def go(self, seqs, new):
        """Each conversation's new tokens in one pass; their states, checked."""
        x = self.g.forward_paged(embed(self.embd, [t for n in new for t in n]) if any(new) else np.zeros((0, self.cfg.n_embd), np.float32),
                                 seqs, [len(n) for n in new], self.pool)
        at = 0
        for s, n in zip(seqs, new):
            self.text[s] += n
            if n:
                want = self.want(s)[-len(n):]
                err = np.abs(x[at:at + len(n)] - want).max()
                assert err <= BARS[self.kv_type] * (1 + np.abs(want).max()), (s, len(n), err)
            at += len(n)
        return x

    def free(self):
        self.pool.free()
        self.g.free()


@pytest.mark.parametrize("kv_type", [bchip.F32, bchip.F16])
@pytest.mark.parametrize("model,neox", [(tiny_model, False), (wide_model, True)])
def test_conversations_in_one_pool(ctx, model, neox, kv_type):
    t = Texts(ctx, model(2, neox), kv_type, 60)
    r = np.random.default_rng(1)
    tok = lambda n: r.integers(0, t.cfg.vocab, n).tolist()  # noqa: E731
    a, b = t.start(), t.start()
    t.go([a, b], [tok(37), tok(5)])
    c = t.start()
    t.go([b, c, a], [tok(1), tok(150), tok(1)])
    t.go([a, b, c], [tok(1), [], tok(40)])
    f = t.fork(c)
    t.go([c, f, a], [tok(1), tok(3), tok(1)])      # c and f part inside a page
    t.go([f, c], [tok(1), tok(1)])
    t.pool.truncate(a, 20)                          # rows that were not accepted
    t.text[a] = t.text[a][:20]
    t.go([a, f], [tok(4), tok(20)])
    t.drop(c)                                       # its pages go to the next
    d = t.start()
    t.go([d, f], [tok(170), tok(1)])
    t.go([a, b, d, f], [tok(1)] * 4)
    t.go([a], [tok(1)])
    t.go([b, d], [[], []])
    t.free()


@pytest.mark.parametrize("kv_type", [bchip.F32, bchip.F16])
def test_beam_search(ctx, kv_type):
    """Two searches of three beams over one pool: each step's picks against every continuation's score
    from the f64 layers over the beams' whole texts."""
    t = Texts(ctx, wide_model(2, False), kv_type, 80)
    searches, beams, vocab = 2, 3, t.cfg.vocab
    r = np.random.default_rng(2)
    live = [[t.start()] for _ in range(searches)]
    x = t.go([s[0] for s in live], [r.integers(0, vocab, n).tolist() for n in (30, 41)])
    x = np.stack([x[29], x[70]])
    sums = np.zeros((searches, 1), np.float32)
    bar = BARS[kv_type]
    for step in range(5):
        best, beam, token = t.g.beams(x, sums, beams)
        states = []
        for i in range(searches):
            z = t.ref.logits(np.stack([t.want(s)[-1] for s in live[i]]))
            lp = z - z.max(1, keepdims=True)
            lp = lp - np.log(np.exp(lp).sum(1, keepdims=True)) + sums[i].astype(np.float64)[:, None]
            off = bar * (1 + np.abs(z).max())
            want = np.sort(lp.reshape(-1))[::-1][:beams]
            assert np.abs(best[i] - want).max() <= off, (step, i)
            assert np.abs(lp[beam[i], token[i]] - want).max() <= 2 * off, (step, i)
        # Every pick goes on in a fork of its beam; the beams behind them end.
        old, live = live, [[t.fork(live[i][b]) for b in beam[i]] for i in range(searches)]
        for s in (s for group in old for s in group):
            t.drop(s)
        seqs = [s for group in live for s in group]
        x = t.go(seqs, [[int(w)] for row in token for w in row])
        sums = best
    t.free()


def test_beams_of_a_batch_in_pieces(ctx):
    """The scores of some searches at a time: the same picks."""
    cfg, layers, head, _ = wide_model(1, False)
    g = GpuLayers(ctx, cfg, layers, head)
    r = np.random.default_rng(3)
    for n, beams in ((7, 4), (5, 1), (1, 3)):
        x, sums = r.standard_normal((n * beams, cfg.n_embd)).astype(np.float32), r.standard_normal((n, beams)).astype(np.float32)
        want = g.beams(x, sums, 6)
        g.SCORE_BYTES = 2 * beams * cfg.vocab * 4
        for a, b in zip(want, g.beams(x, sums, 6)):
            np.testing.assert_array_equal(a, b)
        del g.SCORE_BYTES
    with pytest.raises(ValueError):
        g.beams(x, sums[:, :2], 6)
    g.free()


@pytest.mark.parametrize("kv_type", [bchip.F32, bchip.F16])
def test_captured_calls(ctx, kv_type):
    """A step's append, attention and page copy captured into a graph, from a context that has run nothing
    (lists whole) and from one that has, replayed with other tables, positions and data in the same
    buffers and with other calls in between: the eager calls' bits where the plan is the same."""
    nh, nkv, hd = 8, 2, 128
    rng = np.random.default_rng(4)
    lens, rows = [900, 40, 2500, 333], [1, 1, 6, 60]
    batches = [Batch(np.random.default_rng(s), rows, lens, nkv, hd, kv_type, spare=6) for s in range(3)]
    with bchip.Ctx(0) as c:
        b = batches[0]
        n = b.total
        q0 = [rng.standard_normal((n, nh, hd)).astype(np.float32) for _ in batches]
        kv = [rng.standard_normal((n, nkv, hd)).astype(np.float32) for _ in batches]
        positions = np.concatenate([np.arange(m - r, m) for r, m in zip(rows, lens)]).astype(np.uint32)
        inv, qb, kb, vb, pb = c.upload(O.inv_freq(hd, 1e4)), c.upload(q0[0]), c.upload(kv[0]), c.upload(kv[0]), c.upload(positions)
        kc, vc, table, out = c.upload(b.k), c.upload(b.v), c.upload(b.table), c.zeros(n * nh * hd * 4)
        both = [p for p in range(b.npages) if p not in b.table][:2]

        def step():
            c.rope_append_paged(qb, kb, vb, kc, vc, kv_type, inv, pb, b.starts, lens, table, b.stride, 16, b.npages, nh, nkv, hd, hd, False)
            c.attention_paged(qb, kc, vc, kv_type, out, b.starts, lens, table, b.stride, 16, b.npages, nh, nkv, hd, hd ** -0.5)

        def copy():
            c.copy_pages([kc, vc], kv_type, 16 * nkv * hd, b.npages, [int(b.table[0, 0]), int(b.table[2, 5])], both)

        def put(i):
            x = batches[i]
            for buf, a in ((qb, q0[i]), (kb, kv[i]), (vb, kv[i]), (kc, np.nan_to_num(x.k)), (vc, np.nan_to_num(x.v)), (table, x.table),
                           (out, np.zeros((n, nh, hd), np.float32))):
                c.upload(a, buf)

        def got():
            c.sync()
            return [c.read(out, n * nh * hd, np.uint32), c.read(qb, n * nh * hd, np.uint32), c.read(kc, b.k.size, np.uint16 if kv_type else np.uint32)]

        put(0)
        whole = captured(c, step)
        want = []
        for i in range(3):
            put(i)
            step()
            want.append(got())
        cut, second = captured(c, step), captured(c, step)
        big = Batch(np.random.default_rng(9), [1, 300], [9000, 2000], nkv, hd, kv_type)
        bk, bv, bt, bq = c.upload(np.nan_to_num(big.k)), c.upload(np.nan_to_num(big.v)), c.upload(big.table), c.zeros(301 * nh * hd * 4)
        for i in (1, 0, 2, 1):
            c.attention_paged(bq, bk, bv, kv_type, bq, big.starts, big.lens, bt, big.stride, 16, big.npages, nh, nkv, hd, 0.1)
            for stream, graph in (cut, second):
                put(i)
                hip("hipGraphLaunch", graph, stream)
                for a, w in zip(got(), want[i]):
                    np.testing.assert_array_equal(a, w)
            put(i)
            hip("hipGraphLaunch", whole[1], whole[0])
            a, w = got(), want[i]
            a0, w0 = a[0].view(np.float32), w[0].view(np.float32)
            assert np.abs(a0 - w0).max() <= 4e-6 * np.abs(w0).max()
            np.testing.assert_array_equal(a[1], w[1])
        put(0)
        pages = captured(c, copy)
        for i in (2, 0):
            put(i)
            hip("hipGraphLaunch", pages[1], pages[0])
            c.sync()
            after = c.read(kc, b.k.shape, b.k.dtype)
            np.testing.assert_array_equal(after[both], np.nan_to_num(batches[i].k)[[int(b.table[0, 0]), int(b.table[2, 5])]])
        for g in (whole, cut, second, pages):
            hip("hipGraphExecDestroy", g[1])


def test_a_captured_search(ctx):
    """A search's step captured once its size has run, replayed with other scores and after a larger call."""
    rng = np.random.default_rng(5)
    n, beams, vocab, k = 2, 4, 5000, 8
    with bchip.Ctx(0) as c:
        scores, sums = [rng.standard_normal((n * beams, vocab)).astype(np.float32) * 4 for _ in range(3)], rng.standard_normal((n, beams)).astype(np.float32)
        sb, mb, best, beam, token = c.upload(scores[0]), c.upload(sums), *(c.zeros(n * k * 4) for _ in range(3))
        call = lambda: c.beam_select(sb, mb, n, beams, vocab, k, best, beam, token)  # noqa: E731
        read = lambda: [c.read(x, (n, k), np.uint32) for x in (best, beam, token)]  # noqa: E731
        want = []
        for s in scores:
            c.upload(s, sb)
            call()
            want.append(read())
        stream, graph = captured(c, call)
        big, ids = c.zeros(400 * 60000 * 4), c.zeros(400 * 64 * 4)
        for i in (1, 2, 0, 1):
            c.beam_select(big, big, 100, 4, 60000, 64, ids, ids, ids)
            c.upload(scores[i], sb)
            hip("hipGraphLaunch", graph, stream)
            for a, w in zip(read(), want[i]):
                np.testing.assert_array_equal(a, w)
        hip("hipGraphExecDestroy", graph)
