"""A stage over a cache in 4 bits, as it is used: a prompt in pieces, one-token steps, a verify
pass, a tree and the accepted path kept, the cache grown on the way, and the tokens scored by
their log probabilities (GpuLayers over bchip.Q4, then GpuLayers.logprobs). The check runs the
same layers in f64 (tiny_model.RefModel), attending over the values the device's cache holds:
those are first held against the f64 layers' own K and V, a code step (and a saturated one at the
far end of the scale) apart at most."""
import numpy as np
import pytest

import bchip
import oracle as O
import q4_plain as P
from layers import GpuLayers
from test_matmul_scratch_gpu import captured, hip
from tiny_model import RefModel, embed, wide_model

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = bchip.Ctx(0)
    yield c
    c.close()


class StoredModel(RefModel):
    """RefModel attending over the rows that the device's cache holds."""

    def __init__(self, cfg, layers, head, ctx):
        super().__init__(cfg, layers, head)
        self.ctx = ctx

    def stored(self, buf, slots):
        """A cache buffer's rows, and the scale of each element's block."""
        kvd = self.cfg.n_head_kv * self.cfg.head_dim
        raw = self.ctx.read(buf, bchip.nbytes_of(bchip.Q4, slots * kvd), np.uint8)
        d = np.abs(np.ascontiguousarray(raw.reshape(-1, 144)[:, 128:]).view(np.float16).astype(np.float64)).reshape(-1)
        return P.unpack(raw, slots * kvd).reshape(slots, kvd), np.repeat(d, 32)[:slots * kvd].reshape(slots, kvd)

    def forward(self, x, pos, tree, dev):
        c, rows = self.cfg, len(x)
        hd, nh, nkv = c.head_dim, c.n_head, c.n_head_kv
        positions, visible, base = O.shape(rows, pos, tree)
        see = np.arange(pos + rows)[None] <= (pos + np.arange(rows))[:, None]
        if visible is not None:
            bits = (np.asarray(visible, np.uint64)[:, None] >> np.arange(pos + rows - base, dtype=np.uint64)) & np.uint64(1)
            see = np.concatenate([np.ones((rows, base), bool), bits.astype(bool)], 1)
        x = np.asarray(x, np.float64)
        for w, kb, vb in zip(self.layers, dev.k, dev.v):
            n = self._norm(x, w["attn_norm"])
            q, k, v = n @ w["wq"].T + w["bq"], n @ w["wk"].T, n @ w["wv"].T
            q, k = self._rope(q, nh, positions), self._rope(k, nkv, positions)
            held = []
            for own, buf in ((k, kb), (v, vb)):
                values, step = self.stored(buf, pos + rows)
                off = np.abs(values[pos:] - own)
                # Half a step by rounding, another where 8 saturates at 7, 8 x 2^-7 by the scale's rounding.
                assert (off <= 1.07 * step[pos:] + 1e-4 * np.abs(own).max()).all()
                held.append(values.reshape(-1, nkv, hd))
            att, _, _ = P.attention(q.reshape(rows, nh, hd), *held, nkv, see, hd ** -0.5)
            x = x + att.reshape(rows, -1) @ w["wo"].T
            n = self._norm(x, w["ffn_norm"])
            gate, up = n @ w["gate"].T, n @ w["up"].T
            x = x + (gate / (1.0 + np.exp(-gate)) * up) @ w["down"].T
        return x


@pytest.mark.parametrize("neox", [False, True])
def test_a_conversation_over_4_bits(ctx, neox):
    cfg, layers, head, embd = wide_model(2, neox)
    g, ref = GpuLayers(ctx, cfg, layers, head, bchip.Q4), StoredModel(cfg, layers, head, ctx)
    cache = g.new_cache()
    r = np.random.default_rng(1)

    def go(tokens, pos, tree=None):
        positions, visible, base = O.shape(len(tokens), pos, tree)
        x0 = embed(embd, tokens)
        x = g.forward(x0, pos, positions, None if visible is None else (base, visible), cache)
        want = ref.forward(x0, pos, tree, cache)
        err = np.abs(x - want).max()
        print(f"{len(tokens)} rows at {pos}: states off by {err:.2e} of {np.abs(want).max():.2f}")
        # f32 layers: as tiny_model's exact forward is held elsewhere, 1e-4 of the largest state.
        assert err <= 1e-4 * (1 + np.abs(want).max())
        nxt = r.integers(0, cfg.vocab, len(tokens))
        tok, ent, ids, tops = g.logprobs(x, len(tokens), nxt, top=7)
        z = ref.logits(want)
        lp = z - z.max(1, keepdims=True)
        lp -= np.log(np.exp(lp).sum(1, keepdims=True))
        bar = 1e-4 * (1 + np.abs(z).max())
        assert np.abs(tok - lp[np.arange(len(nxt)), nxt]).max() <= bar
        assert np.abs(ent + (np.exp(lp) * lp).sum(1)).max() <= bar * np.log(cfg.vocab)
        assert np.abs(tops + np.sort(-lp, 1)[:, :7]).max() <= bar
        scores = g.logits(x, len(tokens))
        np.testing.assert_array_equal(ids, np.argsort(-scores, 1, kind="stable")[:, :7])
        assert g.logprobs(x, len(tokens))[0] is None

    prompt = list(r.integers(0, cfg.vocab, 300))
    go(prompt[:37], 0)
    go(prompt[37:], 37)          # past the first 256 slots: the cache grows
    go([5], 300)
    go([6, 7, 8, 9], 301)        # a verify pass, the last two refused
    go([10], 303)
    go([20, 21, 22, 23, 24], 304, [O.ROOT, 0, 0, 1, O.ROOT])
    cache.keep(304, [0, 1, 3])
    go([11], 307)
    go([12, 13], 308)
    cache.free()
    g.free()


def test_a_captured_step(ctx):
    """The decode step and a verify pass captured: from a context without scratch (lists uncut),
    with scratch, and replayed after a larger call has moved the scratch on."""
    nh, nkv, hd, pos = 32, 8, 128, 4000
    kvd, r = nkv * hd, np.random.default_rng(3)
    for rows in (1, 6):
        q, k, v = (r.standard_normal((rows, n * hd)).astype(np.float32) for n in (nh, nkv, nkv))
        kbuf = P.pack(*P.quantise(r.standard_normal((pos + rows, kvd)).astype(np.float32)))
        vbuf = P.pack(*P.quantise(r.standard_normal((pos + rows, kvd)).astype(np.float32)))
        with bchip.Ctx(0) as c:
            qb, kb, vb, kc, vc, ob = (c.upload(a) for a in (q, k, v, kbuf, vbuf, q * 0))
            ib, pb = c.upload(O.inv_freq(hd, 1e4)), c.upload((pos + np.arange(rows)).astype(np.uint32))
            forms = [lambda: c.rope_append_attention_rows(qb, kb, vb, kc, vc, bchip.Q4, ib, pb, rows, nh, nkv, hd, hd, False, pos,
                                                          hd ** -0.5, ob)]
            if rows == 1:
                forms.append(lambda: c.rope_append_attention_noalloc(qb, kb, vb, kc, vc, bchip.Q4, ib, pb, nh, nkv, hd, hd, False, pos,
                                                                     hd ** -0.5, ob))

            def fresh():
                for b, a in ((qb, q), (kc, kbuf), (vc, vbuf), (ob, q * 0)):
                    c.upload(a, b)

            graphs = [captured(c, f) for f in forms]
            fresh()
            forms[0]()
            want = c.read(ob, q.shape)
            graphs += [captured(c, f) for f in forms]
            big = c.zeros(bchip.nbytes_of(bchip.Q4, 300000 * 256 // 8))
            bq = c.zeros(64 * 8 * 256 * 4)
            for _ in range(3):
                c.attention(bq, big, big, bchip.Q4, bq, None, False, 64, 8, 1, 256, 30000, 0.1)
                for i, (stream, graph) in enumerate(graphs):
                    fresh()
                    hip("hipGraphLaunch", graph, stream)
                    got = c.read(ob, q.shape)
                    assert np.abs(got - want).max() <= 4e-6 * np.abs(want).max(), i
                    if i >= len(forms):  # the same plan: the same bits
                        np.testing.assert_array_equal(got, want)
            for _, graph in graphs:
                hip("hipGraphExecDestroy", graph)
