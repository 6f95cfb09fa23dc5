"""A decode step of several conversations in one pool of 4-bit slots
(bchip_rope_append_attention_ragged): the two calls it stands for, bit for bit, in the output, q left
rotated and both caches; each sequence against its formula in 64 bits over what the pool then holds;
nothing else in the pool touched; and a step captured and replayed."""
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


class Pool:
    """Lists of the given lengths with gaps between them, and the inputs of one step."""

    def __init__(self, ctx, lens, nh, nkv, hd, rd, neox, seed):
        r = np.random.default_rng(seed)
        self.ctx, self.lens = ctx, np.asarray(lens, np.uint32)
        self.shape, self.rope = (nh, nkv, hd), (rd, neox)
        seqs, kvd = len(lens), nkv * hd
        self.offs = (np.concatenate([[0], np.cumsum(self.lens + r.integers(0, 4, seqs))])[:-1] + 1).astype(np.uint64)
        order = r.permutation(seqs)  # (lists lie in any order)
        self.lens, self.offs = self.lens[order], self.offs[order]
        self.n = int((self.offs + self.lens).max()) + 2
        self.was = [P.pack(*P.quantise(r.standard_normal((self.n, kvd)).astype(np.float32))) for _ in range(2)]
        self.q, self.k, self.v = (r.standard_normal((seqs, w * hd)).astype(np.float32) for w in (nh, nkv, nkv))
        self.ib, self.pb = ctx.upload(O.inv_freq(rd, 1e4)), ctx.upload(self.lens - 1)
        self.kb, self.vb = ctx.upload(self.k), ctx.upload(self.v)
        self.qb, self.ob = ctx.upload(self.q), ctx.zeros(self.q.nbytes)
        self.caches = [ctx.upload(w) for w in self.was]

    def reset(self):
        self.ctx.upload(self.q, self.qb)
        self.ctx.upload(np.zeros_like(self.q), self.ob)
        for b, w in zip(self.caches, self.was):
            self.ctx.upload(w, b)

    def step(self, ctx=None, two=False):
        ctx, (nh, nkv, hd), (rd, neox) = ctx or self.ctx, self.shape, self.rope
        a = (self.qb, self.kb, self.vb, *self.caches, bchip.Q4, self.ib, self.pb, self.lens, self.offs, nh, nkv, hd, rd, neox)
        if two:
            ctx.rope_append_ragged(*a)
            ctx.attention_ragged(self.qb, *self.caches, bchip.Q4, self.ob, self.lens, self.offs, nh, nkv, hd, hd ** -0.5)
        else:
            ctx.rope_append_attention_ragged(*a, hd ** -0.5, self.ob)

    def read(self):
        shape = (len(self.lens),) + (self.shape[0], self.shape[2])
        return [self.ctx.read(self.ob, shape), self.ctx.read(self.qb, shape)] + [self.ctx.read(b, w.size, np.uint8) for b, w in zip(self.caches, self.was)]

    def free(self):
        for b in (self.ib, self.pb, self.kb, self.vb, self.qb, self.ob, *self.caches):
            b.free()


def lengths(kind, seqs, seed=3):
    """brief: one launch takes them whole; cut: in chunks; mixed: one long list among brief ones."""
    r = np.random.default_rng(seed)
    if kind == "brief":
        return r.integers(1, 200, seqs)
    if kind == "cut":
        return r.integers(1500, 4000, seqs)
    return np.concatenate([[9000], r.integers(1, 60, seqs - 1)])


# Heads of one block to eight, groups of 1 to 16, pairs of both kinds, part of the head rotated.
SHAPES = [(28, 4, 128, 128, True), (14, 2, 64, 64, True), (32, 8, 128, 64, False), (12, 4, 96, 96, False), (4, 4, 32, 16, True),
          (16, 1, 256, 256, False), (7, 1, 160, 32, True)]


@pytest.mark.parametrize("nh,nkv,hd,rd,neox", SHAPES)
@pytest.mark.parametrize("seqs,kind", [(1, "brief"), (3, "brief"), (3, "cut"), (17, "mixed"), (70, "brief")])
def test_the_step_is_its_two_calls(ctx, nh, nkv, hd, rd, neox, seqs, kind):
    p = Pool(ctx, lengths(kind, seqs), nh, nkv, hd, rd, neox, seqs)
    p.step(two=True)
    want = p.read()
    p.reset()
    p.step()
    got = p.read()
    for name, a, b in zip(("out", "q", "K", "V"), got, want):
        np.testing.assert_array_equal(a, b, err_msg=name)
    out, q, kv = got[0], got[1], [P.unpack(b, p.n * nkv * hd).reshape(p.n, nkv, hd) for b in got[2:]]
    was = [P.unpack(b, p.n * nkv * hd).reshape(p.n, nkv, hd) for b in p.was]
    slots = (p.offs + p.lens - 1).astype(np.int64)
    others = np.setdiff1d(np.arange(p.n), slots)
    wants = []
    for i in range(seqs):
        k, v = (t[int(p.offs[i]):int(p.offs[i]) + int(p.lens[i])] for t in kv)
        want, mass, top = P.attention(q[i:i + 1], k, v, nkv, np.ones((1, len(k)), bool), hd ** -0.5)
        assert (np.abs(out[i:i + 1] - want) <= P.bound(mass, top, hd)).all(), f"sequence {i} of {p.lens[i]}"
        wants.append(want)
    # (As in test_attention_q4_gpu.py: what a lost low part would leave is ten times this.)
    assert np.linalg.norm(out - np.concatenate(wants)) <= 8e-6 * np.linalg.norm(out)
    for a, b in zip(kv, was):
        np.testing.assert_array_equal(a[others], b[others])
    np.testing.assert_array_equal(kv[1][slots], P.stored(p.v).reshape(seqs, nkv, hd))
    p.free()


@pytest.mark.parametrize("kind,seqs", [("cut", 130), ("mixed", 256)])
def test_more_sequences_than_a_launch_takes(ctx, kind, seqs):
    """Three and four launches of the append and of the attention over one workspace."""
    p = Pool(ctx, lengths(kind, seqs) if kind == "mixed" else lengths(kind, seqs) // 2, 4, 1, 64, 64, False, 5)
    p.step(two=True)
    want = p.read()
    p.reset()
    p.step()
    for name, a, b in zip(("out", "q", "K", "V"), p.read(), want):
        np.testing.assert_array_equal(a, b, err_msg=name)
    p.free()


@pytest.mark.parametrize("kind", ["brief", "cut"])
def test_a_captured_step(ctx, kind):
    """Replayed as it was captured, the pool and q put back in between: the eager step's bits where
    its scratch had been taken before, and within the formula's bound where it had not (lists run whole)."""
    from test_matmul_scratch_gpu import captured, hip
    for warm in (False, True):
        with bchip.Ctx(0) as c:
            p = Pool(c, lengths(kind, 9), 28, 4, 128, 128, True, 8)
            if warm:
                p.step()
                want = p.read()
                p.reset()
            s, ex = captured(c, p.step)
            for _ in range(3):
                p.reset()
                hip("hipGraphLaunch", ex, s)
                got = p.read()
                if not warm:
                    k, v = (P.unpack(b, p.n * 512).reshape(p.n, 4, 128) for b in got[2:])
                    for i, (o, n) in enumerate(zip(p.offs.astype(np.int64), p.lens)):
                        full, mass, top = P.attention(got[1][i:i + 1], k[o:o + n], v[o:o + n], 4, np.ones((1, n), bool), 128 ** -0.5)
                        assert (np.abs(got[0][i:i + 1] - full) <= P.bound(mass, top, 128)).all()
                    want = got
                for a, b in zip(got, want):
                    np.testing.assert_array_equal(a, b)
            hip("hipGraphExecDestroy", ex)
