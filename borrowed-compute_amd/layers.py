"""One pipeline stage's layers on the GPU: bc-infer's Layers::forward
(crates/bc-infer/src/gpu/mod.rs:428-495), its logits head (mod.rs:499-508, the product
of model.rs:361-370) and the sampler after it (sample.rs, engine.rs:341-350), or the log probabilities of
tokens in its place, issued as this library's entry points instead of a Cmd list.

Per layer, in the reference's order: RMSNorm, the q/k/v products, their biases, RoPE of q
and k with the append of k and v at slot `pos` (the four commands at mod.rs:464-475 as one
bchip_rope_append), attention over the cache (for a line pass, with the append as one
call: bchip_rope_append_attention or its multi-row form), the output product and the
residual add,
RMSNorm, gate and up products, SiLU-mul, the down product and the residual add. Weights
stay in their ggml blocks (bchip_matmul). The cache is a bchip.KvCache (Gpu::reserve's
growth, mod.rs:404-423); positions and the tree's visibility masks come from the caller's
Shape (model.rs:405-443), as in the reference.

GpuLayers.forward_paged takes the rows of several conversations at once instead, their caches pages
of one bchip.PagePool, and GpuLayers.beams picks the continuations of beam searches."""
from __future__ import annotations

import contextlib
import ctypes
import ctypes.util
import math
import operator
from dataclasses import dataclass

import numpy as np

import bchip


@dataclass
class Config:
    """model.rs:27-80 (the fields the layers read)."""
    n_embd: int
    n_layer: int
    n_head: int
    n_head_kv: int
    head_dim: int
    rope_dim: int
    rope_base: float = 10000.0
    rope_neox: bool = False
    eps: float = 1e-5
    vocab: int = 0
    context: int = 4096


_libm = None


def _powf(x: float, y: float) -> float:
    """The C library's single-precision pow, the one the reference's f32::powf calls
    (numpy's float32 power differs from it in the last bit for many of these arguments)."""
    global _libm
    if _libm is None:
        _libm = ctypes.CDLL(ctypes.util.find_library("m") or "libm.so.6")
        _libm.powf.argtypes = [ctypes.c_float, ctypes.c_float]
        _libm.powf.restype = ctypes.c_float
    return _libm.powf(x, y)


def inv_freq(cfg: Config, factors=None) -> np.ndarray:
    """model.rs:208-211: rope_base^(-2i / rope_dim) in f32 (the exponent rounded to f32
    first), over the optional per-pair factors (rope_freqs.weight)."""
    half = cfg.rope_dim // 2
    f = np.empty(half, np.float32)
    for i in range(half):
        e = np.float32(np.float32(-2.0) * np.float32(i)) / np.float32(cfg.rope_dim)
        f[i] = _powf(np.float32(cfg.rope_base), e)
    if factors is not None:
        f = (f / np.asarray(factors, np.float32)[:half]).astype(np.float32)
    return f


@dataclass
class Matrix:
    """A weight matrix as stored: `rows` rows of `cols` weights in ggml blocks of `type`."""
    type: int
    data: bytes
    rows: int
    cols: int


class GpuLayers:
    """The layers of one stage (and the head, on the last stage), resident on the device.

    `layers` holds per layer: attn_norm, ffn_norm (f32 vectors), wq, wk, wv, wo, gate, up,
    down (Matrix), and bq, bk, bv (f32 vectors or None). `head` is (output_norm, output)
    or None."""

    SCORE_BYTES = 256 << 20  # of scores that sample and logprobs hold at once

    def __init__(self, ctx: bchip.Ctx, cfg: Config, layers: list[dict], head=None, kv_type: int = bchip.F32):
        self.ctx, self.cfg, self.kv_type = ctx, cfg, kv_type
        up = lambda a: ctx.upload(np.ascontiguousarray(a, np.float32))
        self.layers = []
        for l in layers:
            d = {k: up(l[k]) for k in ("attn_norm", "ffn_norm")}
            for k in ("wq", "wk", "wv", "wo", "gate", "up", "down"):
                m: Matrix = l[k]
                d[k] = (ctx.upload(np.frombuffer(m.data, np.uint8)), m.type, m.rows, m.cols)
            for k in ("bq", "bk", "bv"):
                d[k] = up(l[k]) if l.get(k) is not None else None
            self.layers.append(d)
        self.head = None
        if head is not None:
            norm, out = head
            self.head = (up(norm), ctx.upload(np.frombuffer(out.data, np.uint8)), out.type, out.rows, out.cols)
        self.freq = up(inv_freq(cfg))
        self.ff = layers[0]["gate"].rows if layers else 0
        self.scratch_rows = 0
        self.scratch: dict[str, bchip.Buf] = {}

    def new_cache(self) -> bchip.KvCache:
        """Gpu::new_cache (mod.rs:398-400)."""
        return bchip.KvCache(self.ctx, len(self.layers), self.cfg.n_head_kv * self.cfg.head_dim, self.kv_type)

    def _scratch(self, rows: int) -> dict:
        """Working buffers of at least `rows` rows, kept between calls (mod.rs:444-449)."""
        if rows > self.scratch_rows:
            c = self.cfg
            qd, kvd = c.n_head * c.head_dim, c.n_head_kv * c.head_dim
            self._free_scratch()
            sizes = {"x": c.n_embd, "n": c.n_embd, "q": qd, "k": kvd, "v": kvd, "att": qd, "o": c.n_embd,
                     "gate": self.ff, "up": self.ff, "pos": 1, "mask": 2}
            try:
                for k, w in sizes.items():
                    self.scratch[k] = self.ctx.zeros(max(rows * w, 1) * 4)
            except BaseException:
                self._free_scratch()
                raise
            self.scratch_rows = rows
        return self.scratch

    def _free_scratch(self) -> None:
        for b in self.scratch.values():
            b.free()
        self.scratch, self.scratch_rows = {}, 0

    def _matmul(self, w, x, out, rows: int, nrows: int | None = None) -> None:
        buf, ty, wr, wc = w
        self.ctx.matmul(buf, ty, x, out, wr if nrows is None else nrows, wc, rows)

    def forward(self, x: np.ndarray, pos: int, positions, masks, cache: bchip.KvCache) -> np.ndarray:
        """mod.rs:428-495: `rows` hidden states at positions `positions` (slots pos..), with
        `masks` = (base, visible) for a tree; returns the updated states."""
        c, ctx = self.cfg, self.ctx
        rows = len(positions)
        cache.reserve(pos + rows, pos, c.context)
        hd, nh, nkv = c.head_dim, c.n_head, c.n_head_kv
        s = self._scratch(rows)
        mb, seen = None, pos
        if masks is not None:
            seen, visible = masks
            ctx.upload(bchip.masks_words(visible), s["mask"])
            mb = s["mask"]
        scale = 1.0 / math.sqrt(hd)

        def attend(kc, vc):
            if rows == 1 and masks is None:
                # A one-token line step: the five commands as one launch (same bits).
                ctx.rope_append_attention(s["q"], s["k"], s["v"], kc, vc, self.kv_type, self.freq, s["pos"], nh, nkv,
                                          hd, c.rope_dim, c.rope_neox, pos, scale, s["att"])
            elif masks is None:
                # A line pass of several rows: one call (one launch where the library can, else
                # its two calls; the same bits either way).
                ctx.rope_append_attention_rows(s["q"], s["k"], s["v"], kc, vc, self.kv_type, self.freq, s["pos"], rows,
                                               nh, nkv, hd, c.rope_dim, c.rope_neox, pos, scale, s["att"])
            else:
                ctx.rope_append(s["q"], s["k"], s["v"], kc, vc, self.kv_type, self.freq, s["pos"], rows, nh, nkv, hd,
                                c.rope_dim, c.rope_neox, pos)
                ctx.attention(s["q"], kc, vc, self.kv_type, s["att"], mb, masks is not None, rows, nh, nkv, hd, seen,
                              scale)

        return self._layers(x, positions, cache, attend)

    def new_pool(self, npages: int, page_slots: int = 16) -> bchip.PagePool:
        """A pool of pages for this stage's caches (kv_type F32 or F16)."""
        return bchip.PagePool(self.ctx, len(self.layers), self.cfg.n_head_kv * self.cfg.head_dim, npages, page_slots, self.kv_type)

    def forward_paged(self, x: np.ndarray, seqs, rows, pool: bchip.PagePool) -> np.ndarray:
        """The layers over new rows of several conversations in one pass: rows[i] hidden states of
        conversation seqs[i] (a piece of a prompt, a token, none), in that order, appended to its pages
        at its next slots; returns the updated states. Pages that a conversation lacks or shares are
        taken first (PagePool.extend). At most 256 conversations a pass. A pass that raises leaves every
        conversation the slots it had (its own copy of a page that it shared may stay)."""
        c, ctx, rows = self.cfg, self.ctx, [operator.index(n) for n in rows]
        if len(x) != sum(rows):
            raise ValueError(f"{len(x)} states for {sum(rows)} rows")
        if len(seqs) > 256:
            raise ValueError(f"{len(seqs)} conversations (at most 256 a pass)")
        if (pool.ctx, pool.n_layer, pool.kvd, pool.kv_type) != (ctx, len(self.layers), c.n_head_kv * c.head_dim, self.kv_type):
            raise ValueError("the pool is another stage's")
        s = self._scratch(max(len(x), 1))
        pool.extend(seqs, rows)
        try:
            lens = [pool.len[s] for s in seqs]
            positions = np.concatenate([np.arange(m - n, m) for n, m in zip(rows, lens)]) if len(x) else np.zeros(0)
            starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.uint32)
            table, stride = pool.table(seqs)
            hd, nh, nkv = c.head_dim, c.n_head, c.n_head_kv
            batch = (starts, np.asarray(lens, np.uint32), table, stride, pool.page_slots, pool.npages, nh, nkv, hd)

            def attend(kc, vc):
                ctx.rope_append_paged(s["q"], s["k"], s["v"], kc, vc, pool.kv_type, self.freq, s["pos"], *batch, c.rope_dim, c.rope_neox)
                ctx.attention_paged(s["q"], kc, vc, pool.kv_type, s["att"], *batch, 1.0 / math.sqrt(hd))

            return self._layers(x, positions, pool, attend)
        except BaseException:
            for q, n in reversed(list(zip(seqs, rows))):
                pool.truncate(q, pool.len[q] - n)
            raise

    def _layers(self, x: np.ndarray, positions, cache, attend) -> np.ndarray:
        """Every layer over the states x at `positions`; attend(kc, vc) turns the layer's q, k and v
        rows, appends, and leaves the attention's output in the scratch."""
        c, ctx = self.cfg, self.ctx
        rows, e = len(positions), c.n_embd
        qd, kvd = c.n_head * c.head_dim, c.n_head_kv * c.head_dim
        if rows == 0:
            return np.zeros((0, e), np.float32)
        s = self._scratch(rows)
        ctx.upload(np.ascontiguousarray(x, np.float32), s["x"])
        ctx.upload(np.ascontiguousarray(positions, np.uint32), s["pos"])
        for l, kc, vc in zip(self.layers, cache.k, cache.v):
            ctx.rms_norm(s["x"], l["attn_norm"], s["n"], rows, e, c.eps)
            self._matmul(l["wq"], s["n"], s["q"], rows)
            self._matmul(l["wk"], s["n"], s["k"], rows)
            self._matmul(l["wv"], s["n"], s["v"], rows)
            for bias, out, dim in ((l["bq"], s["q"], qd), (l["bk"], s["k"], kvd), (l["bv"], s["v"], kvd)):
                if bias is not None:
                    ctx.bias_add(out, bias, rows * dim, dim)
            attend(kc, vc)
            self._matmul(l["wo"], s["att"], s["o"], rows)
            ctx.add(s["x"], s["o"], rows * e)
            ctx.rms_norm(s["x"], l["ffn_norm"], s["n"], rows, e, c.eps)
            self._matmul(l["gate"], s["n"], s["gate"], rows)
            self._matmul(l["up"], s["n"], s["up"], rows)
            ctx.silu_mul(s["gate"], s["up"], rows * self.ff)
            self._matmul(l["down"], s["gate"], s["o"], rows)
            ctx.add(s["x"], s["o"], rows * e)
        return ctx.read(s["x"], (rows, e))

    def logits(self, x: np.ndarray, rows: int, upto: int | None = None) -> np.ndarray:
        """Next-token scores of each row for the first `upto` tokens (mod.rs:499-508):
        RMSNorm with output_norm, then the product against the first `upto` rows of the
        output matrix (Gpu::matmul_rows)."""
        if self.head is None:
            raise ValueError("this stage has no output head")
        norm, out, ty, vr, vc = self.head
        upto = vr if upto is None else min(upto, vr)
        s = self._scratch(rows)
        ctx = self.ctx
        ctx.upload(np.ascontiguousarray(x, np.float32), s["x"])
        ctx.rms_norm(s["x"], norm, s["n"], rows, self.cfg.n_embd, self.cfg.eps)
        scores = ctx.zeros(rows * upto * 4)
        ctx.matmul(out, ty, s["n"], scores, upto, vc, rows)
        got = ctx.read(scores, (rows, upto))
        scores.free()
        return got

    @contextlib.contextmanager
    def _score_rows(self, x: np.ndarray, rows: int, upto: int, *words: int):
        """The logits head of `rows` rows in pieces whose scores take at most SCORE_BYTES (and two rows:
        a row passed alone may differ in its last bits from the same row in a batch, whose size does not
        matter). Gives result buffers of `words` u32s each, and an iterator that computes a piece's scores
        and yields (first row, rows, scores). Every buffer is freed at the end."""
        norm, out, ty, _, vc = self.head
        s, ctx, bufs = self._scratch(rows), self.ctx, []
        ctx.upload(np.ascontiguousarray(x, np.float32), s["x"])
        ctx.rms_norm(s["x"], norm, s["n"], rows, self.cfg.n_embd, self.cfg.eps)
        count = max(1, min(-(-rows * upto * 4 // self.SCORE_BYTES), rows // 2))
        ends = [rows * i // count for i in range(count + 1)]

        def pieces():
            for r, end in zip(ends, ends[1:]):
                ctx.matmul(out, ty, s["n"].offset(r * vc * 4), bufs[-1], upto, vc, end - r)
                yield r, end - r, bufs[-1]
        try:
            for n in (*words, max(b - a for a, b in zip(ends, ends[1:])) * upto):
                bufs.append(ctx.zeros(4 * n))
            yield bufs[:-1], pieces()
        finally:
            for b in bufs:
                b.free()

    def sample(self, x: np.ndarray, rows: int, temperature: float, top_p: float, seed: int, step0: int,
               upto: int | None = None) -> np.ndarray:
        """The last stage's next tokens (engine.rs:341-350): the logits head, then sample.rs's
        pick for each row on the device (bchip_sample; row r at step step0 + r). Only the ids
        come back to the host, not the rows x vocab scores."""
        if self.head is None:
            raise ValueError("this stage has no output head")
        vr = self.head[3]
        upto = vr if upto is None else min(upto, vr)
        with self._score_rows(x, rows, upto, rows) as ((ids,), pieces):
            for r, n, scores in pieces:
                self.ctx.sample(scores, n, upto, temperature, top_p, seed, step0 + r, ids.offset(4 * r))
            return self.ctx.read(ids, (rows,), np.uint32)

    def logprobs(self, x: np.ndarray, rows: int, tokens=None, top: int = 0, temperature: float = 1.0, upto: int | None = None):
        """What the scores of each row say of tokens, on the device (bchip_logprobs): the logits head,
        then the log probability of tokens[r] (None without tokens), the entropy, and the `top` most
        likely tokens with their log probabilities. Only these come back to the host; rows are scored in
        pieces (SCORE_BYTES), with the same results."""
        if self.head is None:
            raise ValueError("this stage has no output head")
        if tokens is not None and len(tokens) != rows:
            raise ValueError(f"{len(tokens)} tokens for {rows} rows")
        vr = self.head[3]
        upto = vr if upto is None else min(upto, vr)
        given = () if tokens is None else (rows,)
        with self._score_rows(x, rows, upto, rows * (2 + top), rows * top, *given) as ((vals, ids, *tk), pieces):
            for b in tk:
                self.ctx.upload(np.ascontiguousarray(tokens, np.uint32), b)
            for r, n, scores in pieces:
                given = (tk[0].offset(4 * r), vals.offset(4 * r)) if tk else (None, None)
                self.ctx.logprobs(scores, n, upto, temperature, *given, vals.offset(4 * (rows + r)), top,
                                  ids.offset(4 * r * top), vals.offset(4 * (2 * rows + r * top)))
            got = self.ctx.read(vals, rows * (2 + top))
            best = self.ctx.read(ids, (rows, top), np.uint32)
        return (None if tokens is None else got[:rows]), got[rows:2 * rows], best, got[2 * rows:].reshape(rows, top)

    def beams(self, x: np.ndarray, sums, k: int, upto: int | None = None):
        """A step of beam search on the device: the logits head of x (a row for every beam, `sums`
        [searches][beams] of them, the log probabilities of the beams so far, -inf for one that is not
        there), then the k best continuations of each search (bchip_beam_select). Gives their scores, beams
        and tokens [searches][k]; only these come back to the host. Searches are scored in pieces of at
        most SCORE_BYTES (one search at least) and the rows that a selection takes, with the same results."""
        if self.head is None:
            raise ValueError("this stage has no output head")
        sums = np.ascontiguousarray(sums, np.float32)
        n, beams = sums.shape
        if len(x) != n * beams:
            raise ValueError(f"{len(x)} states for {n} searches of {beams} beams")
        norm, out, ty, vr, vc = self.head
        upto = vr if upto is None else min(upto, vr)
        if n == 0:
            return np.zeros((0, k), np.float32), np.zeros((0, k), np.uint32), np.zeros((0, k), np.uint32)
        s, ctx, bufs = self._scratch(len(x)), self.ctx, []
        ctx.upload(np.ascontiguousarray(x, np.float32), s["x"])
        ctx.rms_norm(s["x"], norm, s["n"], len(x), self.cfg.n_embd, self.cfg.eps)
        count = max(1, min(-(-len(x) * upto * 4 // self.SCORE_BYTES), n // 2 if beams == 1 else n))
        count = max(count, -(-n // max(1, 65535 // max(1, beams))))
        ends = [n * i // count for i in range(count + 1)]
        try:
            for words in (n * beams, n * k, n * k, n * k, max(b - a for a, b in zip(ends, ends[1:])) * beams * upto):
                bufs.append(ctx.zeros(4 * words))
            sb, best, beam, token, scores = bufs
            ctx.upload(sums, sb)
            for a, b in zip(ends, ends[1:]):
                ctx.matmul(out, ty, s["n"].offset(a * beams * vc * 4), scores, upto, vc, (b - a) * beams)
                at = [y.offset(4 * a * k) for y in (best, beam, token)]
                ctx.beam_select(scores, sb.offset(4 * a * beams), b - a, beams, upto, k, *at)
            return ctx.read(best, (n, k)), ctx.read(beam, (n, k), np.uint32), ctx.read(token, (n, k), np.uint32)
        finally:
            for y in bufs:
                y.free()

    def free(self) -> None:
        for l in self.layers:
            for k, v in l.items():
                if isinstance(v, bchip.Buf):
                    v.free()
                elif isinstance(v, tuple):
                    v[0].free()
        if self.head is not None:
            self.head[0].free()
            self.head[1].free()
        self.freq.free()
        self._free_scratch()
