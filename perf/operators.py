"""What is measured of the operators around a KV cache in 4 bits, and of the log
probabilities after the logits head.

A case's `kind` says which call a pass makes:
  append    one layer's rotation and append of new rows into a cache in 4 bits
            (bchip_rope_append), and the new rows read back out of it (bchip_copy).
  attend    attention over the 4-bit caches of `layers` layers (bchip_attention): one row is
            a decode step, a few a speculative verify pass, many a prompt or a piece of one;
            "tree" gives each row a mask of the rows above it.
  ragged    one decode step's attention of several conversations in one pool, `layers` layers
            (bchip_attention_ragged).
  logprobs  the log probability of a given token in each row of scores, the row's entropy and
            its most likely tokens (bchip_logprobs).

A cache in 4 bits is an array of units of 256 elements, 144 bytes each: 128 bytes of codes, the
even element of a pair in the low four bits, then the f16 scales of the unit's eight blocks of 32
elements. An element is (code - 8) x its block's scale."""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

# (query heads, KV heads, head dim, neox pairs, rope base).
SHAPES = {"qwen05b": (14, 2, 64, True, 1e6), "llama8b": (32, 8, 128, False, 5e5), "qwen7b": (28, 4, 128, True, 1e6),
          "llama70b": (64, 8, 128, False, 5e5), "hd96": (12, 4, 96, True, 1e4), "hd256": (16, 4, 256, False, 1e4)}

_lib = {}


def _ctx():
    """The program's one context of the library, made once."""
    if not _lib:
        sys.path.insert(1, os.path.join(os.getcwd(), "borrowed-compute_amd"))
        import bchip
        _lib["bchip"], _lib["ctx"] = bchip, bchip.Ctx(0)
    return _lib["bchip"], _lib["ctx"]


def listed():
    return [
        # The token of a decode step of a small model: latency.
        {"name": "append_qwen05b_1", "kind": "append", "shape": "qwen05b", "rows": 1, "pos": 510},
        # A piece of a prompt after some history.
        {"name": "append_llama8b_512", "kind": "append", "shape": "llama8b", "rows": 512, "pos": 301},
        # A decode step early in a conversation with a small model, head dim 64.
        {"name": "attend_qwen05b_1_511", "kind": "attend", "shape": "qwen05b", "rows": 1, "pos": 511, "tree": False, "layers": 6},
        # A decode step at a long context.
        {"name": "attend_llama8b_1_32768", "kind": "attend", "shape": "llama8b", "rows": 1, "pos": 32767, "tree": False, "layers": 4},
        # Eight draft tokens verified.
        {"name": "attend_llama70b_8_5003", "kind": "attend", "shape": "llama70b", "rows": 8, "pos": 5003, "tree": False, "layers": 4},
        # A tree of draft tokens.
        {"name": "attend_llama70b_tree33", "kind": "attend", "shape": "llama70b", "rows": 33, "pos": 3001, "tree": True, "layers": 2},
        # A long prompt at once.
        {"name": "attend_llama8b_4096", "kind": "attend", "shape": "llama8b", "rows": 4096, "pos": 0, "tree": False, "layers": 1},
        # A piece of a prompt after some history, odd sizes, head dim 64.
        {"name": "attend_qwen05b_777", "kind": "attend", "shape": "qwen05b", "rows": 777, "pos": 300, "tree": False, "layers": 1},
        # Sixteen conversations of ragged lengths, one step.
        {"name": "ragged_qwen7b_16", "kind": "ragged", "shape": "qwen7b", "seqs": 16, "longest": 24000, "layers": 2},
        # The next token's log probability and five alternatives, the largest vocabulary.
        {"name": "logprobs_151936_1", "kind": "logprobs", "rows": 1, "vocab": 151936, "top": 5, "temperature": 1.0},
        # A batch of conversations, twenty alternatives each, an odd row count.
        {"name": "logprobs_32000_37", "kind": "logprobs", "rows": 37, "vocab": 32000, "top": 20, "temperature": 0.7},
        # A prompt's tokens scored.
        {"name": "logprobs_128256_256", "kind": "logprobs", "rows": 256, "vocab": 128256, "top": 0, "temperature": 1.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "attend", "ragged", "logprobs", "logprobs"])
    if kind == "append":
        return {"kind": kind, "shape": rng.choice(list(SHAPES)), "rows": rng.choice([1, _log(rng, 2, 512)]), "pos": _log(rng, 1, 6000)}
    if kind == "attend":
        shape = rng.choice(list(SHAPES))
        form = rng.choice(["step", "step", "verify", "tree", "prompt", "prompt"])
        if form == "step":
            return {"kind": kind, "shape": shape, "rows": 1, "pos": _log(rng, 2, 32768) - 1, "tree": False, "layers": rng.randint(1, 4)}
        if form == "prompt":
            return {"kind": kind, "shape": shape, "rows": _log(rng, 17, 2000), "pos": rng.choice([0, _log(rng, 1, 1500)]),
                    "tree": False, "layers": 1}
        return {"kind": kind, "shape": shape, "rows": rng.randint(2, 16) if form == "verify" else rng.randint(2, 64),
                "pos": _log(rng, 1, 6100), "tree": form == "tree", "layers": rng.randint(1, 3)}
    if kind == "ragged":
        return {"kind": kind, "shape": rng.choice(list(SHAPES)), "seqs": rng.randint(2, 24), "longest": _log(rng, 20, 12000),
                "layers": rng.randint(1, 2)}
    return {"kind": kind, "rows": rng.choice([1, _log(rng, 2, 200)]), "vocab": rng.choice([32000, 128256, 151936, _log(rng, 100, 150000)]),
            "top": rng.choice([0, 1, 5, 20, 64]), "temperature": rng.choice([1.0, 1.0, 0.3, 0.7, 1.3])}


# ---- inputs, made from the seed alone -----------------------------------------------------


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + 29)
    return g


def _randn(g, *shape, scale=1.0):
    return torch.empty(*shape, device="cuda").normal_(0.0, scale, generator=g)


def _freq(hd, base):
    i = np.arange(hd // 2, dtype=np.float64)
    return torch.from_numpy((base ** (-2.0 * i / hd)).astype(np.float32)).cuda()


def _cache(g, layers, slots, kvd):
    """`layers` caches of `slots` rows of N(0, 1) values in 4 bits: [layers, units, 144] bytes."""
    units = -(-slots * kvd // 256)
    out = torch.empty(layers, units, 144, device="cuda", dtype=torch.uint8)
    for l in range(layers):
        out[l] = _pack(*_quantise(_randn(g, units * 256)))
    return out


def _seen(rows, seed):
    """A random tree's masks: each node's parent is the root or an earlier node, and a row sees
    its ancestors and itself."""
    r = np.random.default_rng(int(seed) + 3)
    seen = []
    for i in range(rows):
        parent = int(r.integers(-1, i)) if i else -1
        seen.append((0 if parent < 0 else seen[parent]) | (1 << i))
    return seen


def _lens(case, seed):
    r = np.random.default_rng(int(seed) + 5)
    n = np.exp(r.uniform(math.log(max(1, case["longest"] // 8)), math.log(case["longest"]), case["seqs"])).astype(np.uint32)
    n = np.maximum(n, 1)
    n[0] = case["longest"]
    return n


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    if kind == "logprobs":
        # Most of a vocabulary is unlikely; a few dozen tokens hold most of the mass.
        rows, vocab, top = case["rows"], case["vocab"], case["top"]
        scores = _randn(g, rows, vocab, scale=2.0)
        at = torch.randint(0, vocab, (rows, 32), device="cuda", generator=g)
        scores.scatter_add_(1, at, 4.0 + 8.0 * torch.rand(rows, 32, device="cuda", generator=g))
        s = {"scores": scores, "tokens": at[:, 0].to(torch.int32), "logprob": torch.empty(rows, device="cuda"),
             "entropy": torch.empty(rows, device="cuda"), "ids": torch.empty(rows, top, device="cuda", dtype=torch.int32),
             "top": torch.empty(rows, top, device="cuda")}
    else:
        nh, nkv, hd, neox, base = SHAPES[case["shape"]]
        s = {"nh": nh, "nkv": nkv, "hd": hd, "neox": neox}
        if kind == "append":
            rows, pos = case["rows"], case["pos"]
            units = -(-(pos + rows) * nkv * hd // 256)
            s |= {"q0": _randn(g, rows, nh, hd, scale=2.0), "k": _randn(g, rows, nkv, hd), "v": _randn(g, rows, nkv, hd),
                  "kc": torch.zeros(units, 144, device="cuda", dtype=torch.uint8), "vc": torch.zeros(units, 144, device="cuda", dtype=torch.uint8),
                  "freq": _freq(hd, base), "positions": torch.arange(pos, pos + rows, device="cuda", dtype=torch.int32),
                  "k16": torch.empty(units * 256, device="cuda", dtype=torch.float16), "v16": torch.empty(units * 256, device="cuda", dtype=torch.float16)}
            s["q"] = torch.empty_like(s["q0"])
        elif kind == "attend":
            rows, pos, L = case["rows"], case["pos"], case["layers"]
            # Queries are larger than keys in earnest: the softmax has its peaks.
            s |= {"q": _randn(g, L, rows, nh, hd, scale=2.0), "kc": _cache(g, L, pos + rows, nkv * hd), "vc": _cache(g, L, pos + rows, nkv * hd),
                  "out": torch.empty(L, rows, nh, hd, device="cuda")}
            if case["tree"]:
                words = np.array(_seen(rows, seed), np.uint64).view(np.uint32).reshape(rows, 2)
                s["masks"] = torch.from_numpy(words.astype(np.int64)).to(torch.int32).cuda()
        else:
            n, L = case["seqs"], case["layers"]
            lens = _lens(case, seed)
            total = int(lens.sum())
            s |= {"q": _randn(g, L, n, nh, hd, scale=2.0), "kc": _cache(g, L, total, nkv * hd), "vc": _cache(g, L, total, nkv * hd),
                  "lens": lens, "offs": np.concatenate([[0], np.cumsum(lens.astype(np.uint64))])[:-1].astype(np.uint64),
                  "out": torch.empty(L, n, nh, hd, device="cuda")}
    torch.cuda.synchronize()  # the library's stream does not wait for torch's
    s["case"] = case
    return s


# ---- one pass -----------------------------------------------------------------------------


def run(s):
    return (_OWN if own else _PLAIN)[s["case"]["kind"]](s, s["case"])


def _own_append(s, case):
    bchip, c = _ctx()
    rows, pos, kvd = case["rows"], case["pos"], s["nkv"] * s["hd"]
    p = {k: s[k].data_ptr() for k in ("q0", "q", "k", "v", "kc", "vc", "freq", "positions", "k16", "v16")}
    c.copy(p["q0"], bchip.F32, p["q"], bchip.F32, 0, s["q0"].numel())  # the q product's place: it is rotated there
    c.rope_append(p["q"], p["k"], p["v"], p["kc"], p["vc"], bchip.Q4, p["freq"], p["positions"], rows, s["nh"], s["nkv"], s["hd"],
                  s["hd"], s["neox"], pos)
    # A call reads from a whole unit: up to seven blocks before the first new row come along.
    unit = pos * kvd // 256
    n, at = (pos + rows) * kvd - unit * 256, pos * kvd - unit * 256
    c.copy(p["kc"] + unit * 144, bchip.Q4, p["k16"], bchip.F16, 0, n)
    c.copy(p["vc"] + unit * 144, bchip.Q4, p["v16"], bchip.F16, 0, n)
    return {"q": s["q"], "k": s["k16"][at:n].view(rows, -1), "v": s["v16"][at:n].view(rows, -1)}


def _own_attend(s, case):
    bchip, c = _ctx()
    rows, tree = case["rows"], case["tree"]
    a = [s[k] for k in ("q", "kc", "vc", "out")]
    at, by = [t.data_ptr() for t in a], [t.stride(0) * t.element_size() for t in a]
    masks = s["masks"].data_ptr() if tree else None
    for l in range(case["layers"]):
        q, kc, vc, out = [x + l * y for x, y in zip(at, by)]
        c.attention(q, kc, vc, bchip.Q4, out, masks, tree, rows, s["nh"], s["nkv"], s["hd"], case["pos"], 1.0 / math.sqrt(s["hd"]))
    return {"out": s["out"]}


def _own_ragged(s, case):
    bchip, c = _ctx()
    a = [s[k] for k in ("q", "kc", "vc", "out")]
    at, by = [t.data_ptr() for t in a], [t.stride(0) * t.element_size() for t in a]
    for l in range(case["layers"]):
        q, kc, vc, out = [x + l * y for x, y in zip(at, by)]
        c.attention_ragged(q, kc, vc, bchip.Q4, out, s["lens"], s["offs"], s["nh"], s["nkv"], s["hd"], 1.0 / math.sqrt(s["hd"]))
    return {"out": s["out"]}


def _own_logprobs(s, case):
    _, c = _ctx()
    top = case["top"]
    c.logprobs(s["scores"].data_ptr(), case["rows"], case["vocab"], case["temperature"], s["tokens"].data_ptr(), s["logprob"].data_ptr(),
               s["entropy"].data_ptr(), top, s["ids"].data_ptr() if top else None, s["top"].data_ptr() if top else None)
    return {"logprob": s["logprob"], "entropy": s["entropy"], "ids": s["ids"], "top": s["top"]}


# The plain forms.


def _quantise(x):
    """Codes (0 .. 15) and scales of x's last dimension in blocks of 32: the value of the largest
    magnitude (the positive one of two) goes to code 0, its scale rounded to 7 significant bits
    within 2^-14 .. 896."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    hi, lo = b.amax(-1), b.amin(-1)
    d = torch.where(hi >= -lo, hi, lo) / -8.0
    u = d.contiguous().view(torch.int32)
    d = ((u + 0xFFFF + ((u >> 17) & 1)) & ~0x1FFFF).view(torch.float32)
    d = torch.where(torch.signbit(d), -1.0, 1.0) * d.abs().clamp(2.0 ** -14, 896.0)
    codes = torch.round(b * (1.0 / d)[..., None]).clamp(-8.0, 7.0) + 8.0
    return codes.to(torch.uint8).reshape(x.shape), d


def _pack(codes, d):
    c = codes.view(-1, 128, 2)
    return torch.cat([c[..., 0] | (c[..., 1] << 4), d.half().view(torch.uint8).view(-1, 16)], 1)


def _unpack(units):
    """[..., units, 144] bytes -> [..., 256 units] values, f32."""
    q = units[..., :128]
    n = torch.stack([q & 15, q >> 4], -1).reshape(*units.shape[:-1], 8, 32).float() - 8.0
    return (n * units[..., 128:].contiguous().view(torch.float16).float()[..., None]).reshape(*units.shape[:-2], -1)


def _rotate(x, positions, freq, neox):
    """x [rows, heads, hd] turned by the f32 angle the operator is defined by."""
    theta = positions.float()[:, None] * freq[None]
    cos, sin, half = theta.cos()[:, None], theta.sin()[:, None], freq.numel()
    a, b = (slice(0, half), slice(half, 2 * half)) if neox else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
    out, u, v = torch.empty_like(x), x[..., a], x[..., b]
    out[..., a], out[..., b] = u * cos - v * sin, u * sin + v * cos
    return out


def _plain_append(s, case):
    rows, out = case["rows"], {"q": _rotate(s["q0"], s["positions"], s["freq"], s["neox"])}
    k = _rotate(s["k"], s["positions"], s["freq"], s["neox"])
    for name, x in (("k", k), ("v", s["v"])):
        codes, d = _quantise(x.reshape(rows, -1))
        out[name] = ((codes.float() - 8.0).view(rows, -1, 32) * d[..., None]).half().view(rows, -1)
    return out


def _softmax(x, seen):
    x = torch.where(seen, x, -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    return p / p.sum(-1, keepdim=True)


def _plain_attend(s, case):
    rows, pos, L, nh, nkv, hd = case["rows"], case["pos"], case["layers"], s["nh"], s["nkv"], s["hd"]
    slots, G = pos + rows, nh // nkv
    k, v = (_unpack(s[n])[:, :slots * nkv * hd].view(L, slots, nkv, hd).transpose(1, 2).contiguous() for n in ("kc", "vc"))
    q = s["q"].view(L, rows, nkv, G, hd).permute(0, 2, 3, 1, 4).reshape(L, nkv, G * rows, hd)
    j = torch.arange(slots, device="cuda")
    if case["tree"]:
        m = s["masks"].long() & 0xFFFFFFFF
        bits = torch.cat([(m[:, :1] >> torch.arange(32, device="cuda")) & 1, (m[:, 1:] >> torch.arange(32, device="cuda")) & 1], 1)
        seen = torch.cat([torch.ones(rows, pos, device="cuda", dtype=torch.bool), bits[:, :rows].bool()], 1)
    else:
        seen = j[None] <= (pos + torch.arange(rows, device="cuda"))[:, None]
    x = (q / math.sqrt(hd)) @ k.transpose(2, 3).contiguous()
    p = _softmax(x.view(L, nkv, G, rows, slots), seen).view(L, nkv, G * rows, slots)
    return {"out": (p @ v).view(L, nkv, G, rows, hd).permute(0, 3, 1, 2, 4).reshape(L, rows, nh, hd)}


def _plain_ragged(s, case):
    n, L, nh, nkv, hd = case["seqs"], case["layers"], s["nh"], s["nkv"], s["hd"]
    lens, offs = torch.from_numpy(s["lens"].astype(np.int64)).cuda(), torch.from_numpy(s["offs"].astype(np.int64)).cuda()
    j = torch.arange(case["longest"], device="cuda")
    seen = j[None] < lens[:, None]
    at = offs[:, None] + torch.minimum(j[None], lens[:, None] - 1)
    total, G = int(s["lens"].sum()), nh // nkv
    k, v = (_unpack(s[m])[:, :total * nkv * hd].view(L, total, nkv, hd)[:, at].transpose(2, 3).contiguous() for m in ("kc", "vc"))
    q = s["q"].view(L, n, nkv, G, hd)
    x = (q / math.sqrt(hd)) @ k.transpose(3, 4).contiguous()
    return {"out": (_softmax(x, seen[:, None, None]) @ v).reshape(L, n, nh, hd)}


def _plain_logprobs(s, case):
    top, scores = case["top"], s["scores"]
    x = (scores - scores.amax(1, keepdim=True)) / case["temperature"]
    e = torch.exp(x)
    total = e.sum(1)
    lse = torch.log(total)
    # Descending scores, ties to the lowest index: one integer key orders both.
    b = (scores + 0.0).view(torch.int32)
    key = ((b ^ ((b >> 31) & 0x7FFFFFFF)).long() << 32) | (0xFFFFFFFF - torch.arange(case["vocab"], device="cuda"))
    ids = 0xFFFFFFFF - (torch.topk(key, top, 1)[0] & 0xFFFFFFFF)
    return {"logprob": x.gather(1, s["tokens"].long()[:, None])[:, 0] - lse, "entropy": lse - (e * x).sum(1) / total,
            "ids": ids.to(torch.int32), "top": x.gather(1, ids) - lse[:, None]}


_OWN = {"append": _own_append, "attend": _own_attend, "ragged": _own_ragged, "logprobs": _own_logprobs}
_PLAIN = {"append": _plain_append, "attend": _plain_attend, "ragged": _plain_ragged, "logprobs": _plain_logprobs}


# ---- what a pass cannot do without --------------------------------------------------------


def work(case):
    kind, q4 = case["kind"], 9.0 / 16.0  # bytes an element of a cache
    if kind == "logprobs":
        return {"bytes": 4.0 * case["rows"] * (case["vocab"] + 3 + 2 * case["top"]), "flops": 5.0 * case["rows"] * case["vocab"]}
    nh, nkv, hd, _, _ = SHAPES[case["shape"]]
    kvd = nkv * hd
    if kind == "append":
        # q read and left rotated, k and v read, their codes written and read back, the f16 rows.
        return {"bytes": case["rows"] * (8.0 * nh * hd + 2 * kvd * (4 + 2 * q4 + 2)), "flops": case["rows"] * (3.0 * (nh + nkv) * hd + 8.0 * kvd)}
    if kind == "ragged":
        # The lengths spread evenly over their logarithm from longest / 8 to longest.
        total = case["longest"] + (case["seqs"] - 1) * case["longest"] * (7.0 / 8.0) / math.log(8.0)
        w = {"bytes": 2.0 * total * kvd * q4 + 8.0 * case["seqs"] * nh * hd, "flops": 4.0 * nh * hd * total}
    else:
        rows, pos = case["rows"], case["pos"]
        # (A tree row sees a few of the tree's rows: about half of a line's here.)
        pairs = rows * pos + rows * (rows + 1) / (4.0 if case["tree"] else 2.0)
        w = {"bytes": 2.0 * (pos + rows) * kvd * q4 + 8.0 * rows * nh * hd, "flops": 4.0 * nh * hd * pairs}
    return {k: v * case["layers"] for k, v in w.items()}


# ---- the same in 64 bits ------------------------------------------------------------------


def _values64(units):
    """[units, 144] bytes -> values."""
    low, high = (units[:, :128] % 16).double(), (units[:, :128] // 16).double()
    d = units[:, 128:].contiguous().view(torch.float16).double()
    n = torch.empty(units.shape[0], 256, device=units.device, dtype=torch.float64)
    n[:, 0::2], n[:, 1::2] = low, high
    return ((n - 8.0).view(-1, 8, 32) * d[:, :, None]).view(-1)


def _stored64(x):
    """x [rows, n] as its 4-bit codes stand for it: each block's scale from the 64-bit values."""
    b = x.view(x.shape[0], -1, 32)
    top, bottom = b.max(2).values, b.min(2).values
    d = torch.where(top + bottom >= 0, top, bottom) / -8.0
    m, e = torch.frexp(d)
    d = torch.ldexp(torch.round(m * 128.0) / 128.0, e)
    size = torch.clamp(d.abs(), 2.0 ** -14, 896.0)
    d = torch.where(d > 0, size, -size)[:, :, None]
    return (torch.clamp(torch.round(b / d), -8, 7) * d).view(x.shape[0], -1)


def _turned64(x, positions, freq, neox):
    theta = (positions.float()[:, None] * freq[None, :]).double()  # the angle is an f32 product by definition
    z = torch.polar(torch.ones_like(theta), theta)[:, None, :]
    half, x = freq.numel(), x.double()
    pair = torch.complex(x[..., :half], x[..., half:]) if neox else torch.complex(x[..., 0::2].contiguous(), x[..., 1::2].contiguous())
    t = pair * z
    return torch.cat([t.real, t.imag], 2) if neox else torch.stack([t.real, t.imag], 3).reshape(x.shape)


def _attend64(q, k, v, nkv, visible):
    """q [rows, nh, hd] over k, v [slots, nkv, hd]; visible [rows, slots]."""
    rows, nh, hd = q.shape
    G, slots, out = nh // nkv, k.shape[0], torch.empty(q.shape, device=q.device, dtype=torch.float64)
    step = max(1, (1 << 26) // slots)
    for h in range(nh):
        kt, vh = k[:, h // G].t().contiguous(), v[:, h // G].contiguous()
        for r in range(0, rows, step):
            x = (q[r:r + step, h].double() @ kt) / math.sqrt(hd)
            x[~visible[r:r + step]] = -math.inf
            out[r:r + step, h] = torch.softmax(x, 1) @ vh
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "logprobs":
        x = s["scores"].double() / case["temperature"]
        lp = torch.log_softmax(x, 1)
        p = lp.exp()
        return {"logprob": lp[torch.arange(case["rows"], device="cuda"), s["tokens"].long()], "entropy": -(p * lp).sum(1), "ids": None,
                "top": torch.sort(lp, 1, descending=True).values[:, :case["top"]]}
    nh, nkv, hd = s["nh"], s["nkv"], s["hd"]
    if kind == "append":
        rows = case["rows"]
        return {"q": _turned64(s["q0"], s["positions"], s["freq"], s["neox"]),
                "k": _stored64(_turned64(s["k"], s["positions"], s["freq"], s["neox"]).reshape(rows, -1)),
                "v": _stored64(s["v"].double().view(rows, -1))}
    out = torch.empty(s["q"].shape, device="cuda", dtype=torch.float64)
    for l in range(case["layers"]):
        k, v = (_values64(s[n][l]) for n in ("kc", "vc"))
        if kind == "ragged":
            for i, (o, n) in enumerate(zip(s["offs"].astype(int), s["lens"].astype(int))):
                ki, vi = (t[o * nkv * hd:(o + n) * nkv * hd].view(n, nkv, hd) for t in (k, v))
                out[l, i:i + 1] = _attend64(s["q"][l, i:i + 1], ki, vi, nkv, torch.ones(1, n, device="cuda", dtype=torch.bool))
            continue
        rows, pos = case["rows"], case["pos"]
        slots = pos + rows
        if case["tree"]:
            see = torch.tensor([[(m >> j) & 1 for j in range(rows)] for m in _seen(rows, seed)], device="cuda", dtype=torch.bool)
            visible = torch.cat([torch.ones(rows, pos, device="cuda", dtype=torch.bool), see], 1)
        else:
            visible = torch.ones(rows, slots, device="cuda", dtype=torch.bool).tril(pos)
        ki, vi = (t[:slots * nkv * hd].view(slots, nkv, hd) for t in (k, v))
        out[l] = _attend64(s["q"][l], ki, vi, nkv, visible)
    return {"out": out}
