"""What is measured of the operators around a KV cache kept in pages, and of beam search.

A pool holds, per layer, K and V as [pages x page slots][KV heads x head dim]; slot t of a sequence
lies in page table[t // page slots] of the pool, t % page slots into it. A sequence's new rows are its
last slots: row r of n new rows over `len` slots sees the slots up to len - n + r, itself among them.

A case's `kind` says which call a pass makes:
  append  one layer's rotation of q and k, and the append of k and v to the pages of each sequence
          (bchip_rope_append_paged); the rotated q and the pool come back.
  attend  attention of each sequence's new rows over its pages, `layers` layers
          (bchip_attention_paged): one row is a decode step, a few a verify pass, many a prompt or a
          piece of one; a batch may mix them.
  pages   whole pages copied to others in the K and V pools of `layers` layers
          (bchip_copy_pages): a conversation that forks, beams that part.
  beam    a step of beam search: the best continuations over the beams and the vocabulary
          (bchip_beam_select), by the sum of a beam's log probability and its next token's."""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

# (query heads, KV heads, head dim, neox pairs, rope base).
SHAPES = {"qwen05b": (14, 2, 64, True, 1e6), "llama8b": (32, 8, 128, False, 5e5), "qwen7b": (28, 4, 128, True, 1e6),
          "llama70b": (64, 8, 128, False, 5e5), "hd80": (10, 5, 80, True, 1e4), "hd256": (16, 4, 256, False, 1e4)}
TYPES = {"f32": torch.float32, "f16": torch.float16}

_lib = {}


def _ctx():
    """The program's one context of the library, made once."""
    if not _lib:
        sys.path.insert(1, os.path.join(os.getcwd(), "borrowed-compute_amd"))
        import bchip
        _lib["bchip"], _lib["ctx"] = bchip, bchip.Ctx(0)
    return _lib["bchip"], _lib["ctx"]


def _batch(kind, shape, cache, page, seqs, chunks, rows, earlier, pad=0, layers=1):
    """`chunks` of the `seqs` sequences have up to `rows` new rows, the others one; up to `earlier` slots
    before them; `pad` rows behind the last sequence's."""
    return {"kind": kind, "shape": shape, "cache": cache, "page": page, "seqs": seqs, "chunks": chunks, "rows": rows,
            "earlier": earlier, "pad": pad, "layers": layers}


def listed():
    return [
        # The token of a decode step of a small model: latency.
        {"name": "append_qwen05b_1", **_batch("append", "qwen05b", "f16", 16, 1, 0, 1, 510)},
        # Pieces of three prompts beside the tokens of six conversations.
        {"name": "append_llama8b_mixed", **_batch("append", "llama8b", "f16", 16, 9, 3, 777, 1500, 5)},
        # A decode step early in a conversation with a small model, head dim 64.
        {"name": "attend_qwen05b_1_400", **_batch("attend", "qwen05b", "f16", 16, 1, 0, 1, 399, layers=4)},
        # Sixteen conversations of ragged lengths, one step.
        {"name": "attend_llama8b_16_steps", **_batch("attend", "llama8b", "f16", 32, 16, 0, 1, 24000)},
        # Five conversations over the reference's own cache type.
        {"name": "attend_qwen7b_5_steps_f32", **_batch("attend", "qwen7b", "f32", 16, 5, 0, 1, 6000, layers=2)},
        # A piece of a long prompt after its first pieces.
        {"name": "attend_llama8b_2048_8192", **_batch("attend", "llama8b", "f16", 16, 1, 1, 2048, 8192)},
        # Pieces of two prompts beside the tokens of ten conversations, a padded batch.
        {"name": "attend_qwen7b_mixed", **_batch("attend", "qwen7b", "f16", 64, 12, 2, 513, 3000, 3)},
        # A prompt's piece over the reference's own cache type, odd sizes.
        {"name": "attend_qwen05b_501_f32", **_batch("attend", "qwen05b", "f32", 16, 1, 1, 501, 300)},
        # Beams that part: three last pages copied, every layer.
        {"name": "pages_llama8b_3", "kind": "pages", "shape": "llama8b", "cache": "f16", "page": 16, "layers": 32, "pages": 3},
        # A conversation forked whole.
        {"name": "pages_qwen7b_400", "kind": "pages", "shape": "qwen7b", "cache": "f16", "page": 16, "layers": 8, "pages": 400},
        # One search of four beams over the largest vocabulary.
        {"name": "beam_151936_1x4", "kind": "beam", "batch": 1, "beams": 4, "vocab": 151936, "k": 8, "first": False},
        # Searches of a batch.
        {"name": "beam_128256_16x8", "kind": "beam", "batch": 16, "beams": 8, "vocab": 128256, "k": 16, "first": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "attend", "attend", "attend", "attend", "pages", "beam", "beam"])
    if kind == "beam":
        beams = rng.choice([1, 2, 3, 4, 5, 8, 16])
        vocab = rng.choice([32000, 128256, 151936, _log(rng, 100, 150000)])
        return {"kind": kind, "batch": rng.choice([1, 1, rng.randint(2, max(2, 96 // beams))]), "beams": beams, "vocab": vocab,
                "k": min(rng.choice([beams, 2 * beams, 2 * beams, 64]), 64), "first": rng.random() < 0.2}
    shape, cache, page = rng.choice(list(SHAPES)), rng.choice(["f16", "f16", "f32"]), rng.choice([16, 16, 32, 64, 256])
    if kind == "pages":
        return {"kind": kind, "shape": shape, "cache": cache, "page": page, "layers": rng.randint(1, 32), "pages": _log(rng, 1, 60)}
    form = rng.choice(["steps", "steps", "verify", "chunk", "mixed"])
    if form == "steps":
        seqs, chunks, rows, earlier = rng.choice([1, rng.randint(2, 40)]), 0, 1, _log(rng, 1, 20000)
    elif form == "verify":
        seqs, rows, earlier = rng.randint(1, 12), rng.randint(2, 12), _log(rng, 1, 8000)
        chunks = seqs
    elif form == "chunk":
        seqs, chunks, rows, earlier = 1, 1, _log(rng, 17, 1500), rng.choice([0, _log(rng, 1, 4000)])
    else:
        chunks = rng.randint(1, 4)
        seqs, rows, earlier = chunks + rng.randint(1, 20), _log(rng, 17, 400), _log(rng, 1, 3000)
    return _batch(kind, shape, cache, page, seqs, chunks, rows, earlier, rng.choice([0, 0, rng.randint(1, 9)]),
                  rng.randint(1, 3) if kind == "attend" and seqs * rows < 64 else 1)


# ---- inputs, made from the seed alone -----------------------------------------------------


def _rows(case):
    """Each sequence's new rows and its slots with them: what a scheduler's step has, spread evenly over
    the logarithm of the largest to an eighth of it."""
    part = lambda i: 8.0 ** -((i * 0.6180339887498949) % 1.0)  # noqa: E731
    rows = [max(1, round(case["rows"] * part(i))) if i < case["chunks"] else 1 for i in range(case["seqs"])]
    return rows, [n + round(case["earlier"] * part(2 * i)) for i, n in enumerate(rows)]


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + 31)
    return g


def _randn(g, *shape, scale=1.0, dtype=torch.float32):
    return torch.empty(*shape, device="cuda").normal_(0.0, scale, generator=g).to(dtype)


def _freq(hd, base):
    i = np.arange(hd // 2, dtype=np.float64)
    return torch.from_numpy((base ** (-2.0 * i / hd)).astype(np.float32)).cuda()


def _first(n, beams):
    """The sums of a search's first step: one beam, the others not there yet."""
    x = torch.full((n, beams), -math.inf, device="cuda")
    x[:, 0] = 0.0
    return x


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    if kind == "beam":
        # Most of a vocabulary is unlikely; a few dozen tokens hold most of the mass. Beams lie some nats apart.
        n, beams, vocab, k = case["batch"], case["beams"], case["vocab"], case["k"]
        scores = _randn(g, n * beams, vocab, scale=2.0)
        at = torch.randint(0, vocab, (n * beams, 32), device="cuda", generator=g)
        scores.scatter_add_(1, at, 4.0 + 8.0 * torch.rand(n * beams, 32, device="cuda", generator=g))
        s = {"scores": scores, "sums": -20.0 - 2.0 * torch.rand(n, beams, device="cuda", generator=g) if not case["first"] else _first(n, beams),
             "best": torch.empty(n, k, device="cuda"), "beam": torch.empty(n, k, device="cuda", dtype=torch.int32),
             "token": torch.empty(n, k, device="cuda", dtype=torch.int32)}
    else:
        nh, nkv, hd, neox, base = SHAPES[case["shape"]]
        t, page = TYPES[case["cache"]], case["page"]
        s = {"nh": nh, "nkv": nkv, "hd": hd, "neox": neox}
        if kind == "pages":
            n, L = case["pages"], case["layers"]
            total = 2 * n + 3
            order = torch.randperm(total, device="cuda", generator=g).cpu().numpy().astype(np.uint32)
            s |= {"src": order[:n].copy(), "dst": order[n:2 * n].copy(),
                  "pool": _randn(g, 2 * L, total, page * nkv * hd, dtype=t)}  # every layer's K and V
        else:
            rows, lens = _rows(case)
            starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.uint32)
            all_rows, L = int(starts[-1]) + case["pad"], case["layers"]
            held = [-(-n // page) for n in lens]
            total = sum(held) + 3
            order = torch.randperm(total, device="cuda", generator=g)
            table = torch.full((len(lens), max(held)), total, device="cuda", dtype=torch.int32)  # past a list: no page
            for i, (a, n) in enumerate(zip(np.cumsum([0] + held), held)):
                table[i, :n] = order[a:a + n].to(torch.int32)
            s |= {"starts": starts, "lens": np.array(lens, np.uint32), "table": table, "total": total}
            if kind == "append":
                positions = np.zeros(all_rows, np.int32)
                for a, n, m in zip(starts, rows, lens):
                    positions[a:a + n] = np.arange(m - n, m)
                s |= {"q0": _randn(g, all_rows, nh, hd, scale=2.0), "k": _randn(g, all_rows, nkv, hd), "v": _randn(g, all_rows, nkv, hd),
                      "kc": _randn(g, total, page, nkv, hd, dtype=t), "vc": _randn(g, total, page, nkv, hd, dtype=t),
                      "freq": _freq(hd, base), "positions": torch.from_numpy(positions).cuda()}
                s["q"] = torch.empty_like(s["q0"])
            else:
                # Queries are larger than keys in earnest: the softmax has its peaks.
                s |= {"q": _randn(g, L, all_rows, nh, hd, scale=2.0), "kc": torch.empty(L, total, page, nkv, hd, device="cuda", dtype=t),
                      "vc": torch.empty(L, total, page, nkv, hd, device="cuda", dtype=t), "out": torch.zeros(L, all_rows, nh, hd, device="cuda")}
                for l in range(L):
                    s["kc"][l], s["vc"][l] = _randn(g, total, page, nkv, hd), _randn(g, total, page, nkv, hd)
    torch.cuda.synchronize()  # the library's stream does not wait for torch's
    s["case"] = case
    return s


# ---- one pass -----------------------------------------------------------------------------


def run(s):
    return (_OWN if own else _PLAIN)[s["case"]["kind"]](s, s["case"])


def _own_append(s, case):
    bchip, c = _ctx()
    t = bchip.F16 if case["cache"] == "f16" else bchip.F32
    p = {k: s[k].data_ptr() for k in ("q0", "q", "k", "v", "kc", "vc", "freq", "positions", "table")}
    c.copy(p["q0"], bchip.F32, p["q"], bchip.F32, 0, s["q0"].numel())  # the q product's place: it is rotated there
    c.rope_append_paged(p["q"], p["k"], p["v"], p["kc"], p["vc"], t, p["freq"], p["positions"], s["starts"], s["lens"], p["table"],
                        s["table"].shape[1], case["page"], s["total"], s["nh"], s["nkv"], s["hd"], s["hd"], s["neox"])
    return {"q": s["q"], "kc": s["kc"], "vc": s["vc"]}


def _own_attend(s, case):
    bchip, c = _ctx()
    t = bchip.F16 if case["cache"] == "f16" else bchip.F32
    a = [s[k] for k in ("q", "kc", "vc", "out")]
    at, by, table = [x.data_ptr() for x in a], [x.stride(0) * x.element_size() for x in a], s["table"].data_ptr()
    for l in range(case["layers"]):
        q, kc, vc, out = [x + l * y for x, y in zip(at, by)]
        c.attention_paged(q, kc, vc, t, out, s["starts"], s["lens"], table, s["table"].shape[1], case["page"], s["total"], s["nh"],
                          s["nkv"], s["hd"], 1.0 / math.sqrt(s["hd"]))
    return {"out": s["out"]}


def _own_pages(s, case):
    bchip, c = _ctx()
    t = bchip.F16 if case["cache"] == "f16" else bchip.F32
    pool = s["pool"]
    bufs = [pool.data_ptr() + i * pool.stride(0) * pool.element_size() for i in range(pool.shape[0])]
    c.copy_pages(bufs, t, pool.shape[2], pool.shape[1], s["src"], s["dst"])
    return {"pool": pool}


def _own_beam(s, case):
    _, c = _ctx()
    c.beam_select(s["scores"].data_ptr(), s["sums"].data_ptr(), case["batch"], case["beams"], case["vocab"], case["k"],
                  s["best"].data_ptr(), s["beam"].data_ptr(), s["token"].data_ptr())
    return {"best": s["best"], "beam": s["beam"], "token": s["token"]}


# The plain forms.


def _places(s, case):
    """Of every slot of every sequence its place in the pool [seqs, longest]: page x page slots + slot."""
    longest = int(s["lens"].max())
    t = torch.arange(longest, device="cuda")
    table = s["table"].long().clamp_max(s["total"] - 1)
    return table[:, t // case["page"]] * case["page"] + t % case["page"], t


def _of_rows(s):
    """Of every row its sequence, and the slot it is (seqs, slots: tensors on the GPU)."""
    starts, lens = (torch.from_numpy(s[n].astype(np.int64)).cuda() for n in ("starts", "lens"))
    n = int(s["starts"][-1])
    r = torch.arange(n, device="cuda")
    seq = torch.searchsorted(starts[1:], r, right=True)
    return seq, lens[seq] - (starts[seq + 1] - r)


def _rotate(x, positions, freq, neox):
    """x [rows, heads, hd] turned by the f32 angle the operator is defined by."""
    theta = positions.float()[:, None] * freq[None]
    cos, sin, half = theta.cos()[:, None], theta.sin()[:, None], freq.numel()
    a, b = (slice(0, half), slice(half, 2 * half)) if neox else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
    out, u, v = torch.empty_like(x), x[..., a], x[..., b]
    out[..., a], out[..., b] = u * cos - v * sin, u * sin + v * cos
    return out


def _plain_append(s, case):
    seq, slot = _of_rows(s)
    n = seq.numel()
    at = s["table"].long()[seq, slot // case["page"]] * case["page"] + slot % case["page"]
    turn = lambda x: _rotate(x, s["positions"][:n], s["freq"], s["neox"])  # noqa: E731
    for pool, x in ((s["kc"], turn(s["k"][:n])), (s["vc"], s["v"][:n])):
        pool.view(-1, s["nkv"], s["hd"])[at] = x.to(pool.dtype)
    return {"q": torch.cat([turn(s["q0"][:n]), s["q0"][n:]]), "kc": s["kc"], "vc": s["vc"]}


def _plain_attend(s, case):
    L, nh, nkv, hd = case["layers"], s["nh"], s["nkv"], s["hd"]
    at, t = _places(s, case)
    seq, slot = _of_rows(s)
    n, G, seqs, longest, most = seq.numel(), nh // nkv, len(s["lens"]), t.numel(), int(np.diff(s["starts"]).max())
    k, v = (s[m].view(L, -1, nkv, hd)[:, at].float().transpose(2, 3).contiguous() for m in ("kc", "vc"))  # [L, seqs, nkv, longest, hd]
    place = torch.arange(n, device="cuda") - torch.from_numpy(s["starts"].astype(np.int64)).cuda()[seq]
    q = torch.zeros(L, seqs, most, nh, hd, device="cuda")
    q[:, seq, place] = s["q"][:, :n]
    far = torch.full((seqs, most), longest - 1, device="cuda", dtype=torch.int64)  # (rows there are not see something)
    far[seq, place] = slot
    q = q.view(L, seqs, most, nkv, G, hd).permute(0, 1, 3, 4, 2, 5).reshape(L, seqs, nkv, G * most, hd)
    x = ((q / math.sqrt(hd)) @ k.transpose(3, 4).contiguous()).view(L, seqs, nkv, G, most, longest)
    x = torch.where(t <= far[:, None, None, :, None], x, -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).view(L, seqs, nkv, G * most, longest)
    o = (p @ v).view(L, seqs, nkv, G, most, hd).permute(0, 1, 4, 2, 3, 5).reshape(L, seqs, most, nh, hd)
    s["out"][:, :n] = o[:, seq, place]
    return {"out": s["out"]}


def _plain_pages(s, case):
    src, dst = (torch.from_numpy(s[n].astype(np.int64)).cuda() for n in ("src", "dst"))
    s["pool"][:, dst] = s["pool"][:, src]
    return {"pool": s["pool"]}


def _plain_beam(s, case):
    n, beams, vocab, k = case["batch"], case["beams"], case["vocab"], case["k"]
    x = s["scores"].double()  # (where sums lie next to each other 32 bits would make ties)
    x = x - x.amax(1, keepdim=True)
    x = (x - torch.log(torch.exp(x).sum(1, keepdim=True))).view(n, beams, vocab) + s["sums"].double()[:, :, None]
    x = x.view(n, beams * vocab)
    # Ties to the lowest beam, then the lowest token.
    low = torch.topk(x, k, 1)[0][:, -1:]
    order = torch.sort(torch.where(x >= low, x, -math.inf), dim=1, descending=True, stable=True)[1][:, :k]
    return {"best": x.gather(1, order).float(), "beam": (order // vocab).to(torch.int32), "token": (order % vocab).to(torch.int32)}


_OWN = {"append": _own_append, "attend": _own_attend, "pages": _own_pages, "beam": _own_beam}
_PLAIN = {"append": _plain_append, "attend": _plain_attend, "pages": _plain_pages, "beam": _plain_beam}


# ---- what a pass cannot do without --------------------------------------------------------


def work(case):
    kind = case["kind"]
    if kind == "beam":
        n = case["batch"] * case["beams"]
        return {"bytes": 4.0 * n * (case["vocab"] + 1) + 12.0 * case["batch"] * case["k"], "flops": 4.0 * n * case["vocab"]}
    nh, nkv, hd, _, _ = SHAPES[case["shape"]]
    kvd, size = nkv * hd, 2 if case["cache"] == "f16" else 4
    if kind == "pages":
        return {"bytes": 4.0 * case["layers"] * case["pages"] * case["page"] * kvd * size, "flops": 0.0}
    rows, lens = _rows(case)
    if kind == "append":
        # q read and left rotated, k and v read and written to their slots.
        return {"bytes": sum(rows) * (8.0 * nh * hd + 2.0 * kvd * (4 + size)), "flops": 3.0 * sum(rows) * (nh + nkv) * hd}
    pairs = sum(n * (m - n) + n * (n + 1) / 2.0 for n, m in zip(rows, lens))
    w = {"bytes": 2.0 * sum(lens) * kvd * size + 8.0 * sum(rows) * nh * hd, "flops": 4.0 * nh * hd * pairs}
    return {k: v * case["layers"] for k, v in w.items()}


# ---- the same in 64 bits ------------------------------------------------------------------


def _turned64(x, positions, freq, neox):
    theta = (positions.float()[:, None] * freq[None, :]).double()  # the angle is an f32 product by definition
    z = torch.polar(torch.ones_like(theta), theta)[:, None, :]
    half, x = freq.numel(), x.double()
    pair = torch.complex(x[..., :half], x[..., half:]) if neox else torch.complex(x[..., 0::2].contiguous(), x[..., 1::2].contiguous())
    t = pair * z
    return torch.cat([t.real, t.imag], 2) if neox else torch.stack([t.real, t.imag], 3).reshape(x.shape)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "beam":
        n, beams, k = case["batch"], case["beams"], case["k"]
        best = []
        for i in range(n):
            lp = torch.log_softmax(s["scores"][i * beams:(i + 1) * beams].double(), 1) + s["sums"][i].double()[:, None]
            best.append(torch.sort(lp.reshape(-1), descending=True).values[:k])
        return {"best": torch.stack(best), "beam": None, "token": None}
    if kind == "pages":
        out = s["pool"].double()
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            out[:, b] = s["pool"][:, a].double()
        return {"pool": out}
    nh, nkv, hd, page = s["nh"], s["nkv"], s["hd"], case["page"]
    table, starts, lens = s["table"].cpu().numpy(), s["starts"].tolist(), s["lens"].tolist()
    if kind == "append":
        q, kc, vc = s["q0"].double(), s["kc"].double(), s["vc"].double()
        for i, m in enumerate(lens):
            a, b = starts[i], starts[i + 1]
            q[a:b] = _turned64(s["q0"][a:b], s["positions"][a:b], s["freq"], s["neox"])
            kr = _turned64(s["k"][a:b], s["positions"][a:b], s["freq"], s["neox"])
            slots = np.arange(m - (b - a), m)
            pg, off = torch.from_numpy(table[i, slots // page].astype(np.int64)).cuda(), torch.from_numpy(slots % page).cuda()
            kc[pg, off], vc[pg, off] = kr, s["v"][a:b].double()
        return {"q": q, "kc": kc, "vc": vc}
    out = torch.zeros(s["out"].shape, device="cuda", dtype=torch.float64)
    G = nh // nkv
    for l in range(case["layers"]):
        for i, m in enumerate(lens):
            a, b = starts[i], starts[i + 1]
            held = torch.from_numpy(table[i, :-(-m // page)].astype(np.int64)).cuda()
            k, v = (s[x][l][held].reshape(-1, nkv, hd)[:m].double() for x in ("kc", "vc"))
            dark = torch.ones(b - a, m, device="cuda", dtype=torch.bool).triu(m - (b - a) + 1)
            for h in range(nh):
                x = s["q"][l, a:b, h].double() @ k[:, h // G].t().contiguous() / math.sqrt(hd)
                out[l, a:b, h] = torch.softmax(x.masked_fill(dark, -math.inf), 1) @ v[:, h // G].contiguous()
    return {"out": out}
