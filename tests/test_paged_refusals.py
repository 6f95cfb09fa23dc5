"""The calls over a cache in pages and beam search on the CPU (host_side.py): what they refuse before any
launch, what they launch, and the host side of a pool (bchip.PagePool)."""
import pytest

import host_side


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    return host_side.build(tmp_path_factory.mktemp("fake"))


SETUP = """
from types import SimpleNamespace
import ctypes
class Args:
    '''A batch that is taken: 3 sequences of 1, 20 and 0 new rows over pages of 16 slots.'''
    def __init__(s, **changed):
        s.nh, s.nkv, s.hd, s.t, s.page, s.npages, s.stride = 8, 2, 64, bchip.F16, 16, 12, 5
        s.starts, s.lens = [0, 1, 21, 21], [40, 70, 3]
        s.rope_dim, s.neox, s.scale = 64, 0, 0.1
        s.__dict__.update(changed)
        rows, es = max(s.starts), 2 if s.t == bchip.F16 else 4
        big = c.zeros(64 << 20)
        s.q, s.k, s.v, s.out, s.kc, s.vc, s.freq, s.pos, s.table = (big.ptr + (i << 20) for i in range(9))
        s.__dict__.update(changed)
    def batch(s):
        return np.array(s.starts, np.uint32), np.array(s.lens, np.uint32), s.table, s.stride, s.page, s.npages, s.nh, s.nkv, s.hd
    def append(s):
        c.rope_append_paged(s.q, s.k, s.v, s.kc, s.vc, s.t, s.freq, s.pos, *s.batch(), s.rope_dim, s.neox)
    def attend(s):
        c.attention_paged(s.q, s.kc, s.vc, s.t, s.out, *s.batch(), s.scale)
"""


def test_a_batch_that_is_taken(fake):
    host_side.run(fake, SETUP + """
for t in (bchip.F16, bchip.F32):
    a = Args(t=t)
    clear()
    a.append()
    assert len(launches()) == 1 and "k_rope_append_paged" in launches()[0][0] and launches()[0][1][0] == 21, launches()
    clear()
    a.attend()
    assert len(launches()) == 1 and "attn_paged_mixed" in launches()[0][0], launches()  # both kinds of rows at once
    for rows, name in ((1, "attn_paged_row"), (20, "attn_paged_tile")):
        a = Args(t=t, starts=[0, rows], lens=[40])
        clear()
        a.attend()
        assert len(launches()) == 1 and name in launches()[0][0], launches()
    a = Args(t=t, hd=256, rope_dim=256)  # f16 heads past 128: a launch a kind
    clear()
    a.attend()
    assert len(launches()) == (2 if t == bchip.F16 else 1), launches()
""")


BATCH = {
    "an element type": ("E_ARG", "t=7"),
    "a cache in 4 bits": ("E_UNSUPPORTED", "t=bchip.Q4"),
    "heads that do not share": ("E_UNSUPPORTED", "nkv=3"),
    "a group past 16": ("E_UNSUPPORTED", "nh=34, nkv=2"),
    "a head dim off 8": ("E_UNSUPPORTED", "hd=60, rope_dim=60"),
    "a head dim past 256": ("E_UNSUPPORTED", "hd=264"),
    "no heads": ("E_UNSUPPORTED", "nh=0"),
    "a slot past 2^20 elements": ("E_UNSUPPORTED", "nh=8192, nkv=8192, hd=256"),
    "pages of 8 slots": ("E_UNSUPPORTED", "page=8"),
    "pages of 24 slots": ("E_UNSUPPORTED", "page=24"),
    "pages of no slots": ("E_UNSUPPORTED", "page=0"),
    "pages past 2^20 slots": ("E_UNSUPPORTED", "page=1 << 21"),
    "a pool of no pages": ("E_ARG", "npages=0"),
    "a pool past its buffer": ("E_ARG", "npages=70000"),
    "a line of too few pages": ("E_ARG", "stride=4"),
    "rows that start late": ("E_ARG", "starts=[1, 1, 21, 21]"),
    "rows that end before they start": ("E_ARG", "starts=[0, 1, 0, 21]"),
    "more rows than slots": ("E_ARG", "lens=[40, 19, 3]"),
    "a list past 2^32 - 256": ("E_UNSUPPORTED", "lens=[0xffffff01, 70, 3], stride=1 << 29"),
    "more than 256 sequences": ("E_ARG", "starts=list(range(258)), lens=[9] * 257"),
    "2^24 rows": ("E_UNSUPPORTED", "starts=[0, 0, 1 << 24, 1 << 24], lens=[1, 1 << 24, 1], stride=1 << 20"),
    "2^31 heads of rows": ("E_UNSUPPORTED", "nh=256, nkv=256, hd=8, rope_dim=8, starts=[0, 0, 1 << 23, 1 << 23], lens=[1, 1 << 23, 1], stride=1 << 20"),
    "an unaligned cache": ("E_ARG", "vc=c.zeros(1 << 20).ptr + 8"),
    "an unaligned q": ("E_ARG", "q=c.zeros(1 << 20).ptr + 4"),
    "an unaligned table": ("E_ARG", "table=c.zeros(1 << 20).ptr + 2"),
    "a table past its buffer": ("E_ARG", "table=c.zeros(4 * 9).ptr"),
    "a short q": ("E_ARG", "q=c.zeros(21 * 8 * 64 * 4 - 4).ptr"),
    "no cache": ("E_ARG", "kc=None"),
    "no table": ("E_ARG", "table=None"),
}


@pytest.mark.parametrize("name", BATCH)
def test_refused_batches(fake, name):
    code, changed = BATCH[name]
    host_side.run(fake, SETUP + f"""
a = Args({changed})
refused(bchip.{code}, a.append)
refused(bchip.{code}, a.attend)
""")


def test_refused_arguments_of_one_call(fake):
    host_side.run(fake, SETUP + """
for changed in (dict(rope_dim=63), dict(rope_dim=66), dict(k=None), dict(v=c.zeros(1 << 20).ptr + 8), dict(k=c.zeros(64).ptr), dict(pos=c.zeros(80).ptr),
                dict(freq=c.zeros(120).ptr)):
    refused(bchip.E_ARG, Args(**changed).append)
for changed in (dict(out=None), dict(out=c.zeros(1 << 20).ptr + 4), dict(out=c.zeros(21 * 8 * 64 * 4 - 4).ptr)):
    refused(bchip.E_ARG, Args(**changed).attend)
for starts, lens in (([0, 1], []), ([0], [1]), ([], [])):
    a = Args(starts=[0, 1], lens=[1])
    try:
        c.attention_paged(a.q, a.kc, a.vc, a.t, a.out, starts, lens, a.table, 5, 16, 12, 8, 2, 64, 0.1)
    except ValueError:
        pass
    else:
        raise AssertionError("taken")
""")


def test_batches_without_work(fake):
    """No sequences, and sequences without rows (whose lengths and table lines are not looked at): no launch, no error."""
    host_side.run(fake, SETUP + """
clear()
for a in (Args(starts=[0], lens=[]), Args(starts=[0, 0, 0], lens=[0, 0xffffffff], stride=1)):
    a.append()
    a.attend()
assert not launches()
""")


def test_scratch_of_a_call(fake):
    """A call that finds no memory, or that is captured before its size has run, takes its lists whole."""
    host_side.run(fake, SETUP + """
for lens, starts in (([3000, 2000], [0, 1, 2]), ([3000], [0, 30])):
    a = Args(lens=lens, starts=starts, stride=200, npages=320)
    clear()
    a.attend()
    assert len(launches()) == 2 and "fold" in launches()[1][0], launches()
    first = launches()
    fresh = bchip.Ctx(0)
    old, c = c, fresh
    with capturing():
        clear()
        a.attend()
        assert len(launches()) == 1 and not mallocs(), launches()
    fake.fake_budget(1 << 10)
    clear()
    a.attend()
    assert len(launches()) == 1, launches()
    fake.fake_budget((1 << 64) - 1)
    clear()
    a.attend()
    assert launches() == first
    c = old
    fresh.close()
""")


def test_refused_copies(fake):
    host_side.run(fake, """
pool = [c.zeros(10 * 2048) for _ in range(3)]
def copy(src, dst, bufs=pool, t=bchip.F16, elems=1024, npages=10):
    return lambda: c.copy_pages(bufs, t, elems, npages, src, dst)
clear()
copy([0, 0, 3], [1, 2, 4])()
assert len(launches()) == 1 and launches()[0][1] == (1, 3, 3), launches()
clear()
copy([], [])()
copy([0], [1], bufs=[])()
assert not launches()
for call in (copy([10], [1]), copy([0], [10]), copy([0, 1], [2, 2]), copy([0, 1], [1, 2]), copy([3], [3]), copy([0], [1], t=5), copy([0], [1], elems=0),
             copy([0], [1], elems=1020), copy([0], [1], npages=11), copy([0], [1], bufs=[pool[0].ptr + 8]), copy([0], [1], bufs=[pool[0], None]), copy([0], [1], elems=1 << 62),
             copy([0], [1], bufs=pool + [c.zeros(10 * 2048 - 16)])):
    refused(bchip.E_ARG, call)
refused(bchip.E_UNSUPPORTED, copy([0], [1], t=bchip.Q4))
try:
    copy([0, 1], [2])()
except ValueError:
    pass
else:
    raise AssertionError("taken")
""")


def test_refused_searches(fake):
    host_side.run(fake, """
s, m, a, b, d = (c.zeros(1 << 20) for _ in range(5))
def select(n=2, beams=3, vocab=100, k=5, **p):
    p = {"scores": s, "sums": m, "best": a, "beam": b, "token": d, **p}
    return lambda: c.beam_select(p["scores"], p["sums"], n, beams, vocab, k, p["best"], p["beam"], p["token"])
clear()
select()()
assert [n for n, _ in launches()] and len(launches()) == 2
clear()
select(n=0)()
assert not launches()
for call in (select(vocab=0), select(beams=0), select(beams=65), select(k=0), select(k=65), select(beams=1, vocab=4), select(n=30000), select(scores=None), select(sums=None),
             select(best=None), select(beam=None), select(token=None), select(vocab=1 << 20), select(sums=c.zeros(20)), select(best=c.zeros(36)), select(token=c.zeros(36))):
    refused(bchip.E_ARG, call)
select(n=1, beams=64, vocab=1, k=64)()
# Without scratch there is no search; the capture goes on.
fresh = bchip.Ctx(0)
c = fresh
with capturing():
    refused(bchip.E_OOM, select())
fake.fake_budget(1 << 4)
refused(bchip.E_OOM, select())
fake.fake_budget((1 << 64) - 1)
select()()
""")


POOL = """
p = bchip.PagePool(c, 2, 64, 10, 16, bchip.F16)
def check():
    held = [x for pages in p.pages.values() for x in pages]
    assert sorted(p.spare + list(set(held))) == list(range(10)), (p.spare, held)
    assert [held.count(x) for x in range(10)] == p.users
    assert all(len(p.pages[s]) == -(-p.len[s] // 16) for s in p.pages)
"""


def test_a_pool(fake):
    """Pages taken, shared, copied on the first write, truncated and given back."""
    host_side.run(fake, POOL + """
a, b = p.new(), p.new()
p.extend([a, b], [20, 16])
check()
assert p.len == {a: 20, b: 16} and [len(p.pages[s]) for s in (a, b)] == [2, 1]
clear()
f, g = p.fork(a), p.fork(a)
check()
assert p.pages[f] == p.pages[a]
p.extend([a, f, g, b], [1, 2, 0, 1])  # a and f write into the shared last page: two copies, g keeps it
check()
copies = [n for n in launches() if "k_copy_pages" in n[0]]
assert len(copies) == 1 and copies[0][1][1:] == (2, 4), launches()
assert len({p.pages[s][1] for s in (a, f, g)}) == 3 and len({p.pages[s][0] for s in (a, f, g)}) == 1
clear()
p.extend([g], [12])  # the page is its own by now
assert not launches()
check()
p.truncate(g, 16)
check()
p.truncate(g, 3)  # into the first page, which the others share
clear()
p.extend([g], [1])
assert len(launches()) == 1
check()
for s in (a, f, g, b):
    p.drop(s)
check()
assert len(p.spare) == 10 and not p.pages
""")


def test_a_pool_with_too_few_pages_is_left_as_it_was(fake):
    host_side.run(fake, POOL + """
a = p.new()
p.extend([a], [100])
f = p.fork(a)
was = (dict(p.len), {s: list(x) for s, x in p.pages.items()}, list(p.spare), list(p.users))
for seqs, rows in (([a], [16 * 3 + 13]), ([a, f], [12, 13 + 16 * 2]), ([f, a], [5, 60])):
    try:
        p.extend(seqs, rows)
    except MemoryError:
        pass
    else:
        raise AssertionError("taken")
    assert was == (dict(p.len), {s: list(x) for s, x in p.pages.items()}, list(p.spare), list(p.users))
for call in (lambda: p.extend([a, a], [1, 1]), lambda: p.extend([a], [1, 2]), lambda: p.truncate(a, 101)):
    try:
        call()
    except ValueError:
        pass
    else:
        raise AssertionError("taken")
p.extend([a, f], [12, 13 + 16])
check()
""")


STAGE = POOL + """
import layers as L
m = L.Matrix(0, bytes(4 * 64 * 64), 64, 64)
one = dict(attn_norm=np.ones(64), ffn_norm=np.ones(64), **{k: m for k in ("wq", "wk", "wv", "wo", "gate", "up", "down")})
cfg = L.Config(n_embd=64, n_layer=2, n_head=2, n_head_kv=2, head_dim=32, rope_dim=32)
def raises(what, call):
    try:
        call()
    except what as e:
        return str(e)
    raise AssertionError("taken")
"""


def test_a_refused_pass_takes_no_pages(fake):
    """What forward_paged refuses, and a pass without memory for its rows, leave the pool as it was."""
    host_side.run(fake, STAGE + """
g = L.GpuLayers(c, cfg, [one, one], None, bchip.F16)
many = [p.new() for _ in range(257)]
def untouched():
    assert len(p.spare) == 10 and not any(p.len.values()), p.len
x = lambda n: np.zeros((n, 64), np.float32)
assert "257" in raises(ValueError, lambda: g.forward_paged(x(1), many, [1] + [0] * 256, p)); untouched()
raises(ValueError, lambda: g.forward_paged(x(2), many[:1], [1], p)); untouched()
raises(ValueError, lambda: g.forward_paged(x(1), many[:2], [2, -1], p)); untouched()
raises(ValueError, lambda: g.forward_paged(x(1), many[:1], [1, 0], p)); untouched()
fake.fake_budget(1 << 10)
raises(bchip.BchipError, lambda: g.forward_paged(x(40), many[:1], [40], p)); untouched()
fake.fake_budget((1 << 64) - 1)
g.forward_paged(x(40), many[:256], [40] + [0] * 255, p)
assert p.len[many[0]] == 40 and len(p.spare) == 7
""")


def test_pools_of_another_stage(fake):
    """A stage takes pools of its own layers, elements and context."""
    host_side.run(fake, STAGE + """
x = np.zeros((1, 64), np.float32)
for n, t in ((1, bchip.F16), (3, bchip.F16), (2, bchip.F32)):
    g = L.GpuLayers(c, cfg, [one] * n, None, t)
    s = p.new()
    raises(ValueError, lambda: g.forward_paged(x, [s], [1], p))
    assert p.len[s] == 0
g = L.GpuLayers(c, cfg, [one] * 2, None, bchip.F16)
small = bchip.PagePool(c, 2, 32, 10)
s = small.new()
raises(ValueError, lambda: g.forward_paged(x, [s], [1], small))
with bchip.Ctx(0) as other:
    theirs = bchip.PagePool(other, 2, 64, 10)
    s = theirs.new()
    raises(ValueError, lambda: g.forward_paged(x, [s], [1], theirs))
    theirs.free()
""")


def test_pools_that_are_refused(fake):
    host_side.run(fake, STAGE + """
raises(ValueError, lambda: bchip.PagePool(c, 2, 64, 10, 16, bchip.Q4))
for slots in (0, 8, 24, 1 << 21):
    raises(ValueError, lambda: bchip.PagePool(c, 2, 64, 10, slots))
raises(ValueError, lambda: bchip.PagePool(c, 2, 64, 0))
raises(ValueError, lambda: L.GpuLayers(c, cfg, [one], None, bchip.Q4).new_pool(10))
s = p.new()
p.extend([s], [20])
for call in (lambda: p.truncate(s, -1), lambda: p.extend([s], [-1])):
    raises(ValueError, call)
    assert p.len[s] == 20
    check()
""")
