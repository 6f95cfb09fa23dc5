"""A pool of pages after a call that failed, on the CPU (host_side.py): conversations keep the slots they had, and the
next call is as if the failed one had not been."""
import pytest

import host_side
from test_paged_refusals import POOL, STAGE


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    return host_side.build(tmp_path_factory.mktemp("fake"))


STATE = """
def state():
    return dict(p.len), {s: list(x) for s, x in p.pages.items()}, list(p.spare), list(p.users)
x = lambda n: np.zeros((n, 64), np.float32)
def no_table(*a):
    raise bchip.BchipError(bchip.E_OOM, "no memory for a table")
"""


def test_a_pass_that_is_refused_after_its_pages_were_taken(fake):
    """No memory for the table; heads that the library refuses; states of another width; an error in a layer behind
    the first, whose rows are appended by then."""
    host_side.run(fake, STAGE + STATE + """
g = L.GpuLayers(c, cfg, [one, one], None, bchip.F16)
a, b, e = p.new(), p.new(), p.new()
g.forward_paged(x(25), [a, b], [20, 5], p)
was, real = state(), p.table
def again():  # the same pass, as if nothing had been
    g.forward_paged(x(24), [b, a, e], [20, 3, 1], p)
    check()
    assert p.len == {a: 23, b: 25, e: 1}
    for s, n in ((a, 20), (b, 5), (e, 0)):
        p.truncate(s, n)
    check()
run = lambda: g.forward_paged(x(24), [b, a, e], [20, 3, 1], p)
p.table = no_table
assert "table" in raises(bchip.BchipError, run)
assert state() == was
p.table = real
again()
was = state()
g.cfg.n_head = 17 * cfg.n_head_kv
g.scratch_rows = 0
assert "group" in raises(bchip.BchipError, run)
g.cfg.n_head = 2
assert state() == was
again()
was = state()
wide = np.zeros((24, 640), np.float32)
raises(bchip.BchipError, lambda: g.forward_paged(wide, [b, a, e], [20, 3, 1], p))
assert state() == was
again()
was, real, calls = state(), c.attention_paged, []
def second(*args):
    calls.append(1)
    if len(calls) == 2:
        raise KeyboardInterrupt
    return real(*args)
c.attention_paged = second
raises(KeyboardInterrupt, run)
c.attention_paged = real
assert state() == was
again()
""")


def test_a_refused_pass_of_forks(fake):
    """A conversation's own copy of a page that it shared may stay; its slots, and the others', are as they were."""
    host_side.run(fake, STAGE + STATE + """
g = L.GpuLayers(c, cfg, [one, one], None, bchip.F16)
a = p.new()
g.forward_paged(x(20), [a], [20], p)
f, h = p.fork(a), p.fork(a)
lens, real = dict(p.len), p.table
p.table = no_table
raises(bchip.BchipError, lambda: g.forward_paged(x(32), [f, a], [2, 30], p))
p.table = real
assert p.len == lens
check()
assert p.pages[h][0] == p.pages[f][0] == p.pages[a][0]
spare = len(p.spare)
g.forward_paged(x(32), [f, a], [2, 30], p)
check()
assert p.len == {a: 50, f: 22, h: 20} and spare - len(p.spare) == 2  # (a's two; the copies are there already)
""")


def test_copies_that_fail(fake):
    """A page that was to be copied stays shared, and its conversation's."""
    host_side.run(fake, STAGE + STATE + """
g = L.GpuLayers(c, cfg, [one, one], None, bchip.F16)
a = p.new()
p.extend([a], [20])
f, h = p.fork(a), p.fork(a)
was, real = state(), c.copy_pages
def refused_copy(*args):
    assert state() == was  # the tables name no page that was not copied
    raise bchip.BchipError(bchip.E_HIP, "a copy")
c.copy_pages = refused_copy
raises(bchip.BchipError, lambda: p.extend([f, a], [2, 30]))
assert state() == was
raises(bchip.BchipError, lambda: g.forward_paged(x(32), [f, a], [2, 30], p))
assert state() == was
seen = []
c.copy_pages = lambda bufs, t, n, pages, src, dst: (seen.append((list(src), list(dst))), real(bufs, t, n, pages, src, dst))
p.extend([f, a], [2, 30])
check()
assert p.len == {a: 50, f: 22, h: 20}
(src, dst), = seen
assert src == [p.pages[h][1]] * 2 and dst == [p.pages[f][1], p.pages[a][1]], (src, dst)
""")


def test_a_table_that_found_no_memory(fake):
    """The pool goes on with tables that there is memory for, and frees each buffer once."""
    host_side.run(fake, STAGE + STATE + """
a = p.new()
p.extend([a], [40])
first, _ = p.table([a])
for size in (first.nbytes, 64):  # a larger one is refused: then one of the first's size, and a small one
    raises(bchip.BchipError, lambda: (fake.fake_budget(64), p.table([a] * 3000)))
    fake.fake_budget((1 << 64) - 1)
    seqs = [a] * (size // 12)
    buf, stride = p.table(seqs)
    assert buf.ptr and buf.nbytes >= 12 * len(seqs) and stride == 3
    got = c.read(buf, (len(seqs), 3), np.uint32)
    assert (got == p.pages[a]).all()
was = fake.fake_live_count()
p.free()
assert was - fake.fake_live_count() == 5  # two layers' K and V, the table
""")


def test_a_stage_that_found_no_memory_for_its_rows(fake):
    """It goes on with passes that there is memory for, and keeps no buffer of the refused one."""
    host_side.run(fake, STAGE + STATE + """
g = L.GpuLayers(c, cfg, [one, one], None, bchip.F16)
a = p.new()
g.forward_paged(x(4), [a], [4], p)
kept = fake.fake_live_count()
zeros, had = c.zeros, []
def some(nbytes):
    if len(had) == fit:
        raise bchip.BchipError(bchip.E_OOM, "no more")
    had.append(nbytes)
    return zeros(nbytes)
for fit in (0, 1, 5):  # buffers that there is memory for
    c.zeros = some
    had.clear()
    raises(bchip.BchipError, lambda: g.forward_paged(x(100), [a], [100], p))
    assert len(had) == fit
    c.zeros = zeros
    assert p.len[a] == 4
    assert fake.fake_live_count() <= kept
    g.forward_paged(x(4), [a], [4], p)
    p.truncate(a, 4)
    assert fake.fake_live_count() == kept
g.forward_paged(x(100), [a], [100], p)
""")


def test_a_pool_that_finds_no_memory_keeps_none(fake):
    """A pool is asked for again with fewer pages: what the refused one had got is free by then."""
    host_side.run(fake, """
Buf, had = bchip.Buf, []
class Some(Buf):
    def __init__(self, ctx, nbytes):
        if len(had) == fit:
            raise bchip.BchipError(bchip.E_OOM, "no more")
        had.append(nbytes)
        super().__init__(ctx, nbytes)
was = fake.fake_live_count()
for fit in (0, 1, 3, 7):  # of four layers' K and V
    bchip.Buf = Some
    had.clear()
    try:
        bchip.PagePool(c, 4, 64, 10)
    except bchip.BchipError as e:
        assert e.code == bchip.E_OOM
    else:
        raise AssertionError("there was room")
    assert len(had) == fit and fake.fake_live_count() == was, fit
    bchip.Buf = Buf
p = bchip.PagePool(c, 4, 64, 10)
assert fake.fake_live_count() == was + 8
p.free()
assert fake.fake_live_count() == was
""")


@pytest.mark.parametrize("kind", ["uint8", "uint32", "uint64", "int32"])
def test_numbers_of_numpys_types(fake, kind):
    """Rows and lengths as arrays hold them (a device's accepted lengths are u32): as Python's numbers."""
    host_side.run(fake, STAGE + STATE + f"kind = np.{kind}" + """
g = L.GpuLayers(c, cfg, [one, one], None, bchip.F16)
a, b = p.new(), p.new()
p.extend([a, b], np.array([20, 33], kind))
check()
assert p.len == {a: 20, b: 33}
p.truncate(b, kind(16))
check()
assert len(p.pages[b]) == 1
p.truncate(a, np.array([3], kind)[0])
check()
g.forward_paged(x(30), np.array([b, a], kind), np.array([1, 29], kind), p)
check()
assert p.len == {a: 32, b: 17}
was, real = state(), p.table
p.table = no_table
raises(bchip.BchipError, lambda: g.forward_paged(x(30), [b, a], np.array([1, 29], kind), p))
p.table = real
assert state() == was
assert all(type(n) is int for n in p.len.values())
p.extend([a], [20])
check()
""")
