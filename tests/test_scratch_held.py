"""The context's scratch and graph capture, on the CPU (host_side.py): a block that a captured call
was given stays allocated until the context ends, whichever call outgrows it, since its graph may
be replayed; a block that no capture took is freed when it is outgrown."""
import pytest

import host_side


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    return host_side.build(tmp_path_factory.mktemp("fake"))


SETUP = """
def kv(t, n, kvd):
    return c.zeros(bchip.nbytes_of(t, n * kvd)), c.zeros(bchip.nbytes_of(t, n * kvd))
f, i = c.zeros(4 << 20), c.zeros(1 << 20)
def attention(t, rows, n, nh=8, nkv=2, hd=128):
    k, v = kv(t, n, nkv * hd)
    return lambda: c.attention(f, k, v, t, f, None, False, rows, nh, nkv, hd, n - rows, 0.1)
def ragged(t, seqs, n, nh=8, nkv=2, hd=128):
    k, v = kv(t, n, nkv * hd)
    return lambda: c.rope_append_attention_ragged(f, f, f, k, v, t, f, i, [n] * seqs, [0] * seqs, nh, nkv, hd, hd, 0, 0.1, f)
def matmul(n, rows=64, cols=4096):
    w, x, o = c.zeros(rows * cols // 32 * 34), c.zeros(n * cols * 4), c.zeros(n * rows * 4)
    return lambda: c.matmul(w, 8, x, o, rows, cols, n)
def sample(rows, vocab=30000):
    s = c.zeros(rows * vocab * 4)
    return lambda: c.sample(s, rows, vocab, 1.0, 0.9, 1, 0, i)
def logprobs(rows, vocab, top):
    s = c.zeros(rows * vocab * 4)
    return lambda: c.logprobs(s, rows, vocab, 1.0, None, None, None, top, f, f)
def blocks(call):  # that a call makes the workspace allocate
    clear()
    call()
    return mallocs()
"""

CALLS = {
    "matmul": "matmul(12)",
    "sample": "sample(1)",
    "logprobs": "logprobs(3, 70000, 20)",
    "f16 step": "attention(bchip.F16, 1, 900)",
    "f16 verify": "attention(bchip.F16, 8, 900)",
    "f16 prompt": "attention(bchip.F16, 2048, 2048, 64, 64, 128)",
    "f32 verify": "attention(bchip.F32, 8, 900)",
    "4-bit step": "attention(bchip.Q4, 1, 3000)",
    "4-bit verify": "attention(bchip.Q4, 8, 900)",
    "f16 ragged step": "ragged(bchip.F16, 2, 900)",
}


@pytest.mark.parametrize("name", CALLS)
def test_what_a_capture_took_outlives_larger_calls(fake, name):
    host_side.run(fake, SETUP + f"""
if {name!r} == "f16 prompt":
    f = c.zeros(2048 * 64 * 128 * 4)
call = {CALLS[name]}
took = blocks(call)
assert took, "this call takes no scratch"
with capturing():
    clear()
    call()
    assert launches() and not mallocs()
for larger in (logprobs(300, 120000, 64), matmul(3000), sample(40), attention(bchip.Q4, 1, 30000), attention(bchip.F16, 8, 20000),
               attention(bchip.Q4, 600, 9000), ragged(bchip.F16, 40, 900)):
    larger()
    assert all(live(m) for m in took), "a block of the graph's was freed"
c.close()
assert fake.fake_live_count() == 0  # the context's end frees them
""")


@pytest.mark.parametrize("name,larger", [("matmul(12)", "matmul(300)"), ("sample(1)", "sample(9)"), ("logprobs(3, 70000, 20)", "matmul(300)"),
                                         ("attention(bchip.F16, 1, 900)", "attention(bchip.Q4, 8, 20000)"),
                                         ("ragged(bchip.F16, 2, 900)", "ragged(bchip.F16, 40, 900)")])
def test_what_no_capture_took_is_freed_when_it_is_outgrown(fake, name, larger):
    """Also where a graph holds other blocks, or held one that has been outgrown since."""
    host_side.run(fake, SETUP + f"""
call, larger = {name}, {larger}
other = matmul(2) if "attention" in {name!r} or "ragged" in {name!r} else attention(bchip.Q4, 1, 3000)
other()
with capturing():
    other()  # of a block that `call` does not take
took = blocks(call)
assert took
grown = blocks(larger)
assert grown and not any(live(m) for m in took), "a block that no graph can use was kept"
""")
    host_side.run(fake, SETUP + f"""
call, larger = {name}, {larger}
call()
with capturing():
    call()
took = blocks(larger)  # the captured block is outgrown, and this one no graph has taken
assert took
more = (matmul(2000), sample(40), attention(bchip.Q4, 1, 120000), attention(bchip.F16, 8, 30000), ragged(bchip.F16, 200, 900))
for m in more:
    m()
assert not any(live(m) for m in took), "a block that no graph can use was kept"
""")


def test_a_capture_without_scratch_takes_none(fake):
    """Where nothing can be allocated, the calls that have a form without scratch take it, and leave
    the workspace as it is."""
    host_side.run(fake, SETUP + """
small, calls = attention(bchip.Q4, 1, 900), (attention(bchip.Q4, 1, 30000), matmul(12), logprobs(3, 70000, 20))
took = blocks(small)
assert took
for call in calls:
    with capturing():
        clear()
        call()
        assert launches()
    assert all(live(m) for m in took)
clear()
small()
assert not mallocs()
""")


def test_where_memory_is_full_lists_run_whole(fake):
    """A call whose scratch cannot be had runs without it, one after it that can takes it again, and a
    graph's block is not given up for an attempt that fails."""
    host_side.run(fake, SETUP + """
small, large, lp, mm = attention(bchip.Q4, 1, 3000), attention(bchip.Q4, 1, 120000), logprobs(3, 70000, 20), matmul(300)
took = blocks(small)
with capturing():
    small()
fake.fake_budget(1000)
for call, most in ((large, 1), (lp, 1), (mm, None)):
    got = blocks(call)
    assert not got and (most is None or len(launches()) == most), launches()
fake.fake_budget(1 << 40)
assert all(live(m) for m in took), "the graph's block was freed"
for call in (small, large, lp):
    clear()
    call()
    assert len(launches()) == 2, launches()  # the fold, the join
""")
