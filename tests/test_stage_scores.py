"""What GpuLayers.logprobs and GpuLayers.sample hold of scores, on the CPU (host_side.py)."""
import pytest

import host_side


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    return host_side.build(tmp_path_factory.mktemp("fake"))


SETUP = """
from layers import Config, GpuLayers, Matrix
cfg = Config(n_embd=64, n_layer=0, n_head=1, n_head_kv=1, head_dim=64, rope_dim=64, vocab=1000)
g = GpuLayers(c, cfg, [], head=(np.ones(64, np.float32), Matrix(8, bytes(1000 * 68), 1000, 64)))
def x(rows):
    return np.zeros((rows, 64), np.float32)
def pieces():  # rows of each product, from the rows of the call after it
    return [grid[1] if "k_logprobs" in name else grid[0 if "argmax" in name else 1] for name, grid in launches() if "k_logprobs" in name or "argmax" in name]
"""


@pytest.mark.parametrize("call", ["g.logprobs(x(rows), rows, [1] * rows, top=3)", "g.sample(x(rows), rows, 0.0, 1.0, 1, 0)"])
def test_scores_are_held_in_pieces(fake, call):
    """No more than SCORE_BYTES at once, in pieces of two rows or more."""
    host_side.run(fake, SETUP + f"""
for rows, most, want in ((100, 1 << 30, [100]), (100, 40 * 4000, [33, 33, 34]), (7, 4000, [2, 2, 3]), (7, 1, [2, 2, 3]), (1, 1, [1]), (2, 1, [2]), (3, 1, [3])):
    g.SCORE_BYTES = most
    g._scratch(rows)
    clear()
    {call}
    assert pieces() == want, (rows, most, pieces())
    sizes = sorted(n for _, n, _ in mallocs())
    assert max(want) * 4000 in sizes and sizes[-1] <= max(most, 3 * 4000, max(want) * 4000), sizes
""")


def test_a_call_that_fails_leaves_no_buffers(fake):
    """An argument that is refused, and a buffer that cannot be had."""
    host_side.run(fake, SETUP + """
g._scratch(50)
calls = [lambda: g.logprobs(x(50), 50, [1] * 50, top=65), lambda: g.logprobs(x(50), 50, [1] * 50, temperature=-1.0)]
for call in calls:
    was = fake.fake_live_count()
    try:
        call()
    except bchip.BchipError as e:
        assert e.code == bchip.E_ARG
    else:
        raise AssertionError("not refused")
    assert fake.fake_live_count() == was
for call in (lambda: g.logprobs(x(50), 50, [1] * 50, top=3), lambda: g.sample(x(50), 50, 0.0, 1.0, 1, 0)):
    was = fake.fake_live_count()
    fake.fake_budget(50 * 4000 - 1)  # the scores do not fit
    try:
        call()
    except bchip.BchipError as e:
        assert e.code == bchip.E_OOM
    else:
        raise AssertionError("there was room")
    fake.fake_budget(1 << 40)
    assert fake.fake_live_count() == was, "a buffer was left"
    call()
    assert fake.fake_live_count() == was
""")
