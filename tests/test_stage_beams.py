"""How GpuLayers.beams cuts its searches into calls, on the CPU (host_side.py)."""
import pytest

import host_side


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    return host_side.build(tmp_path_factory.mktemp("fake"))


SETUP = """
from layers import Config, GpuLayers, Matrix
cfg = Config(n_embd=32, n_layer=0, n_head=1, n_head_kv=1, head_dim=32, rope_dim=32, vocab=1000)
g = GpuLayers(c, cfg, [], head=(np.ones(32, np.float32), Matrix(8, bytes(1000 * 34), 1000, 32)))
def pieces(n, beams, k=2, upto=None):  # searches of each selection
    clear()
    got = g.beams(np.zeros((n * beams, 32), np.float32), np.zeros((n, beams), np.float32), k, upto)
    assert [x.shape for x in got] == [(n, k)] * 3
    return [grid[0] for name, grid in launches() if "k_beam_join" in name]
"""


def test_searches_of_more_rows_than_a_call_takes(fake):
    """A selection takes 65535 rows: more searches of a short vocabulary go in several, though their scores would fit."""
    host_side.run(fake, SETUP + """
assert pieces(65535, 1, upto=8) == [65535]
for n, beams in ((65536, 1), (70000, 1), (40000, 2), (21846, 3), (1024, 64), (5000, 64)):
    got = pieces(n, beams, upto=8)
    most = 65535 // beams
    assert sum(got) == n and max(got) <= most and len(got) == -(-n // most), (n, beams, got)
""")


def test_scores_are_held_in_pieces(fake):
    host_side.run(fake, SETUP + """
for n, beams, most, want in ((100, 3, 1 << 30, [100]), (100, 1, 40 * 4000, [33, 33, 34]), (7, 2, 1, [1] * 7), (7, 1, 1, [2, 2, 3]), (1, 1, 1, [1]), (9, 2, 5 * 8000, [4, 5])):
    g.SCORE_BYTES = most
    assert pieces(n, beams) == want, (n, beams, most, pieces(n, beams))
""")


def test_searches_that_are_refused_leave_no_buffers(fake):
    host_side.run(fake, SETUP + """
g._scratch(400)
was = fake.fake_live_count()
for n, beams, k, code in ((2, 65, 2, bchip.E_ARG), (2, 0, 2, bchip.E_ARG), (2, 3, 65, bchip.E_ARG), (2, 3, 0, bchip.E_ARG)):
    try:
        pieces(n, beams, k)
    except bchip.BchipError as e:
        assert e.code == code, e
    else:
        raise AssertionError((n, beams, k))
    assert fake.fake_live_count() == was, (n, beams, k)
for x, sums in ((5, np.zeros((2, 3))), (6, np.zeros(6))):
    try:
        g.beams(np.zeros((x, 32), np.float32), sums, 2)
    except ValueError:
        pass
    else:
        raise AssertionError("taken")
assert pieces(0, 3) == []
""")


def test_scratch_of_a_selection(fake):
    """As include/bchip.h has it: a 256th of the bytes of rows of whole 1024 scores, and up to 1 KB a row."""
    host_side.run(fake, """
big = c.zeros(64 << 20).ptr
for n, beams, vocab in ((1, 1, 1), (1, 4, 1024), (1, 4, 1025), (3, 5, 151), (2, 8, 128256), (1, 16, 600000), (2000, 4, 900)):
    with bchip.Ctx(0) as fresh:
        clear()
        fresh.beam_select(big, big, n, beams, vocab, 1, big, big, big)
        taken = sum(size for _, size, _ in mallocs())
    rows = n * beams
    groups = rows * -(-vocab // 1024) * 1024 * 4 // 256
    assert groups < taken <= groups + 1024 * rows, (n, beams, vocab, taken)
""")
