"""What bchip_logprobs takes of the context's scratch, on the CPU (host_side.py)."""
import pytest

import host_side


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    return host_side.build(tmp_path_factory.mktemp("fake"))


SETUP = """
def call(rows, vocab, top):
    # (The scores' address is not the library's: nothing of their size is allocated here.)
    ids = c.zeros(max(1, rows * top) * 4)
    clear()
    c.logprobs(1 << 40, rows, vocab, 1.0, None, None, None, top, ids if top else None, ids if top else None)
    return sum(n for _, n, _ in mallocs()), launches()
"""


@pytest.mark.parametrize("rows,vocab,top", [(1, 151936, 64), (40, 151936, 64), (300, 128256, 20), (1023, 151936, 64), (1024, 600001, 64),
                                            (2047, 151936, 64), (2047, 600001, 0)])
def test_scratch_is_what_the_launch_writes(fake, rows, vocab, top):
    """A state of 16 bytes a unit of a row, and `top` keys a workgroup of a row: no more, whatever
    the vocabulary and the rows."""
    host_side.run(fake, SETUP + f"""
rows, vocab, top = {rows}, {vocab}, {top}
took, (first, join) = call(rows, vocab, top)
parts = first[1][0]
blocks = -(-vocab // 8192)
units = -(-blocks // -(-blocks // 64))
assert first[1] == (parts, rows, 1) and join[1] == (rows, 1, 1)
assert took == rows * (units * 16 + parts * top * 8), (took, parts, units)
assert took < 4300000
""")


def test_rows_that_fill_the_gpu_take_none(fake):
    """From 2048 rows on a workgroup takes a whole row: one launch, no scratch, up to the most rows."""
    host_side.run(fake, SETUP + """
for rows, vocab in ((2048, 151936), (4096, 151936), (8000, 9001), (65535, 600001)):
    took, run = call(rows, vocab, 64)
    assert took == 0 and [g for _, g in run] == [(1, rows, 1)], (rows, took, run)
""")


def test_a_capture_uses_scratch_that_is_large_enough(fake):
    """500 rows have fewer workgroups a row than one row has, and need no more than is there."""
    host_side.run(fake, SETUP + """
held, _ = call(2047, 16384, 64)
need = 500 * (19 * 16 + 5 * 64 * 8)
assert need < held < 500 * (19 * 16 + 19 * 64 * 8)
ids = c.zeros(500 * 64 * 4)
with capturing():
    clear()
    c.logprobs(1 << 40, 500, 151936, 1.0, None, None, None, 64, ids, ids)
    assert [g for _, g in launches()] == [(5, 500, 1), (500, 1, 1)], launches()
""")
