"""What bchip_rope_append_attention_ragged refuses over 4-bit pools, and what it launches, on the CPU
(host_side.py)."""
import pytest

import host_side


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    return host_side.build(tmp_path_factory.mktemp("fake"))


SETUP = """
f, i = c.zeros(256 * 4 * 4096), c.zeros(1 << 10)
pool = c.zeros(144 * 40)  # ten slots of 8 x 128
def step(lens, offs, kc=None, vc=None, nh=32, nkv=8, hd=128, rd=128, q=f, k=f, t=bchip.Q4, out=f):
    return lambda: c.rope_append_attention_ragged(q, k, k, kc or pool, vc or pool, t, i, i, lens, offs, nh, nkv, hd, rd, 0, 0.1, out)
"""


def test_what_is_refused(fake):
    host_side.run(fake, SETUP + """
A, U = bchip.E_ARG, bchip.E_UNSUPPORTED
refused(A, step([0], [1]))                               # an empty list
refused(A, step([3, 3], [0, 8]))                         # past the pool, the second one
refused(A, step([3], [(1 << 64) // 1024]))               # an offset that overflows
refused(A, step([1] * 257, [0] * 257))                   # too many
refused(A, step([3], [0], kc=pool.ptr + 8))              # alignment
refused(A, step([3], [0], vc=pool.ptr + 8))
refused(A, step([3], [0], q=f.ptr + 4))
refused(A, step([3], [0], out=f.ptr + 4))
refused(A, step([3], [0], rd=130))
refused(A, step([3], [0], rd=63))
refused(A, step([3], [0], t=3))
refused(U, step([3], [0], nh=33))
refused(U, step([3], [0], nh=0, nkv=0))
refused(A, step([1] * 100, [0] * 100, k=c.zeros(99 * 4096)))  # past k
refused(A, lambda: c.rope_append_attention_ragged(f, f, f, None, pool, bchip.Q4, i, i, [1], [0], 32, 8, 128, 128, 0, 0.1, f))
refused(U, step([3], [0], hd=80, rd=80))                 # whole blocks
refused(U, step([3], [0], nh=34, nkv=2, hd=32, rd=32))   # 17 heads a group
refused(U, step([(1 << 32) - 255], [0], nh=1, nkv=1, hd=32, rd=32))
refused(U, step([3], [0], nh=8193, nkv=8193))            # slots past 2^20 elements
step([10], [0])()                                        # the last slot is one of the pool's
step([], [])()
""")


@pytest.mark.parametrize("seqs", [1, 64, 65, 256])
def test_what_is_launched(fake, seqs):
    """An append and an attention for each 64 sequences, the fold of lists that are cut, nothing else."""
    host_side.run(fake, SETUP + f"""
long = c.zeros(144 * 1000)  # 4000 slots of 64
for n, fold in ((300, 0), (4000, 1)):
    clear()
    step([n] * {seqs}, [0] * {seqs}, kc=long, vc=long, nh=4, nkv=1, hd=64, rd=64)()
    got = [name.split("attn_q4_")[-1][:4] if "attn_q4_" in name else "append" if "rope_append_q4" in name else name for name, _ in launches()]
    parts = ({seqs} + 63) // 64
    assert got == ["append"] * parts + ["rowI", "fold"][:1 + fold] * parts, got
""")
