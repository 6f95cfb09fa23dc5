"""Which kernels attention over 4-bit caches launches, on the CPU (host_side.py)."""
import pytest

import host_side


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    return host_side.build(tmp_path_factory.mktemp("fake"))


SETUP = """
import re
def kernels(rows, nh, nkv, hd, pos, tree=False):
    # (Addresses that are not the library's: nothing of their size is allocated here.)
    clear()
    c.attention(1 << 40, 1 << 41, 1 << 42, bchip.Q4, 1 << 43, 1 << 44 if tree else None, tree, rows, nh, nkv, hd, pos, 0.1)
    got = []
    for name, grid in launches():
        kind, args = re.search(r"attn_q4_(row|tile|fold)I(.*?)EEv", name).groups()
        got.append((kind,) + tuple(map(int, re.findall(r"L[ib](\\d+)E", args + "E"))) + grid)
    return got
"""

# The passes that test_attention_q4_gpu.py runs for waves of 32 query rows, and its long passes of 16.
WIDE = [(1500, 32, 8, 128, 0), (1701, 28, 4, 128, 333), (7100, 14, 2, 64, 77), (3800, 12, 4, 96, 0), (6200, 16, 8, 32, 5)]
LONG = [(1100, 32, 8, 128, 0), (1037, 32, 8, 128, 333), (2345, 14, 2, 64, 77), (2801, 12, 4, 96, 0), (9000, 2, 2, 32, 5), (700, 16, 4, 256, 301)]


@pytest.mark.parametrize("rows,nh,nkv,hd,pos", WIDE + [(4096, 32, 8, 128, 0), (2000, 32, 8, 128, 100000), (5632, 8, 8, 128, 1 << 20)])
def test_waves_of_32_rows_take_whole_lists(fake, rows, nh, nkv, hd, pos):
    """One launch, a workgroup for 128 query rows of a KV head, however long the lists."""
    host_side.run(fake, SETUP + f"""
got = kernels({rows}, {nh}, {nkv}, {hd}, {pos})
assert got == [("tile", {hd} // 32, 2, {nkv}, 1, -(-{rows} * {nh} // {nkv} // 128))], got
assert not mallocs()
""")


@pytest.mark.parametrize("rows,nh,nkv,hd,pos", LONG)
def test_fewer_workgroups_take_16_rows_a_wave(fake, rows, nh, nkv, hd, pos):
    host_side.run(fake, SETUP + f"""
got = kernels({rows}, {nh}, {nkv}, {hd}, {pos})
assert got[0][:4] == ("tile", {hd} // 32, 1, {nkv}) and got[0][5] == -(-{rows} * {nh} // {nkv} // 64), got
assert [g[0] for g in got[1:]] == ["fold"] * (got[0][4] > 1), got
""")


def test_a_tree_of_many_heads_takes_whole_lists(fake):
    host_side.run(fake, SETUP + """
got = kernels(64, 768, 48, 96, 70, tree=True)
assert got == [("tile", 3, 2, 48, 1, 8)], got
""")


def test_a_tree_whose_masks_could_name_slots_past_the_longest_list_is_refused(fake):
    """A mask names slots up to 63 behind pos; lists reach slot 2^32 - 256 at most. What was named past
    that was left out in silence."""
    host_side.run(fake, SETUP + """
most = (1 << 32) - 256
kernels(2, 1, 1, 32, most - 64, tree=True)
kernels(2, 1, 1, 32, most - 2)
refused(bchip.E_UNSUPPORTED, lambda: kernels(2, 1, 1, 32, most - 63, tree=True))
refused(bchip.E_UNSUPPORTED, lambda: kernels(2, 1, 1, 32, most - 1))
""")
