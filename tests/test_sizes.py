"""Sizes of elements and buffers by type."""
import pytest

import bchip


def test_elements_and_buffers():
    assert [bchip.esize(t) for t in (bchip.F32, bchip.F16)] == [4, 2]
    assert [bchip.nbytes_of(t, 300) for t in (bchip.F32, bchip.F16, bchip.Q4)] == [1200, 600, 288]
    assert [bchip.nbytes_of(bchip.Q4, n) for n in (0, 32, 256, 288)] == [0, 144, 144, 288]


@pytest.mark.parametrize("t", [bchip.Q4, 3, -1])
def test_a_type_without_a_size_of_its_own_is_refused(t):
    with pytest.raises(ValueError):
        bchip.esize(t)
    if t != bchip.Q4:
        with pytest.raises(ValueError):
            bchip.nbytes_of(t, 32)
