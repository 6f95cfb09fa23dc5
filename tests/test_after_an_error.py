"""A call after one that failed is not failed by it, on the CPU (host_side.py) and on the GPU."""
import numpy as np
import pytest

import bchip
import host_side


def test_a_call_after_memory_ran_out(tmp_path):
    host_side.run(host_side.build(tmp_path), """
x = c.zeros(4096)
fake.fake_budget(1 << 20)
for attempt in (lambda: c.zeros(1 << 21), lambda: c.sample(x, 1, 1000, 1.0, 0.9, 1, 0, x)):
    fake.fake_budget(100)
    refused(bchip.E_OOM, attempt)
    c.add(x, x, 1024)
    fake.fake_budget(1 << 20)
    c.add(x, x, 1024)
""")


@pytest.mark.gpu
def test_a_call_after_memory_ran_out_on_the_gpu():
    """An allocation past any card's memory, then ordinary work."""
    with bchip.Ctx(0) as c:
        x = c.upload(np.arange(1000, dtype=np.float32))
        with pytest.raises(bchip.BchipError) as e:
            c.zeros(1 << 44)
        assert e.value.code == bchip.E_OOM
        c.add(x, x, 1000)
        np.testing.assert_array_equal(c.read(x, 1000), 2 * np.arange(1000, dtype=np.float32))
