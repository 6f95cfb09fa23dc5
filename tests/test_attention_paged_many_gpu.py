"""bchip_attention_paged over more sequences than a launch takes, with lists that are cut: every launch's chunks take
scratch, the second's more than the first's, and in the other order less."""
import numpy as np
import pytest

import bchip
from paged_plain import Batch
from test_attention_paged_gpu import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv_type", [bchip.F16, bchip.F32])
@pytest.mark.parametrize("mixed", [False, True])
@pytest.mark.parametrize("longer_last", [True, False])
def test_two_launches_of_cut_lists(longer_last, mixed, kv_type):
    """A context of its own, whose first call grows the scratch between its launches while the first one may run."""
    rng = np.random.default_rng(4 * kv_type + 2 * mixed + longer_last)
    lens = rng.integers(700, 1000, 128).tolist() + rng.integers(3000, 5000, 60).tolist()
    if not longer_last:
        lens.reverse()
    rows = [(25 if mixed and i % 40 == 7 else 1) for i in range(len(lens))]
    b = Batch(rng, rows, lens, 2, 64, kv_type, page_slots=32, pad=1)
    q = (2 * rng.standard_normal((b.total, 8, 64))).astype(np.float32)
    with bchip.Ctx(0) as fresh:
        got = check(fresh, b, q, 8, 0.125)
        again = check(fresh, b, q, 8, 0.125)
    np.testing.assert_array_equal(got.view(np.uint32), again.view(np.uint32))
