"""bchip_beam_select over the shortest vocabularies, whose rows fill a part of a group of scores, with beams that have
no distribution among them: every continuation that is asked for is one of the search's, named once, numbers
first."""
import numpy as np
import pytest

import bchip
from test_beam_gpu import formula, select

pytestmark = pytest.mark.gpu

# A row's form: a distribution, one with a masked token, a beam that is not there, and rows without a distribution.
FORMS = ["whole", "masked", "absent", "nan", "inf", "nothing", "nan sum"]


@pytest.fixture(scope="module")
def ctx():
    with bchip.Ctx(0) as c:
        yield c


def drawn(rng, n, beams, vocab):
    """Scores a whole number apart within a row, sums 100 apart: no two continuations that are numbers lie near
    each other, but for those at -inf."""
    scores = np.stack([rng.permutation(vocab) for _ in range(n * beams)]).astype(np.float32)
    sums = -100.0 * np.stack([rng.permutation(beams) for _ in range(n)]).astype(np.float32)
    form = rng.integers(0, len(FORMS), (n, beams))
    form[0] = 0                      # all whole
    form[1] = FORMS.index("nan")     # none of them
    form[2] = [0] + [FORMS.index("nan")] * (beams - 1)
    for i in range(n):
        for b in range(beams):
            row, f = scores[i * beams + b], FORMS[form[i, b]]
            t = rng.integers(vocab)
            if f == "masked" and vocab > 1:
                row[t] = -np.inf
            elif f == "absent":
                sums[i, b] = -np.inf
            elif f in ("nan", "inf"):
                row[t] = np.nan if f == "nan" else np.inf
            elif f == "nothing":
                row[:] = -np.inf
            elif f == "nan sum":
                sums[i, b] = np.nan
    return scores, sums


@pytest.mark.parametrize("vocab", [1, 2, 3, 4, 5, 63, 65, 193, 257])
@pytest.mark.parametrize("beams", [2, 3, 8, 21, 64])
def test_every_continuation_is_named_once(ctx, beams, vocab):
    rng = np.random.default_rng(100 * beams + vocab)
    n = 12
    scores, sums = drawn(rng, n, beams, vocab)
    full = formula(scores, sums).reshape(n, -1)
    place = np.arange(beams * vocab)
    # (NaN behind every number, equal ones by their place.)
    order = np.stack([np.lexsort((place, -np.where(np.isnan(x), 0, x), np.isnan(x))) for x in full])
    most = min(64, beams * vocab)
    for k in sorted({*range(1, min(most, 12) + 1), most // 2, most - 1, most} - {0}):
        best, beam, token = select(ctx, scores, sums, k)
        np.testing.assert_array_equal(beam.astype(np.int64) * vocab + token, order[:, :k], f"k {k}")
        want = np.take_along_axis(full, order[:, :k], 1)
        # The result's rounding, 2^-24 of it; log of a sum of at most 257 f32 terms, 2^-17 (test_beam_gpu.check).
        with np.errstate(invalid="ignore"):
            ok = (np.isnan(best) & np.isnan(want)) | (best == want) | (np.abs(best - want) <= 2.0 ** -17 + 2.0 ** -24 * np.abs(want))
        assert ok.all(), (k, best[~ok], want[~ok])
