"""The codes of values half-way between two, for every scale a block can have: the value times the
scale's f32 reciprocal, to the nearest even, as include/bchip.h says (a division would break some of
these ties the other way); and how near its code a value is."""
import numpy as np
import pytest

import bchip
import q4_plain as P

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = bchip.Ctx(0)
    yield c
    c.close()


def blocks():
    """A block for each mantissa of 7 bits, both signs and some exponents: its largest value 8 scales,
    the ties between codes, and values a unit in the last place beside some of them."""
    out = []
    for e in (-9, 0, 6):
        for m in range(64, 128):
            for sign in (1, -1):
                d = np.float32(sign * m * 2.0 ** (e - 6))
                ties = ((np.arange(-8, 7) + 0.5) * np.float64(d)).astype(np.float32)  # exact: 7 bits times 5
                near = np.concatenate([np.nextafter(ties[:8], np.float32(np.inf)), np.nextafter(ties[7:], np.float32(-np.inf))])
                out.append(np.concatenate([[np.float32(-8) * d], ties, near]))
    return np.array(out, np.float32)


@pytest.mark.parametrize("src", ["copy", "append"])
def test_ties_follow_the_reciprocal(ctx, src):
    x = blocks()
    assert x.shape[1] == 32
    n = x.size
    xb, kc, vc = ctx.upload(x), ctx.zeros(bchip.nbytes_of(bchip.Q4, n)), ctx.zeros(bchip.nbytes_of(bchip.Q4, n))
    if src == "copy":
        ctx.copy(xb, bchip.F32, vc, bchip.Q4, 0, n)
    else:
        ctx.rope_append(ctx.zeros(n * 4), xb, xb, kc, vc, bchip.Q4, ctx.zeros(64), ctx.zeros(4 * len(x)), len(x), 1, 1, 32, 0, False, 0)
    raw = ctx.read(vc, bchip.nbytes_of(bchip.Q4, n), np.uint8)
    codes, d = P.quantise(x)
    np.testing.assert_array_equal(raw, P.pack(codes, d))
    # 2^-24 of the reciprocal and 2^-24 of the product, of at most 8.
    d = d.astype(np.float64).reshape(-1, 1)
    ratio = x / d
    assert (np.abs(ratio - (codes.astype(np.float64) - 8))[ratio < 7.5] <= 0.5 + 2.0 ** -20).all()
    divided = np.clip(np.rint(ratio), -8, 7) + 8
    assert (divided != codes).any(), "these values do not tell the two apart"
    for b in (xb, kc, vc):
        b.free()
