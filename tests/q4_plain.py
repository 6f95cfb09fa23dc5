"""The 4-bit cache format and attention over it, restated in numpy for the tests: units of 256
elements, 128 bytes of codes (the even element of a pair in the low four bits) and eight f16
scales, an element (code - 8) x scale."""
import numpy as np


def quantise(x):
    """Codes and scales of x's last dimension in blocks of 32, in the f32 steps the format is
    defined by (a scale is the value of the largest magnitude over -8, the positive one of two,
    in 7 significant bits within 2^-14 .. 896; a block that is not finite has the scale NaN)."""
    b = np.asarray(x, np.float32).reshape(*np.shape(x)[:-1], -1, 32)
    bad = ~np.isfinite(b).all(-1)
    b = np.where(bad[..., None], np.float32(0), b)
    hi, lo = b.max(-1), b.min(-1)
    pos = hi >= -lo
    mag = np.where(pos, hi, -lo).astype(np.float32) * np.float32(0.125)
    u = mag.view(np.uint32).astype(np.uint64)
    u = (u + 0xFFFF + ((u >> 17) & 1)) & ~np.uint64(0x1FFFF)
    d = np.clip(u.astype(np.uint32).view(np.float32), np.float32(2.0 ** -14), np.float32(896.0))
    d = np.where(pos, -d, d).astype(np.float32)
    n = np.clip(np.rint(b * (np.float32(1.0) / d)[..., None]), -8, 7) + 8
    n[bad] = 8
    d[bad] = np.nan
    return n.astype(np.uint8).reshape(np.shape(x)), d.astype(np.float16)


def pack(codes, d):
    """A buffer's bytes: whole units, the last one filled up with zero bytes."""
    codes, d = codes.reshape(-1), d.reshape(-1)
    units = -(-codes.size // 256)
    c = np.zeros(units * 256, np.uint8)
    s = np.zeros(units * 8, np.float16)
    c[:codes.size], s[:d.size] = codes, d
    out = np.empty((units, 144), np.uint8)
    c = c.reshape(units, 128, 2)
    out[:, :128] = c[..., 0] | (c[..., 1] << 4)
    out[:, 128:] = s.view(np.uint8).reshape(units, 16)
    return out.reshape(-1)


def unpack(buf, n):
    """The first n elements of a buffer, in f64."""
    u = np.asarray(buf, np.uint8).reshape(-1, 144)
    codes = np.stack([u[:, :128] & 15, u[:, :128] >> 4], -1).reshape(-1, 8, 32).astype(np.float64) - 8.0
    d = np.ascontiguousarray(u[:, 128:]).view(np.float16).astype(np.float64)
    with np.errstate(invalid="ignore"):
        return (codes * d[..., None]).reshape(-1)[:n]


def stored(x):
    """x as a 4-bit buffer gives it back."""
    codes, d = quantise(x)
    return unpack(pack(codes, d), codes.size).reshape(np.shape(x))


def attention(q, k, v, nkv, visible, scale):
    """q [rows, nh, hd]; k, v [slots, nkv, hd] f64; visible [rows, slots]. A row that sees nothing
    gives zeros; unseen values are not touched. Also each output's sums of weight x |v| and of |v|,
    and each row's largest sum of |scale q k|, what rounding errors go by."""
    rows, nh, hd = q.shape
    G = nh // nkv
    out, mass, low, top = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape), np.zeros((rows, nh))
    q = q.astype(np.float64)
    for r in range(rows):
        see = np.flatnonzero(visible[r])
        if not len(see):
            continue
        for h in range(nh):
            kk, vv = k[see, h // G], v[see, h // G]
            s = kk @ q[r, h] * scale
            with np.errstate(invalid="ignore"):
                p = np.exp(s - s.max())
                p /= p.sum()
                out[r, h], mass[r, h] = p @ vv, p @ np.abs(vv)
            low[r, h] = np.abs(vv).sum(0)
            top[r, h] = (np.abs(kk) @ np.abs(q[r, h])).max() * abs(scale)
    return out, (mass, low), top


def bound(mass, top, hd):
    """How far an f32-grade result may be from the formula, by its roundings. A score's error: q
    as two f16 keeps 2^-22 of each product, q x scale rounds by 2^-24, and the sum of a head's
    products, 32 an MFMA with its two parts in turn, rounds at most 16 times an MFMA, 2 hd / 32 of
    them: 2^-24 of the sum of magnitudes each. With every score off by at most ds, a weight e^s / sum
    e^s lies within a factor e^(2 ds) of its own: off by at most e^(2 ds) - 1 of itself (2 ds only
    where ds is small), and so is the sum of weight x |v|. 2^-20 more for exp2, the weights' two
    parts and the weighted sum's roundings. And a weight is held as two f16 of itself over the
    largest times 2^11 or more, whose smallest step is 2^-24: half of it twice, 2^-35 of the
    largest weight, which is at most 1, is lost whatever the weight, times |v|."""
    mass, low = mass
    ds = top * (2.0 ** -22 + 2.0 ** -24 * (hd + 2))
    with np.errstate(over="ignore", invalid="ignore"):
        # (Weights that sum to 1 move a result by no more than twice the largest |v|, whatever ds.)
        return np.fmin(mass * np.expm1(2 * ds[..., None]), 2 * low) + 2.0 ** -20 * mass + 2.0 ** -35 * low + 1e-30
