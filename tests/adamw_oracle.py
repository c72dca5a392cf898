"""AdamW and its 8-bit states in 64 bits (numpy), from the formulas.

`U` is half a step of float32 relative to the value (2^-24).  Each function
that gives a value gives the largest difference that float32 evaluation,
operation by operation, may have from it: the roundings on the way, counted."""
import numpy as np

U = 2.0 ** -24
BLOCK = 256
MASK = 0xFFFFFFFF


def clip_factor(norm, max_norm):
    return min(1.0, max_norm / (norm + 1e-6)) if max_norm else 1.0


def step(p, g, m, r, t, lr, beta1=0.9, beta2=0.999, eps=1e-8, wd=1e-2, coef=1.0, clipped=False, bits=32):
    """One step t from p, gradient g, first moment m and second moment's root r, all float64, where m and r are float32
    values: with 32-bit states m and the rounded root of v, with 8-bit states the rounded products of code and scale.
    Returns (p, m, v) and their bounds (dp, dm, dv), in units of U (half a step of float32), term by term:

    32 bits.  m: beta's rounding, the product's, the sum's.  v: the same on beta2 v, and v's root, rounded (2 in v), is
      what is known of it; the square's rounding, the factor's, the product's and the sum's on (1 - beta2) g^2.
    8 bits.  m: the known m's rounding, beta's, its product's with the scale, the sum's.  v = (root(beta2) r)^2 +
      (root(1 - beta2) g)^2: the known r's, the root's, its product's with the scale and the product's with the code
      count twice, the sum's once; of g's term the root's and the product's twice, the square's and the sum's once.
      sqrt is within two units, one reciprocal within two.
    Clipping: the factor's rounding and the product's, on g.
    p: 1 - lr wd and its product; of the update the factor lr / (1 - beta1^t), its product, the factor of r, its
      product, the sum with eps, the quotient (8 bits: reciprocal, two), what m and r carry; the difference."""
    c = 2 if clipped else 0
    g = g * coef
    a, b = np.abs(beta1 * m), np.abs((1 - beta1) * g)
    m2 = beta1 * m + (1 - beta1) * g
    x, y = beta2 * r * r, (1 - beta2) * g * g
    v2 = x + y
    if bits == 32:
        dm, dv, root = U * (3 * a + (3 + c) * b), U * (5 * x + (4 + 2 * c) * y), 1
    else:
        dm, dv, root = U * (4 * a + (3 + c) * b), U * (9 * x + (6 + 2 * c) * y), 2
    r2 = np.sqrt(v2)
    dr = np.where(v2 > 0, dv / (2 * np.maximum(r2, 1e-300)), 0.0) + root * U * r2
    root_c2 = np.sqrt(1 - beta2 ** t)
    denom = r2 / root_c2 + eps
    step_ = lr / (1 - beta1 ** t)
    upd = step_ * m2 / denom
    p2 = p * (1 - lr * wd) - upd
    dupd = step_ * dm / denom + np.abs(upd) * (7 * U + dr / (r2 + eps * root_c2))
    # second-order terms: every relative error here is below 1e-5
    dp = (2 * U * np.abs(p * (1 - lr * wd)) + dupd) * (1 + 1e-5) + U * np.abs(p2) + 1e-45
    # Products below the smallest normal number lose up to half of the smallest one, and v and r with them.
    tiny = 2.0 ** -149
    return (p2, m2, v2), (dp, dm + 2 * tiny, dv + 3 * tiny)


# ------------------------------------------------------------- 8-bit states

def e4m3_table():
    """The values of the 256 codes (sign, 4 exponent bits of bias 7, 3 mantissa bits; 0x7F is NaN)."""
    c = np.arange(256)
    e, f = (c >> 3) & 15, c & 7
    x = np.where(e == 0, f * 2.0 ** -9, (1 + f / 8) * 2.0 ** (e - 7.0))
    x[(c & 0x7F) == 0x7F] = np.nan
    return np.where(c & 0x80, -x, x)


GRID = e4m3_table()[:0x7F]  # 0 .. 448, rising


def blocks(x):
    """x in rows of one block, 0 behind its end."""
    n = -(-x.size // BLOCK) * BLOCK
    out = np.zeros(n, x.dtype)
    out[: x.size] = x
    return out.reshape(-1, BLOCK)


def scales(x):
    """Each block's scale: its largest magnitude / 448, 0 below 2^-100, NaN where it is not finite."""
    with np.errstate(invalid="ignore"):
        top = np.abs(blocks(x)).max(1)
    return np.where(np.isfinite(top), np.where(top < 2.0 ** -100, 0.0, top / 448.0), np.nan)


def mix(x):
    x = x & MASK
    x = ((x ^ (x >> 16)) * 0x6A09E667) & MASK
    x = ((x ^ (x >> 15)) * 0xBB67AE85) & MASK
    return x ^ (x >> 16)


def random16(n, seed, t):
    """The 16 random bits of elements 0 .. n-1 of a tensor with this seed at step t."""
    key = mix(mix(t) ^ (seed & MASK))
    i = np.arange(n, dtype=np.uint64)
    block = mix(np.uint64(key) + i // np.uint64(BLOCK))
    word = mix(block + (i % np.uint64(BLOCK)) // np.uint64(2) * np.uint64(0x9E3779B9))
    return np.where(i % 2 == 0, word & np.uint64(0xFFFF), word >> np.uint64(16)).astype(np.int64)


def neighbours(y):
    """The grid's values below (or at) and above 0 <= y <= 448."""
    k = np.clip(np.searchsorted(GRID, y, side="right") - 1, 0, len(GRID) - 1)
    return GRID[k], GRID[np.minimum(k + 1, len(GRID) - 1)]


def stochastic(y, bits):
    """y rounded by the bits, and how near the choice was: |distance - threshold| in steps of the grid."""
    y = np.where(y > 0, np.clip(y, 2.0 ** -9, 448.0), 0.0)
    lo, hi = neighbours(y)
    gap = np.where(hi > lo, hi - lo, 1.0)
    frac = (y - lo) / gap
    threshold = 1 - (bits * 16 + 8) / 2.0 ** 20
    return np.where(frac >= threshold, hi, lo), np.abs(frac - threshold)
