"""Microscaled 4-bit rows in 64 bits, from the format's definition (numpy)."""
import numpy as np

LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def blocks(cols):
    return (cols + 31) // 32


def scale_row(cols):
    return (blocks(cols) + 3) // 4 * 4


def quant(x):
    """Rows of finite or non-finite values -> codes, scales (uint8)."""
    x = np.asarray(x, np.float64)
    rows, cols = x.shape
    nb = blocks(cols)
    v = np.zeros((rows, nb * 32))
    v[:, :cols] = x
    v = v.reshape(rows, nb, 32)
    bad = ~np.isfinite(v).all(2)
    v = np.where(bad[..., None], 0.0, v)
    top = np.abs(v).max(2)
    exp = np.where(top > 0, np.frexp(top)[1] - 3, -127).clip(-127, 127)
    a = np.ldexp(v, -exp[..., None])
    # distance to every level; a tie goes to the even code
    d = np.abs(np.abs(a)[..., None] - LEVELS)
    best = d.min(3, keepdims=True)
    tie = d == best
    code = np.where(tie[..., 0::2].any(3), 2 * tie[..., 0::2].argmax(3),
                    2 * tie[..., 1::2].argmax(3) + 1)
    code = (code + 8 * np.signbit(a)).astype(np.uint8)
    code = np.where(bad[..., None], 0, code).reshape(rows, nb * 32).astype(np.uint8)
    scales = np.zeros((rows, scale_row(cols)), np.uint8)
    scales[:, :nb] = np.where(bad, 255, exp + 127)
    return code[:, 0::2] | code[:, 1::2] << 4, scales


def values(codes, scales, cols):
    rows, nb = codes.shape[0], blocks(cols)
    c = np.stack([codes & 15, codes >> 4], 2).reshape(rows, nb, 32)
    v = np.where(c >= 8, -1.0, 1.0) * LEVELS[c & 7]
    f = np.where(scales[:, :nb] == 255, np.nan, np.ldexp(1.0, scales[:, :nb].astype(int) - 127))
    return (v * f[..., None]).reshape(rows, nb * 32)[:, :cols]


def random_rows(rng, rows, cols, lo, hi):
    """Uniform codes (0 past cols) and scales lo..hi."""
    nb = blocks(cols)
    c = rng.integers(0, 16, (rows, nb * 32)).astype(np.uint8)
    c[:, cols:] = 0
    s = np.zeros((rows, scale_row(cols)), np.uint8)
    s[:, :nb] = rng.integers(lo, hi + 1, (rows, nb))
    return c[:, 0::2] | c[:, 1::2] << 4, s
