"""8-bit floating point rows in blocks of 128, the norm and the scored routing
in 64 bits, from their definitions (numpy)."""
import numpy as np


def blocks(cols):
    return (cols + 127) // 128


def level(code):
    """The value of e4m3 codes (uint8 array)."""
    c = np.asarray(code).astype(np.int64)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e == 0, m / 512.0, np.ldexp(1 + m / 8.0, e - 7))
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(c >= 128, -v, v)


LEVELS = level(np.arange(127))     # ascending, 0 .. 448
MID = (LEVELS[1:] + LEVELS[:-1]) / 2


def encode(a):
    """The nearest codes of values up to 448 in magnitude, ties to even."""
    m = np.abs(a)
    lo = np.searchsorted(MID, m, side="left")       # ties: the lower code
    hi = np.searchsorted(MID, m, side="right")      # ties: the upper one
    c = np.where(lo == hi, lo, np.where(lo % 2 == 0, lo, hi))
    return (c + 128 * np.signbit(a)).astype(np.uint8)


def quant(x, block=1):
    """Rows -> codes [rows][128 nb], scales [ceil(rows / block)][nb]."""
    x = np.asarray(x, np.float64)
    rows, cols = x.shape
    nb, rb = blocks(cols), -(-rows // block)
    v = np.zeros((rb * block, nb * 128))
    v[:rows, :cols] = x
    v = v.reshape(rb, block, nb, 128)
    bad = ~np.isfinite(v).all((1, 3))
    v = np.where(bad[:, None, :, None], 0.0, v)
    top = np.abs(v).max((1, 3))
    k = np.full(top.shape, -120)
    some = top > 448 * 2.0 ** -120
    # the least k with top <= 448 * 2^k
    f, e = np.frexp(top[some] / 448)
    k[some] = np.where(f == 0.5, e - 1, e)
    codes = encode(np.ldexp(v, -k[:, None, :, None])).reshape(rb * block, nb * 128)[:rows]
    return codes, np.where(bad, np.nan, np.ldexp(1.0, k)).astype(np.float32)


def values(codes, scales, cols, block=1):
    rows, nb = codes.shape[0], blocks(cols)
    s = np.repeat(np.asarray(scales, np.float64), block, 0)[:rows]
    v = level(codes).reshape(rows, nb, 128) * s[:, :, None]
    return v.reshape(rows, nb * 128)[:, :cols]


def route(z, topk, sigmoid=0, bias=None, groups=1, keep=1, group_top=1, renorm=True, scale=1.0):
    """ids and 64-bit weights of rows of logits."""
    z = np.asarray(z, np.float64)
    z = np.where(np.isnan(z), -np.inf, np.minimum(z, np.finfo(np.float32).max))
    out = z == -np.inf
    T, E = z.shape
    with np.errstate(over="ignore", invalid="ignore"):
        if sigmoid:
            s = 1 / (1 + np.exp(-z))
        else:
            e = np.where(out, 0, np.exp(z - z.max(1, keepdims=True)))
            s = np.divide(e, e.sum(1, keepdims=True), out=np.zeros_like(e),
                          where=e.sum(1, keepdims=True) > 0)
        s = np.where(out, 0, s)
        key = s if bias is None else s + np.asarray(bias, np.float64)
    key = np.where(out | np.isnan(key), -np.inf, key)
    if bias is None:
        rank = z        # the same order, and of scores that round alike too
    else:
        rank = key
    ids = np.full((T, topk), -1, np.int32)
    w = np.zeros((T, topk))
    size = E // groups
    for t in range(T):
        best = []
        for g in range(groups):
            k = sorted(key[t, g * size:(g + 1) * size], reverse=True)[:group_top]
            k = [v for v in k if v > -np.inf]
            best.append(sum(k) if k else -np.inf)
        order = sorted(range(groups), key=lambda g: (-best[g], g))
        stay = [g for g in order[:keep] if best[g] > -np.inf] if groups > 1 else [0]
        cand = [e for g in sorted(stay) for e in range(g * size, (g + 1) * size)
                if key[t, e] > -np.inf]
        cand.sort(key=lambda e: (-rank[t, e], e))
        for k, e in enumerate(cand[:topk]):
            ids[t, k], w[t, k] = e, s[t, e]
        if renorm:
            total = w[t].sum()
            w[t] = w[t] / total if total > 0 else 0
    return ids, w * scale
