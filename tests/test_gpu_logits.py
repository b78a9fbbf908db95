"""q4mi_logits_process against its formula in 64 bits (numpy).

Tolerance: the fp32 steps (divide or multiply, freq * n, two subtractions,
k - 1 additions of biases and one of their sum) round at most k + 5 times,
each by 2^-24 of a value that is at most M = |z| max(rep, 1/rep) + |freq| n +
|pres| + sum |bias|; then one rounding to the type, half a step of |z| (or
half the smallest subnormal)."""
import numpy as np
import pytest
import torch

import q4mi

pytestmark = pytest.mark.gpu

TYPES = {q4mi.T_F32: torch.float32, q4mi.T_F16: torch.float16, q4mi.T_BF16: torch.bfloat16}


def dev(a, t=None):
    d = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return d if t is None else d.to(t)


def formula(x, hist, gen, pen, bias, masks, mask_row):
    """z and the tolerance's M and rounding counts; hist: a list of id arrays,
    bias: a list of (ids, values); each of the three may be None."""
    z = x.astype(np.float64).copy()
    b, v = z.shape
    m, k = np.abs(z), np.full(z.shape, 5.0)
    for i in range(b):
        if hist is not None:
            rep, freq, pres = (float(p) for p in pen[i])
            ok = (hist[i] >= 0) & (hist[i] < v)
            seen = np.unique(hist[i][ok])
            wrote = hist[i][gen[i]:][ok[gen[i]:]]
            n = np.bincount(wrote, minlength=v)
            with np.errstate(invalid="ignore"):
                z[i, seen] = np.where(z[i, seen] > 0, z[i, seen] / rep, z[i, seen] * rep)
                m[i] = np.maximum(m[i], m[i] * max(rep, 1 / rep))
                hit = n > 0
                z[i, hit] -= freq * n[hit] + pres
            m[i] += abs(freq) * n + abs(pres)
        if bias is not None:
            ids, val = bias[i]
            ok = (ids >= 0) & (ids < v)
            with np.errstate(invalid="ignore"):
                np.add.at(z[i], ids[ok], val[ok].astype(np.float64))
            np.add.at(m[i], ids[ok], np.abs(val[ok].astype(np.float64)))
            np.add.at(k[i], ids[ok], 1)
        if masks is not None and mask_row[i] >= 0:
            if mask_row[i] >= len(masks):
                z[i] = -np.inf
            else:
                bits = np.unpackbits(masks[mask_row[i]].view(np.uint8), bitorder="little")[:v]
                z[i, bits == 0] = -np.inf
    return z, m, k


def flat(lists, t):
    off = np.concatenate([[0], np.cumsum([len(a) for a in lists])]).astype(np.int64)
    return dev(np.concatenate(lists).astype(t)) if off[-1] else None, dev(off)


def call(L, xt, x, v, hist=None, gen=None, pen=None, bias=None, masks=None, mask_row=None,
         out=None, name_rows=True):
    """x [b][ld] on the device; returns out."""
    b = x.shape[0]
    out = torch.full_like(x, -7.0) if out is None else out
    keep = []

    def p(t):
        keep.append(t)
        return q4mi.ptr(t)

    h = ho = g = pe = bi = bv = bo = m = mr = None
    if hist is not None:
        h, ho = flat(hist, np.int32)
        g = dev(np.asarray(gen, np.int32)) if gen is not None else None
        pe = dev(np.asarray(pen, np.float32))
    if bias is not None:
        bi, bo = flat([a for a, _ in bias], np.int32)
        bv, _ = flat([a for _, a in bias], np.float32)
    if masks is not None:
        m = dev(masks.view(np.int32))
        mr = dev(np.asarray(mask_row, np.int32)) if name_rows else None
    q4mi.check(L.q4mi_logits_process(
        x.data_ptr(), xt, x.shape[1], b, v, p(h), p(ho), p(g), p(pe), p(bi), p(bv), p(bo), p(m),
        0 if masks is None else masks.shape[1], 0 if masks is None else len(masks), p(mr),
        out.data_ptr(), out.shape[1]), "logits")
    torch.cuda.synchronize()
    return out


def check(out, x, v, want, t):
    z, m, k = want
    got = out.double().cpu().numpy()
    assert (got[:, v:] == -7).all()
    got = got[:, :v]
    f = torch.finfo(t)
    with np.errstate(invalid="ignore"):
        tol = k * 2.0 ** -24 * m + np.abs(z) * f.eps / 2 + f.smallest_normal * f.eps / 2
        same = (got == z) | (np.isnan(got) & np.isnan(z))
        near = np.abs(got - z) <= tol
    assert (same | (near & np.isfinite(z))).all()


def make(rng, b, v, hmax, bmax, masks):
    hist = [rng.zipf(1.3, rng.integers(0, hmax + 1)) % (v + 2) - 1 for _ in range(b)]
    gen = [int(rng.integers(0, len(h) + 1)) for h in hist]
    pen = np.stack([rng.uniform(0.5, 2, b), rng.uniform(-0.5, 0.5, b), rng.uniform(-1, 1, b)],
                   1).astype(np.float32)
    bias = [(rng.integers(-1, v + 1, n), rng.uniform(-5, 5, n).astype(np.float32))
            for n in rng.integers(0, bmax + 1, b)]
    words = (v + 31) // 32
    ms = rng.integers(0, 1 << 32, (masks, words + 1), dtype=np.uint64).astype(np.uint32)
    ms[0] = 0
    return hist, gen, pen, bias, ms, rng.integers(-1, masks, b)


@pytest.mark.parametrize("xt", sorted(TYPES))
@pytest.mark.parametrize("b,v,pad,hmax,bmax", [
    (1, 1, 0, 5, 3), (1, 100, 0, 50, 10), (3, 32003, 5, 4000, 100), (5, 4096, 0, 300, 0),
    (2, 4097, 7, 0, 700), (9, 1000, 24, 2000, 2000), (1, 151936, 0, 3000, 50),
    (3, 5001, 0, 600, 60), (4, 2047, 2, 100, 9), (130, 10000, 1, 300, 20), (40, 60001, 0, 900, 30)])
def test_all_three(gpu, xt, b, v, pad, hmax, bmax):
    rng = np.random.default_rng(b * 100 + v)
    hist, gen, pen, bias, ms, rows = make(rng, b, v, hmax, bmax, 3)
    x = dev(4 * rng.standard_normal((b, v + pad)), TYPES[xt])
    want = formula(x[:, :v].double().cpu().numpy(), hist, gen, pen, bias, ms, rows)
    check(call(gpu, xt, x, v, hist, gen, pen, bias, ms, rows), x, v, want, TYPES[xt])


@pytest.mark.parametrize("parts", ["", "h", "b", "m", "hb", "hm", "bm"])
def test_each_part_alone(gpu, parts):
    rng = np.random.default_rng(len(parts) + 1)
    b, v = 4, 5003
    hist, gen, pen, bias, ms, rows = make(rng, b, v, 900, 40, 4)
    x = dev(4 * rng.standard_normal((b, v)), torch.float32)
    kw = {}
    if "h" in parts:
        kw.update(hist=hist, gen=gen, pen=pen)
    if "b" in parts:
        kw.update(bias=bias)
    if "m" in parts:
        kw.update(masks=ms, mask_row=rows)
    want = formula(x.double().cpu().numpy(), kw.get("hist"), gen, pen, kw.get("bias"),
                   kw.get("masks"), rows)
    out = call(gpu, 0, x, v, **kw)
    check(out, x, v, want, torch.float32)
    if not parts:
        assert torch.equal(out, x)


def test_defaults_of_gen_and_mask_rows(gpu):
    """No gen: the whole history counts as written; no mask_row: row b."""
    rng = np.random.default_rng(2)
    b, v = 3, 700
    hist, _, pen, _, ms, _ = make(rng, b, v, 500, 0, 3)
    x = dev(rng.standard_normal((b, v)), torch.float32)
    want = formula(x.double().cpu().numpy(), hist, [0] * b, pen, None, ms, [0, 1, 2])
    check(call(gpu, 0, x, v, hist, None, pen, None, ms, None, name_rows=False), x, v, want,
          torch.float32)


@pytest.mark.parametrize("v", [1, 7, 100, 538])
def test_biases_of_few_tokens(gpu, v):
    """Many biases a token: their fp32 sum in list order, to the bit."""
    rng = np.random.default_rng(v)
    b = 3
    x = rng.standard_normal((b, v)).astype(np.float32)
    bias = [(rng.integers(-1, v + 1, n), rng.uniform(-5, 5, n).astype(np.float32))
            for n in (1461, 64, 1000)]
    bias[1][0][:] = v - 1               # a whole wave's entries of one token
    want = np.empty_like(x)
    for i, (ids, val) in enumerate(bias):
        add = np.zeros(v, np.float32)
        for t, d in zip(ids, val):
            if 0 <= t < v:
                add[t] = add[t] + d
        want[i] = x[i] + add
    got = call(gpu, 0, dev(x), v, bias=bias).cpu().numpy()
    assert np.array_equal(got, want)


@pytest.mark.parametrize("v", [4096, 4093])
@pytest.mark.parametrize("xt", [q4mi.T_F16, q4mi.T_BF16])
def test_rounding_to_16_bits(gpu, xt, v):
    """Every kind of fp32 value, given as a bias of logits 0, is stored as its
    nearest 16-bit value, ties to even: halves between neighbours and the
    values beside them, subnormals, overflow, infinities, NaN."""
    rng = np.random.default_rng(v)
    t = TYPES[xt]
    step = 1 << (13 if xt == q4mi.T_F16 else 16)        # of the 16-bit type, in fp32 bits
    top = 0x47800000 if xt == q4mi.T_F16 else 0x7f800000
    bits = (rng.integers(0, top // step, (v, ), dtype=np.int64) * step + step // 2
            + rng.integers(-1, 2, v)).astype(np.uint32)
    small = np.arange(0, 600) * step // 2 + rng.integers(-1, 2, 600)
    bits[:600] = np.maximum(small, 0).astype(np.uint32)
    if xt == q4mi.T_F16:                                # halves of its subnormal step, 2^-24
        half = (np.arange(600) * 2.0 ** -25).astype(np.float32).view(np.uint32).astype(np.int64)
        bits[600:1200] = np.maximum(half + rng.integers(-1, 2, 600), 0).astype(np.uint32)
    edge = torch.finfo(t).max
    last = np.array([edge, np.inf, np.nan], np.float32).view(np.uint32)
    bits[1200:1209] = [last[0], last[0] + step // 2 - 1, last[0] + step // 2, last[0] + step // 2 + 1,
                       last[1], last[2], 0x7fffffff, 0, 1]
    val = (bits ^ (rng.integers(0, 2, v).astype(np.uint32) << np.uint32(31))).view(np.float32)
    x = torch.zeros((1, v), dtype=t, device="cuda")
    got = call(gpu, xt, x, v, bias=[(np.arange(v), val)]).cpu()
    want = torch.from_numpy(val).reshape(1, v).to(t)
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan) and int(nan.sum()) >= 2
    assert torch.equal(got[~nan], want[~nan])


def test_special_values(gpu):
    """Infinities and NaN in the logits, masked and not; infinite biases; a
    mask row out of range masks everything; the same id listed often."""
    v = 300
    x = np.linspace(-3, 3, 4 * v).reshape(4, v).astype(np.float32)
    x[:, 0], x[:, 1], x[:, 2], x[:, 3] = np.inf, -np.inf, np.nan, 0
    hist = [np.array([0, 1, 2, 3, 4, 4, 4, 299]), np.array([], int), np.arange(v),
            np.full(2000, 7)]
    gen = [0, 0, 100, 1000]
    pen = np.array([[1.5, 0.1, 0.2], [2, 1, 1], [0.7, -0.3, 0], [1.2, 0.01, 0.5]], np.float32)
    bias = [(np.array([5, 5, 5, 6]), np.array([1, 2, -3, np.inf], np.float32)),
            (np.array([], int), np.array([], np.float32)),
            (np.array([8, 1, 0]), np.array([-np.inf, 1, -1], np.float32)),
            (np.tile([9, 10, 11, 9], 60), np.linspace(-1, 1, 240).astype(np.float32))]
    ms = np.full((2, 10), 0xffffffff, np.uint32)
    ms[1, 0] = 0xffffffff ^ 0x7          # masks the inf, the -inf and the NaN
    rows = [0, 2, 1, -1]
    d = dev(x)
    want = formula(x, hist, gen, pen, bias, ms, rows)
    check(call(gpu, 0, d, v, hist, gen, pen, bias, ms, rows), d, v, want, torch.float32)
    assert np.isneginf(want[0][1]).all() and np.isneginf(want[0][2, :3]).all()


def test_in_place_repeatable(gpu):
    """In place gives the bits of out of place, call after call (duplicate
    biases are added in list order)."""
    rng = np.random.default_rng(6)
    b, v = 6, 9001
    hist, gen, pen, bias, ms, rows = make(rng, b, v, 3000, 3000, 4)
    bias = [(ids % 50, val) for ids, val in bias]
    x = dev(4 * rng.standard_normal((b, v)), torch.float32)
    first = call(gpu, 0, x, v, hist, gen, pen, bias, ms, rows)
    for _ in range(3):
        y = x.clone()
        call(gpu, 0, y, v, hist, gen, pen, bias, ms, rows, out=y)
        assert torch.equal(y.view(torch.int32), first.view(torch.int32))


def test_logits_graph(gpu):
    """Captured once, replayed as the history grows in place."""
    rng = np.random.default_rng(9)
    b, v, cap = 2, 3001, 400
    x = torch.empty((b, v), device="cuda")
    z = torch.empty_like(x)
    hist = dev(rng.integers(0, v, b * cap).astype(np.int32))
    off = torch.zeros(b + 1, dtype=torch.int64, device="cuda")
    pen = dev(np.array([[1.3, 0.1, 0.4]] * b, np.float32))

    def go():
        q4mi.check(gpu.q4mi_logits_process(
            x.data_ptr(), 0, v, b, v, hist.data_ptr(), off.data_ptr(), None, pen.data_ptr(), None,
            None, None, None, 0, 0, None, z.data_ptr(), v), "logits")

    x.normal_()
    go()
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph):
            q4mi.use_torch_stream()
            go()
    finally:
        q4mi.use_torch_stream()
    for n in (0, 1, 150, 400):
        x.normal_()
        off.copy_(dev(np.array([0, n, n + n // 2], np.int64)))
        go()
        torch.cuda.synchronize()
        want = z.clone()
        z.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(z, want)
