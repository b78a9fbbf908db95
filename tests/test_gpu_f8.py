"""8-bit floating point rows in blocks of 128 on the GPU, against the format's
definition in 64 bits (f8_ref).

Codes and scales are exact.  Products come in two kinds of data:
  - codes of whole numbers up to 8 in magnitude and scales 1/4 .. 1 (powers of
    two): every partial sum in any order is a multiple of 2^-4 below 2^20 for
    rows of up to 16384 values (64 * 16384), so fp32 sums are exact and y must be
    the 64-bit result, rounded once;
  - any data.  With S the sum over all values of |w x| and nb blocks: a block's
    sum is at most 128 additions, each off by at most 2^-23 of a partial sum
    (2^-24 if to nearest; hardware sums may cut off); the two scales' product and
    its use with the addition 2^-24 each; nb blocks and at most 32 parts of them
    are added.  So y is off by at most (2 * 128 + 2 + nb + 32) * 2^-24 * S, then
    by one rounding to its type.  16-bit outputs of more than sixteen rows may lose
    more in one eight of products (test_gpu_f8_paths has that bound); the data here
    stay within the narrower one.
"""
import numpy as np
import pytest
import torch

import f8_ref as ref
import q4mi

pytestmark = pytest.mark.gpu

TYPES = {q4mi.T_F32: torch.float32, q4mi.T_F16: torch.float16, q4mi.T_BF16: torch.bfloat16}
F8 = q4mi.T_F8


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def host(t):
    return t.cpu().numpy()


def quant(L, x, xt, ld, rows, cols, block=1, ids=None):
    nb = ref.blocks(cols)
    c = torch.full((rows, nb * 128), 0xcd, dtype=torch.uint8, device="cuda")
    s = torch.full((-(-rows // block), nb), -7.0, device="cuda")
    q4mi.check(L.q4mi_f8_quant(x.data_ptr(), xt, ld, q4mi.ptr(ids), rows, cols, block,
                               c.data_ptr(), s.data_ptr()), "quant")
    return c, s


# ------------------------------------------------------------- quantisation

@pytest.mark.parametrize("block", [1, 128])
@pytest.mark.parametrize("xt", sorted(TYPES))
@pytest.mark.parametrize("rows,cols,pad,shift", [
    (1, 1, 0, 0), (1, 127, 0, 0), (3, 128, 0, 0), (2, 129, 3, 1), (5, 100, 28, 0), (1, 2048, 0, 0),
    (127, 513, 7, 0), (129, 256, 0, 0), (260, 640, 8, 0), (19, 1013, 1, 3)])
def test_quant_exact(gpu, xt, rows, cols, pad, shift, block):
    rng = np.random.default_rng(rows * 1000 + cols)
    ld = cols + pad
    v = rng.standard_normal((rows, ld)) * np.exp2(rng.integers(-12, 9, (rows, ld)))
    v[rng.random((rows, ld)) < 0.05] = 0
    flat = torch.zeros(rows * ld + shift, dtype=TYPES[xt], device="cuda")
    flat[shift:] = dev(v.reshape(-1)).to(TYPES[xt])
    x = flat[shift:]
    c, s = quant(gpu, x, xt, ld, rows, cols, block)
    want = ref.quant(host(x.double()).reshape(rows, ld)[:, :cols], block)
    assert np.array_equal(host(s), want[1])
    assert np.array_equal(host(c), want[0])


def test_quant_every_boundary(gpu):
    """Every code, tie and a tie's neighbours at every scale, subnormals and the
    largest values included; largest magnitudes on both sides of 448 * 2^k."""
    up, down = (np.nextafter(ref.MID.astype(np.float32), np.float32(d)) for d in (1e9, 0))
    vals = np.concatenate([ref.LEVELS, ref.MID, up, down]).astype(np.float32)
    vals = np.concatenate([vals, -vals, [0.0, -0.0, 1e-30]]).astype(np.float32)
    vals = np.concatenate([vals, np.zeros(-len(vals) % 127, np.float32)]).reshape(-1, 127)
    rows = []
    for e in list(range(-149, -100)) + list(range(-12, 13)) + list(range(100, 120)):
        for top in (448.0, 447.99997, 448.00003, 256.0):
            r = np.concatenate([np.full((len(vals), 1), top, np.float32), vals], 1)
            rows.append(np.ldexp(np.clip(r, -top, top), e).astype(np.float32))
    x = np.concatenate(rows)
    assert np.isfinite(x).all()
    c, s = quant(gpu, dev(x), q4mi.T_F32, 128, len(x), 128)
    want = ref.quant(x)
    assert np.array_equal(host(s), want[1])
    assert np.array_equal(host(c), want[0])
    y = torch.empty((len(x), 128), device="cuda")
    q4mi.check(gpu.q4mi_f8_dequant(c.data_ptr(), s.data_ptr(), None, len(x), 128, 1, y.data_ptr(),
                                   0, 128), "dequant")
    assert np.array_equal(host(y), ref.values(*want, 128).astype(np.float32))


@pytest.mark.parametrize("block", [1, 128])
def test_quant_non_finite(gpu, block):
    x = np.ones((130, 384), np.float32)
    x[0, 5], x[1, 140], x[129, 383], x[2, 0] = np.inf, np.nan, -np.inf, np.nan
    for xt, t in TYPES.items():
        c, s = quant(gpu, dev(x).to(t), xt, 384, 130, 384, block)
        want = ref.quant(x, block)
        assert np.array_equal(host(s), want[1], equal_nan=True)
        assert np.array_equal(host(c), want[0])
        y = torch.empty((130, 384), device="cuda")
        q4mi.check(gpu.q4mi_f8_dequant(c.data_ptr(), s.data_ptr(), None, 130, 384, block,
                                       y.data_ptr(), 0, 384), "dequant")
        assert np.array_equal(host(y), ref.values(*want, 384, block), equal_nan=True)


@pytest.mark.parametrize("block", [1, 128])
def test_quant_gather_and_repeat(gpu, block):
    rng = np.random.default_rng(5)
    x = rng.standard_normal((9, 160)).astype(np.float32)
    ids = rng.integers(0, 9, 300).astype(np.int32)
    c, s = quant(gpu, dev(x), q4mi.T_F32, 160, len(ids), 160, block, dev(ids))
    want = ref.quant(x[ids], block)
    assert np.array_equal(host(c), want[0]) and np.array_equal(host(s), want[1])


@pytest.mark.parametrize("block", [1, 128])
def test_quant_past_one_group(gpu, block):
    """Blocks past one group of rows of a launch, and codes past 32-bit offsets
    (4.3 GB of them and more)."""
    cols, few = 4096 if block == 1 else 128, 32
    rows = ((32 << 24) // 32 if block == 1 else (1 << 24) * 128 // 64) + 300
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn((few, cols), device="cuda", generator=g).to(torch.bfloat16)
    # stretches of 128 rows of one row, so that both kinds of block have its scale
    pick = torch.randint(0, few, (-(-rows // 128),), dtype=torch.int32, device="cuda", generator=g)
    ids = pick.repeat_interleave(128)[:rows].contiguous()
    c0, s0 = quant(gpu, x, q4mi.T_BF16, cols, few, cols)
    c, s = quant(gpu, x, q4mi.T_BF16, cols, rows, cols, block, ids)
    assert c.numel() > 1 << 31
    assert torch.equal(s, s0[(ids if block == 1 else pick).long()])
    for r in range(0, rows, 1 << 18):
        assert torch.equal(c[r:r + (1 << 18)], c0[ids[r:r + (1 << 18)].long()]), r


@pytest.mark.parametrize("yt", sorted(TYPES))
@pytest.mark.parametrize("rows,cols,pad,shift,block", [
    (1, 1, 0, 0, 1), (5, 130, 3, 1, 1), (130, 384, 0, 0, 128), (7, 2047, 1, 0, 128)])
def test_dequant(gpu, yt, rows, cols, pad, shift, block):
    rng = np.random.default_rng(cols)
    nb = ref.blocks(cols)
    c = rng.integers(0, 127, (rows, nb * 128)) + 128 * rng.integers(0, 2, (rows, nb * 128))
    c = c.astype(np.uint8)
    s = rng.uniform(0.001, 2, (-(-rows // block), nb)).astype(np.float32)
    ids = rng.integers(0, rows, rows).astype(np.int32)
    ld = cols + pad
    flat = torch.full((rows * ld + shift,), 77.0, dtype=TYPES[yt], device="cuda")
    d = [dev(a) for a in (c, s, ids)]
    q4mi.check(gpu.q4mi_f8_dequant(d[0].data_ptr(), d[1].data_ptr(), d[2].data_ptr(), rows, cols,
                                   block, flat[shift:].data_ptr(), yt, ld), "dequant")
    y = flat[shift:].view(rows, ld)
    v = ref.values(c, s, cols, block)[ids].astype(np.float32)      # one rounding to fp32
    assert torch.equal(y[:, :cols], dev(v).to(TYPES[yt]))
    assert (y[:, cols:] == 77).all() and (flat[:shift] == 77).all()


# ----------------------------------------------------------------- products

def random_rows(rng, rows, cols, exact, block):
    """Codes, scales, values; exact: whole numbers to 8 and scales 1/4 .. 1."""
    nb, rb = ref.blocks(cols), -(-rows // block)
    if exact:
        c = ref.encode(rng.integers(-8, 9, (rows, nb * 128)).astype(np.float64))
        s = np.exp2(rng.integers(-2, 1, (rb, nb)))
    else:
        c = ref.encode(rng.standard_normal((rows, nb * 128)) * 60)
        s = rng.uniform(0.5, 2, (rb, nb)) * np.exp2(rng.integers(-9, -6, (rb, nb)))
    c[:, cols:] = 0
    s = s.astype(np.float32)
    return c, s, ref.values(c, s, cols, block)


class Output:
    """Rows with a gap behind each, and what they should hold."""

    def __init__(self, rows, cols, yt, ld):
        self.yt, self.ld, self.cols = yt, ld, cols
        self.y = torch.full((rows, ld), 77.0, dtype=TYPES[yt], device="cuda")
        self.want = np.full((rows, ld), 77.0)
        self.room = np.zeros((rows, ld))

    def set(self, p, v, room):
        self.want[p, :self.cols] = v
        self.room[p, :self.cols] = room

    def check(self):
        y = host(self.y.double())
        t = TYPES[self.yt]
        want = host(dev(self.want).to(t).double())
        if not self.room.any():
            assert np.array_equal(y, want)
        else:
            room = self.room + torch.finfo(t).eps / 2 * (np.abs(self.want) + self.room)
            left = self.room == 0
            bad = np.where(left, y != want, np.abs(y - self.want) > room)
            assert not bad.any(), (np.argwhere(bad)[:5], np.abs(y - self.want).max())


def room_of(wv, xv, cols, exact):
    """How far fp32 sums may be off (see above)."""
    if exact:
        return np.zeros((len(xv), len(wv)))
    return (2 * 128 + 2 + ref.blocks(cols) + 32) * 2.0 ** -24 * (np.abs(xv) @ np.abs(wv).T)


@pytest.mark.parametrize("exact", [True, False])
@pytest.mark.parametrize("n,rows,cols,yt", [
    (1, 1, 1, 0), (1, 16, 128, 0), (1, 17, 129, 1), (2, 100, 1000, 30), (3, 2048, 2048, 0),
    (8, 130, 640, 1), (16, 300, 384, 0), (17, 300, 384, 30), (15, 33, 8192, 0), (31, 1000, 640, 0),
    (32, 64, 2176, 30), (33, 250, 256, 0), (64, 513, 128, 1), (65, 128, 1280, 0),
    (100, 1030, 900, 30), (128, 256, 512, 0), (129, 700, 2048, 30), (256, 256, 256, 0),
    (300, 2600, 130, 1), (520, 1290, 384, 30), (1, 5, 16384, 0), (20, 40, 16000, 0),
    (700, 5000, 256, 30), (1100, 4100, 640, 30)])
def test_mul(gpu, n, rows, cols, yt, exact):
    rng = np.random.default_rng(n + rows + cols)
    w, ws, wv = random_rows(rng, rows, cols, exact, 128)
    x, xs, xv = random_rows(rng, n, cols, exact, 1)
    out = Output(n, rows, yt, rows + 3)
    out.set(slice(None), xv @ wv.T, room_of(wv, xv, cols, exact))
    d = [dev(a) for a in (w, ws, x, xs)]
    for _ in range(2):
        q4mi.check(gpu.q4mi_f8_mul(d[0].data_ptr(), d[1].data_ptr(), rows, cols, d[2].data_ptr(),
                                   d[3].data_ptr(), F8, 0, n, out.y.data_ptr(), yt, out.ld), "mul")
        out.check()


@pytest.mark.parametrize("xt", sorted(TYPES))
@pytest.mark.parametrize("n,rows,cols,pad", [
    (1, 2048, 2048, 0), (1, 17, 100, 1), (3, 64, 1000, 3), (16, 130, 640, 0), (9, 5, 8200, 1)])
def test_mul_float_rows(gpu, xt, n, rows, cols, pad):
    """Float rows are quantised on the way in: the same bits as codes give, and
    codes and scales as the quantiser's."""
    rng = np.random.default_rng(n * cols)
    w, ws, wv = random_rows(rng, rows, cols, False, 128)
    ld = cols + pad
    x = dev(rng.standard_normal((n, ld)) * 3).to(TYPES[xt])
    c, s = quant(gpu, x, xt, ld, n, cols)
    xv = ref.values(host(c), host(s), cols)
    out = Output(n, rows, 0, rows)
    out.set(slice(None), xv @ wv.T, room_of(wv, xv, cols, False))
    dw, ds = dev(w), dev(ws)
    q4mi.check(gpu.q4mi_f8_mul(dw.data_ptr(), ds.data_ptr(), rows, cols, x.data_ptr(), None, xt, ld,
                               n, out.y.data_ptr(), 0, rows), "mul")
    out.check()
    y = torch.empty((n, rows), device="cuda")
    q4mi.check(gpu.q4mi_f8_mul(dw.data_ptr(), ds.data_ptr(), rows, cols, c.data_ptr(), s.data_ptr(),
                               F8, 0, n, y.data_ptr(), 0, rows), "mul")
    assert torch.equal(y, out.y)


@pytest.mark.parametrize("n,rows,cols", [(2, 40, 256), (40, 200, 256), (300, 300, 384)])
def test_mul_nan_stays_in_its_row(gpu, n, rows, cols):
    """A block of x without finite values makes its row NaN, a block of W's
    scales that is NaN its 128 outputs; the others are as they were."""
    rng = np.random.default_rng(n)
    w, ws, wv = random_rows(rng, rows, cols, True, 128)
    x, xs, xv = random_rows(rng, n, cols, True, 1)
    want = xv @ wv.T
    xs[n // 2, 1] = np.nan
    x[n // 2, 128:256] = 0
    want[n // 2] = np.nan
    ws[-1, 0] = np.nan
    want[:, (rows - 1) // 128 * 128:] = np.nan
    y = torch.empty((n, rows), device="cuda")
    d = [dev(a) for a in (w, ws, x, xs)]
    q4mi.check(gpu.q4mi_f8_mul(d[0].data_ptr(), d[1].data_ptr(), rows, cols, d[2].data_ptr(),
                               d[3].data_ptr(), F8, 0, n, y.data_ptr(), 0, rows), "mul")
    assert np.array_equal(host(y), want.astype(np.float32), equal_nan=True)


def experts(rng, E, rows, cols, exact):
    """Experts at strides of their own, with bytes of another kind between."""
    nb, rb = ref.blocks(cols), -(-rows // 128)
    wst, sst = rows * nb * 128 + 48, rb * nb * 4 + 12
    w = np.full((E, wst), 0x7f, np.uint8)
    ws = np.full((E, sst // 4), np.nan, np.float32)
    wv = []
    for e in range(E):
        c, s, v = random_rows(rng, rows, cols, exact, 128)
        w[e, :wst - 48], ws[e, :rb * nb] = c.reshape(-1), s.reshape(-1)
        wv.append(v)
    return dev(w), dev(ws), wst, sst, wv


@pytest.mark.parametrize("exact", [True, False])
@pytest.mark.parametrize("tokens,topk,E,rows,cols,div,yt", [
    (1, 10, 16, 1024, 2048, 10, 0), (4, 10, 64, 130, 512, 1, 0), (8, 3, 4, 33, 100, 3, 30),
    (1, 1, 1, 1, 1, 1, 1), (37, 2, 3, 200, 640, 2, 0), (300, 2, 5, 17, 130, 1, 0)])
def test_sel(gpu, tokens, topk, E, rows, cols, div, yt, exact):
    rng = np.random.default_rng(tokens + rows)
    n = tokens * topk
    w, ws, wst, sst, wv = experts(rng, E, rows, cols, exact)
    x, xs, xv = random_rows(rng, -(-n // div), cols, exact, 1)
    eid = rng.integers(0, E, n)
    if n > 4:
        eid[n // 2:n // 2 + 3] = [-1, E, -(1 << 31)]
    out = Output(n, rows, yt, rows + 1)
    for p in range(n):
        if 0 <= eid[p] < E:
            v = xv[p // div:p // div + 1]
            out.set(p, (v @ wv[eid[p]].T)[0], room_of(wv[eid[p]], v, cols, exact)[0])
    d = [dev(a) for a in (x, xs, eid.astype(np.int32))]
    q4mi.check(gpu.q4mi_f8_mul_sel(w.data_ptr(), ws.data_ptr(), rows, cols, wst, sst, E,
                                   d[0].data_ptr(), d[1].data_ptr(), F8, 0, div, d[2].data_ptr(),
                                   n, out.y.data_ptr(), yt, out.ld), "sel")
    out.check()


@pytest.mark.parametrize("xt", sorted(TYPES))
@pytest.mark.parametrize("n,E,div", [(10, 16, 10), (40, 512, 1), (100, 3, 2)])
def test_sel_float_rows(gpu, xt, n, E, div):
    rng = np.random.default_rng(n)
    rows, cols, ld = 96, 700, 703
    w, ws, wst, sst, wv = experts(rng, E, rows, cols, False)
    xr = -(-n // div)
    x = dev(rng.standard_normal((xr, ld))).to(TYPES[xt])
    c, s = quant(gpu, x, xt, ld, xr, cols)
    eid = dev(rng.integers(0, E, n).astype(np.int32))
    got = []
    for p, b, t in ((x, None, xt), (c, s, F8)):
        y = torch.zeros((n, rows), device="cuda")
        q4mi.check(gpu.q4mi_f8_mul_sel(w.data_ptr(), ws.data_ptr(), rows, cols, wst, sst, E,
                                       p.data_ptr(), q4mi.ptr(b), t, ld, div, eid.data_ptr(), n,
                                       y.data_ptr(), 0, rows), "sel")
        got.append(y)
    assert torch.equal(*got)
    xv = ref.values(host(c), host(s), cols)
    for p in range(n):
        e, v = int(eid[p]), xv[p // div:p // div + 1]
        off = np.abs(host(got[0][p].double()) - (v @ wv[e].T)[0])
        want = np.abs(v @ wv[e].T)[0]
        room = room_of(wv[e], v, cols, False)[0]
        assert (off <= room + 2.0 ** -24 * (want + room)).all()


@pytest.mark.parametrize("exact", [True, False])
@pytest.mark.parametrize("counts,rows,cols,yt,gather", [
    ([3], 16, 128, 0, True), ([0, 1, 0, 16, 17, 0], 130, 300, 0, True),
    ([40, 0, 7, 129, 64, 65, 1], 300, 640, 30, True), ([5, 5], 33, 1, 1, False),
    ([300, 20, 0, 33], 520, 256, 30, False), ([0, 0, 0], 16, 128, 0, True),
    ([1] * 60 + [700], 64, 384, 0, True), ([257, 1, 128, 32, 31], 1100, 1000, 30, True),
    ([600, 300, 90, 2], 2048, 130, 0, True)])
def test_id(gpu, counts, rows, cols, yt, gather, exact):
    """Stretches that begin past row 0 and end before the last row, activation
    rows that do not exist."""
    rng = np.random.default_rng(rows + cols)
    E, first, spare = len(counts), 2, 3
    w, ws, wst, sst, wv = experts(rng, E, rows, cols, exact)
    bounds = np.concatenate([[0], np.cumsum(counts)]) + first
    total = int(bounds[-1]) + spare
    xrows = max(1, total // 3 if gather else total - 4)
    x, xs, xv = random_rows(rng, xrows, cols, exact, 1)
    act = rng.integers(0, xrows, total) if gather else np.arange(total)
    if gather:
        bad = rng.permutation(total)[:total // 20]
        act[bad] = rng.choice([-1, -(1 << 31), xrows, (1 << 31) - 1], len(bad))
    out = Output(total, rows, yt, rows + 5)
    for e in range(E):
        p = np.arange(bounds[e], bounds[e + 1])
        p = p[(act[p] >= 0) & (act[p] < xrows)]
        if len(p):
            v = xv[act[p]]
            out.set(p, v @ wv[e].T, room_of(wv[e], v, cols, exact))
    d = [dev(a) for a in (x, xs, act.astype(np.int32), bounds.astype(np.int32))]
    for _ in range(2):
        q4mi.check(gpu.q4mi_f8_mul_id(w.data_ptr(), ws.data_ptr(), rows, cols, wst, sst, E,
                                      d[0].data_ptr(), d[1].data_ptr(), xrows,
                                      d[2].data_ptr() if gather else None, d[3].data_ptr(), total,
                                      out.y.data_ptr(), yt, out.ld), "id")
        out.check()


def test_last_stretch_says_more_than_there_is(gpu):
    """bounds past total_rows end there."""
    rng = np.random.default_rng(1)
    rows, cols, total = 40, 256, 37
    w, ws, wst, sst, wv = experts(rng, 2, rows, cols, True)
    x, xs, xv = random_rows(rng, total, cols, True, 1)
    d = [dev(a) for a in (x, xs, np.array([0, 20, 90], np.int32))]
    out = Output(total + 2, rows, 0, rows)
    out.set(slice(0, 20), xv[:20] @ wv[0].T, 0)
    out.set(slice(20, total), xv[20:] @ wv[1].T, 0)
    q4mi.check(gpu.q4mi_f8_mul_id(w.data_ptr(), ws.data_ptr(), rows, cols, wst, sst, 2,
                                  d[0].data_ptr(), d[1].data_ptr(), total, None, d[2].data_ptr(),
                                  total, out.y.data_ptr(), 0, rows), "id")
    out.check()


def test_places_past_32_bits(gpu):
    """Experts 3 GiB apart, output rows that begin past 2^32 elements."""
    rng = np.random.default_rng(2)
    E, rows, cols, far, ld = 3, 40, 200, 3 << 30, (1 << 31) + 1
    nb = ref.blocks(cols)
    w = torch.empty(2 * far + rows * nb * 128, dtype=torch.uint8, device="cuda")
    ws = torch.empty(2 * far // 4 + nb, device="cuda")
    wv = []
    for e in range(E):
        c, s, v = random_rows(rng, rows, cols, True, 128)
        w[e * far:][:c.size], ws[e * far // 4:][:s.size] = dev(c).view(-1), dev(s).view(-1)
        wv.append(v)
    x, xs, xv = random_rows(rng, E, cols, True, 1)
    flat = torch.zeros(2 * ld + rows, dtype=torch.float16, device="cuda")
    y = torch.as_strided(flat, (E, rows), (ld, 1))
    want = torch.stack([dev(wv[e] @ xv[e]) for e in range(E)]).half()
    d = [dev(a) for a in (x, xs, np.arange(E + 1, dtype=np.int32))]
    arena = (w.data_ptr(), ws.data_ptr(), rows, cols, far, far, E, d[0].data_ptr(), d[1].data_ptr())
    q4mi.check(gpu.q4mi_f8_mul_sel(*arena, F8, 0, 1, d[2].data_ptr(), E, flat.data_ptr(), 1, ld),
               "sel")
    assert torch.equal(y, want)
    y.zero_()
    q4mi.check(gpu.q4mi_f8_mul_id(*arena, E, None, d[2].data_ptr(), E, flat.data_ptr(), 1, ld),
               "id")
    assert torch.equal(y, want)
    want = dev(xv @ wv[0].T).half()
    for n in (2, 3):
        y.zero_()
        q4mi.check(gpu.q4mi_f8_mul(w.data_ptr(), ws.data_ptr(), rows, cols, d[0].data_ptr(),
                                   d[1].data_ptr(), F8, 0, n, flat.data_ptr(), 1, ld), "mul")
        assert torch.equal(y[:n], want[:n])
