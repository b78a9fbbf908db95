"""Microscaled 4-bit quantisation and products on the GPU, against the
format's definition in 64 bits (mx4_ref).

Codes and scales are exact.  Products come in two kinds of data:
  - scales within a factor of 4 and rows up to 4096 values, where every
    partial sum in any order is a whole multiple of 2^-4 below 2^20 (36 * 4 *
    4096 < 2^20), so fp32 sums are exact and y must be the 64-bit result;
  - any data: at most cols + 1 additions in whatever order, each off by at
    most 2^-23 of a partial sum that is at most S = sum |w x| (2^-24 if it is
    to nearest; hardware sums may cut off), then one rounding to the type.
"""
import ctypes

import numpy as np
import pytest
import torch

import mx4_ref as ref
import q4mi

pytestmark = pytest.mark.gpu

TYPES = {q4mi.T_F32: torch.float32, q4mi.T_F16: torch.float16, q4mi.T_BF16: torch.bfloat16}
MX4 = q4mi.T_MXFP4


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def host(t):
    return t.cpu().numpy()


def quant(L, x, xt, ld, rows, cols, ids=None):
    nb = ref.blocks(cols)
    c = torch.full((rows, nb * 16), 0xcd, dtype=torch.uint8, device="cuda")
    s = torch.full((rows, ref.scale_row(cols)), 0xcd, dtype=torch.uint8, device="cuda")
    q4mi.check(L.q4mi_mx4_quant(x.data_ptr(), xt, ld, q4mi.ptr(ids), rows, cols, c.data_ptr(),
                                s.data_ptr()), "quant")
    return c, s


# ------------------------------------------------------------- quantisation

@pytest.mark.parametrize("xt", sorted(TYPES))
@pytest.mark.parametrize("rows,cols,pad,shift", [
    (1, 1, 0, 0), (1, 31, 0, 0), (3, 32, 0, 0), (2, 33, 3, 1), (5, 100, 28, 0), (1, 2048, 0, 0),
    (7, 129, 7, 0), (65, 512, 0, 0), (64, 2560, 8, 0), (19, 1013, 1, 3)])
def test_quant_exact(gpu, xt, rows, cols, pad, shift):
    rng = np.random.default_rng(rows * 1000 + cols)
    ld = cols + pad
    v = rng.standard_normal((rows, ld)) * np.exp2(rng.integers(-20, 9, (rows, ld)))
    v[rng.random((rows, ld)) < 0.05] = 0
    flat = torch.zeros(rows * ld + shift, dtype=TYPES[xt], device="cuda")
    flat[shift:] = dev(v.reshape(-1)).to(TYPES[xt])
    x = flat[shift:]
    c, s = quant(gpu, x, xt, ld, rows, cols)
    want = ref.quant(host(x.double()).reshape(rows, ld)[:, :cols])
    assert np.array_equal(host(c), want[0])
    assert np.array_equal(host(s), want[1])


def test_quant_every_boundary(gpu):
    """Every tie and its neighbours at every scale, subnormals and the largest
    values included."""
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0], np.float32)
    near = np.concatenate([ties, np.nextafter(ties, np.float32(0)),
                           np.nextafter(ties, np.float32(9))])
    block = np.zeros(32, np.float32)
    block[:27] = near
    block[27] = 4.0
    block[28:] = [-0.25, -0.0, 1e-30, -5.0]
    x = np.stack([np.ldexp(block, e) for e in range(-148, 126)]).astype(np.float32)
    assert np.isfinite(x).all()
    d = dev(x)
    c, s = quant(gpu, d, q4mi.T_F32, 32, len(x), 32)
    want = ref.quant(x)
    assert np.array_equal(host(s), want[1])
    assert np.array_equal(host(c), want[0])


def test_quant_non_finite(gpu):
    x = np.ones((4, 96), np.float32)
    x[0, 5], x[1, 40], x[2, 95], x[2, 0] = np.inf, np.nan, -np.inf, np.nan
    for xt, t in TYPES.items():
        c, s = quant(gpu, dev(x).to(t), xt, 96, 4, 96)
        want = ref.quant(x)
        assert np.array_equal(host(s), want[1]) and np.array_equal(host(c), want[0])
        y = torch.empty((4, 96), device="cuda")
        q4mi.check(gpu.q4mi_mx4_dequant(c.data_ptr(), s.data_ptr(), None, 4, 96, y.data_ptr(), 0,
                                        96), "dequant")
        assert np.array_equal(np.isnan(host(y)), np.isnan(ref.values(*want, 96)))


def test_quant_gather_and_repeat(gpu):
    rng = np.random.default_rng(5)
    x = rng.standard_normal((9, 160)).astype(np.float32)
    ids = np.array([8, 0, 0, 3, 8, 8, 1], np.int32)
    c, s = quant(gpu, dev(x), q4mi.T_F32, 160, len(ids), 160, dev(ids))
    want = ref.quant(x[ids])
    assert np.array_equal(host(c), want[0]) and np.array_equal(host(s), want[1])


def test_quant_past_one_group(gpu):
    """More than 2^29 blocks, 8.6 GB of codes: past one group of rows and past
    32-bit offsets."""
    cols, few = 16384, 64
    rows = (1 << 29) // (cols // 32) + 300
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn((few, cols), device="cuda", generator=g).to(torch.bfloat16)
    ids = torch.randint(0, few, (rows,), dtype=torch.int32, device="cuda", generator=g)
    c0, s0 = quant(gpu, x, q4mi.T_BF16, cols, few, cols)
    c, s = quant(gpu, x, q4mi.T_BF16, cols, rows, cols, ids)
    for r in range(0, rows, 1 << 16):
        i = ids[r:r + (1 << 16)].long()
        assert torch.equal(c[r:r + (1 << 16)], c0[i]) and torch.equal(s[r:r + (1 << 16)], s0[i]), r


@pytest.mark.parametrize("yt", sorted(TYPES))
@pytest.mark.parametrize("rows,cols,pad,shift", [
    (1, 1, 0, 0), (3, 40, 0, 0), (17, 257, 7, 1), (64, 2048, 8, 0), (5, 96, 1, 0)])
def test_dequant_exact(gpu, yt, rows, cols, pad, shift):
    """Values rounded once to the type; columns past cols untouched."""
    rng = np.random.default_rng(rows + cols)
    c, s = ref.random_rows(rng, rows + 2, cols, 0, 254)
    s[0, 0] = 255
    ids = rng.integers(0, rows + 2, rows).astype(np.int32)
    ids[0] = 0
    ld = cols + pad
    y = torch.full((rows * ld + shift,), -7.0, dtype=TYPES[yt], device="cuda")
    dc, ds, di = dev(c), dev(s), dev(ids)
    q4mi.check(gpu.q4mi_mx4_dequant(dc.data_ptr(), ds.data_ptr(), di.data_ptr(), rows, cols,
                                    y[shift:].data_ptr(), yt, ld), "dequant")
    got = host(y[shift:].double()).reshape(rows, ld)
    with np.errstate(over="ignore"):
        want = host(torch.from_numpy(ref.values(c, s, cols)[ids]).float().to(TYPES[yt]).double())
    assert np.array_equal(got[:, :cols], want, equal_nan=True)
    assert (got[:, cols:] == -7).all() and (host(y[:shift].float()) == -7).all()


# ----------------------------------------------------------------- products

def tol(cols, s, y, t):
    """See the head of the file; t's rounding is half a step of |y|, or half
    the smallest subnormal."""
    f = torch.finfo(t)
    return (cols + 1) * 2.0 ** -23 * s + np.abs(y) * f.eps / 2 + f.smallest_normal * f.eps / 2


def close(got, y, s, cols, t):
    got = host(got.double())
    assert (np.abs(got - y) <= tol(cols, s, y, t)).all(), \
        np.nanmax(np.abs(got - y) / tol(cols, s, y, t))


SIZES = [(1, 1, 1), (1, 16, 32), (1, 2048, 2048), (3, 130, 96), (8, 33, 4096), (9, 64, 160),
         (16, 100, 640), (17, 257, 1013), (31, 48, 33), (64, 512, 2560), (77, 300, 352),
         (128, 128, 128), (130, 260, 288), (257, 513, 1024), (300, 1000, 96), (512, 768, 544)]


@pytest.mark.parametrize("n,rows,cols", SIZES)
def test_mul_exact(gpu, n, rows, cols):
    """Sums that fp32 holds exactly: y is the 64-bit result."""
    rng = np.random.default_rng(n * 7 + rows)
    w, ws = ref.random_rows(rng, rows, cols, 126, 128)
    x, xs = ref.random_rows(rng, n, cols, 126, 128)
    want = ref.values(x, xs, cols) @ ref.values(w, ws, cols).T
    ld = rows + 3
    y = torch.full((n + 1, ld), -7.0, device="cuda")
    d = [dev(a) for a in (w, ws, x, xs)]
    q4mi.check(gpu.q4mi_mx4_mul(d[0].data_ptr(), d[1].data_ptr(), rows, cols, d[2].data_ptr(),
                                d[3].data_ptr(), MX4, 0, n, y.data_ptr(), 0, ld), "mul")
    got = host(y)
    assert np.array_equal(got[:n, :rows], want)
    assert (got[n:] == -7).all() and (got[:, rows:] == -7).all()


@pytest.mark.parametrize("n,rows,cols", [
    (700, 5000, 352), (700, 5000, 2080), (1300, 5000, 800), (1300, 5000, 256), (2100, 5000, 96),
    (2100, 5000, 1056), (2309, 4609, 544), (20, 20000, 608), (32, 9000, 1024)])
def test_mul_large_tiles(gpu, n, rows, cols):
    """Sizes that fill the chip with each of the larger tiles, none of them
    whole, with whole and partial stages of K; sums exact in fp32.  The torch
    product in fp64 on the device is the reference."""
    g = torch.Generator(device="cuda").manual_seed(n + cols)
    nb = ref.blocks(cols)

    def rand(r):
        c = torch.randint(0, 256, (r, nb * 16), dtype=torch.uint8, device="cuda", generator=g)
        s = torch.zeros((r, ref.scale_row(cols)), dtype=torch.uint8, device="cuda")
        s[:, :nb] = torch.randint(126, 129, (r, nb), dtype=torch.uint8, device="cuda", generator=g)
        t = torch.tensor(np.concatenate([ref.LEVELS, -ref.LEVELS]), device="cuda")
        v = torch.stack([t[(c & 15).long()], t[(c >> 4).long()]], 2).view(r, nb, 32)
        return c, s, (v * torch.exp2(s[:, :nb].double() - 127)[..., None]).view(r, nb * 32)

    w, ws, wv = rand(rows)
    x, xs, xv = rand(n)
    want = xv @ wv.t()
    y = torch.full((n + 1, rows + 4), -7.0, device="cuda")
    q4mi.check(gpu.q4mi_mx4_mul(w.data_ptr(), ws.data_ptr(), rows, cols, x.data_ptr(),
                                xs.data_ptr(), MX4, 0, n, y.data_ptr(), 0, rows + 4), "mul")
    assert torch.equal(y[:n, :rows].double(), want)
    assert bool((y[n:] == -7).all()) and bool((y[:, rows:] == -7).all())


@pytest.mark.parametrize("n,rows,cols", [(1, 50, 16384), (8, 40, 8224), (16, 70, 9000),
                                         (16, 5000, 4128), (40, 64, 16000), (300, 260, 8192)])
def test_mul_long_rows(gpu, n, rows, cols):
    """Rows of many K segments; one scale, so sums are multiples of 1/4 below
    36 * 16384 < 2^20: exact."""
    rng = np.random.default_rng(cols)
    w, ws = ref.random_rows(rng, rows, cols, 127, 127)
    x, xs = ref.random_rows(rng, n, cols, 127, 127)
    want = ref.values(x, xs, cols) @ ref.values(w, ws, cols).T
    y = torch.empty((n, rows), device="cuda")
    d = [dev(a) for a in (w, ws, x, xs)]
    q4mi.check(gpu.q4mi_mx4_mul(d[0].data_ptr(), d[1].data_ptr(), rows, cols, d[2].data_ptr(),
                                d[3].data_ptr(), MX4, 0, n, y.data_ptr(), 0, rows), "mul")
    assert np.array_equal(host(y), want)


@pytest.mark.parametrize("yt", sorted(TYPES))
@pytest.mark.parametrize("n,rows,cols", [(1, 64, 2048), (5, 100, 333), (40, 200, 640),
                                         (200, 384, 1024), (260, 270, 2560)])
def test_mul_types(gpu, yt, n, rows, cols):
    """Normal data of any scale to each output type, odd row strides."""
    rng = np.random.default_rng(n + rows + yt)
    w, ws = ref.quant(rng.standard_normal((rows, cols)) / np.sqrt(cols))
    x, xs = ref.quant(rng.standard_normal((n, cols)) * np.exp2(rng.integers(-6, 6, (n, 1))))
    wv, xv = ref.values(w, ws, cols), ref.values(x, xs, cols)
    ld = rows + 1
    y = torch.full((n, ld), -7.0, dtype=TYPES[yt], device="cuda")
    d = [dev(a) for a in (w, ws, x, xs)]
    q4mi.check(gpu.q4mi_mx4_mul(d[0].data_ptr(), d[1].data_ptr(), rows, cols, d[2].data_ptr(),
                                d[3].data_ptr(), MX4, 0, n, y.data_ptr(), yt, ld), "mul")
    close(y[:, :rows], xv @ wv.T, np.abs(xv) @ np.abs(wv).T, cols, TYPES[yt])
    assert (host(y[:, rows:].float()) == -7).all()


@pytest.mark.parametrize("xt", sorted(TYPES))
@pytest.mark.parametrize("n,rows,cols,pad", [(1, 64, 2048, 0), (1, 100, 1, 0), (8, 128, 640, 8),
                                             (5, 37, 77, 5), (3, 4000, 2560, 0), (8, 16, 8192, 0)])
def test_mul_float_rows(gpu, xt, n, rows, cols, pad):
    """Float activations: the bits of quantising them first."""
    rng = np.random.default_rng(n + rows)
    ld = cols + pad
    x = dev(rng.standard_normal((n, ld))).to(TYPES[xt])
    w, ws = (dev(a) for a in ref.quant(rng.standard_normal((rows, cols))))
    c, s = quant(gpu, x, xt, ld, n, cols)
    y = torch.empty((2, n, rows), device="cuda")
    q4mi.check(gpu.q4mi_mx4_mul(w.data_ptr(), ws.data_ptr(), rows, cols, x.data_ptr(), None, xt,
                                ld, n, y[0].data_ptr(), 0, rows), "float rows")
    q4mi.check(gpu.q4mi_mx4_mul(w.data_ptr(), ws.data_ptr(), rows, cols, c.data_ptr(),
                                s.data_ptr(), MX4, 0, n, y[1].data_ptr(), 0, rows), "codes")
    y = host(y)
    assert np.array_equal(y[0], y[1])


@pytest.mark.parametrize("n,rows,cols", [(1, 40, 96), (8, 40, 2048), (40, 300, 352),
                                         (300, 300, 512)])
def test_mul_nan_blocks(gpu, n, rows, cols):
    """A NaN block makes its row's products NaN, and no others."""
    rng = np.random.default_rng(3)
    w, ws = ref.random_rows(rng, rows, cols, 126, 128)
    x, xs = ref.random_rows(rng, n, cols, 126, 128)
    ws[7, 1] = ws[rows - 1, 0] = 255
    ws[:, ref.blocks(cols):] = 255          # bytes past the last block mean nothing
    xs[:, ref.blocks(cols):] = 255
    xs[n // 2, 2] = 255
    want = ref.values(x, xs, cols) @ ref.values(w, ws, cols).T
    y = torch.empty((n, rows), device="cuda")
    d = [dev(a) for a in (w, ws, x, xs)]
    q4mi.check(gpu.q4mi_mx4_mul(d[0].data_ptr(), d[1].data_ptr(), rows, cols, d[2].data_ptr(),
                                d[3].data_ptr(), MX4, 0, n, y.data_ptr(), 0, rows), "mul")
    assert np.array_equal(host(y), want, equal_nan=True)


def test_mul_extreme_scales(gpu):
    """Scales at both ends: exact products where fp32 holds them, zeros below
    its range, infinities above."""
    cols, rows = 64, 16
    c = np.full((1, 32), 0x22, np.uint8)                  # all ones
    for sw, sx in ((254, 0), (0, 254), (1, 200), (127, 20), (200, 60), (254, 127), (90, 60)):
        w, ws = np.repeat(c, rows, 0), np.full((rows, 4), sw, np.uint8)
        d = [dev(a) for a in (w, ws, c, np.full((1, 4), sx, np.uint8))]
        y = torch.empty((1, rows), device="cuda")
        q4mi.check(gpu.q4mi_mx4_mul(d[0].data_ptr(), d[1].data_ptr(), rows, cols, d[2].data_ptr(),
                                    d[3].data_ptr(), MX4, 0, 1, y.data_ptr(), 0, rows), "mul")
        with np.errstate(over="ignore"):
            want = np.float32(64 * 2.0 ** (sw + sx - 254))
        assert (host(y) == want).all(), (sw, sx, host(y)[0, 0], want)


# ------------------------------------------------------------ routed experts

def arena(rng, experts, rows, cols, lo=126, hi=128):
    w, ws = ref.random_rows(rng, experts * rows, cols, lo, hi)
    v = ref.values(w, ws, cols).reshape(experts, rows, cols)
    return dev(w), dev(ws), v, rows * w.shape[1], rows * ws.shape[1]


@pytest.mark.parametrize("tokens,topk,experts,rows,cols,div", [
    (1, 10, 16, 64, 256, 10), (4, 3, 8, 100, 96, 3), (8, 8, 512, 17, 33, 1), (1, 1, 1, 16, 32, 1),
    (2, 10, 32, 1024, 2048, 10), (5, 2, 4, 250, 640, 1), (1, 2, 3, 64, 8192, 2)])
def test_mul_sel_exact(gpu, tokens, topk, experts, rows, cols, div):
    rng = np.random.default_rng(tokens * topk + rows)
    w, ws, wv, st, sst = arena(rng, experts, rows, cols)
    n = tokens * topk
    x, xs = ref.random_rows(rng, (n + div - 1) // div, cols, 126, 128)
    xv = ref.values(x, xs, cols)
    eid = rng.integers(0, experts, n).astype(np.int32)
    eid[n // 2:n // 2 + 2] = [-1, experts][:len(eid[n // 2:n // 2 + 2])]
    want = np.full((n, rows + 2), -7.0)
    for p in range(n):
        if 0 <= eid[p] < experts:
            want[p, :rows] = wv[eid[p]] @ xv[p // div]
    dx, dxs, de = dev(x), dev(xs), dev(eid)
    fx = dev(xv.astype(np.float32))
    for a, b, t in ((dx, dxs, MX4), (fx, None, q4mi.T_F32)):
        if t == q4mi.T_F32 and cols % 32 == 0:
            # the float rows are values of the format, but their own scales may differ
            q, s = ref.quant(xv)
            if not np.array_equal(ref.values(q, s, cols), xv):
                continue
        y = torch.full((n, rows + 2), -7.0, device="cuda")
        q4mi.check(gpu.q4mi_mx4_mul_sel(w.data_ptr(), ws.data_ptr(), rows, cols, st, sst, experts,
                                        a.data_ptr(), q4mi.ptr(b), t, cols, div, de.data_ptr(), n,
                                        y.data_ptr(), 0, rows + 2), "sel")
        assert np.array_equal(host(y), want)


@pytest.mark.parametrize("xt", sorted(TYPES))
def test_mul_sel_float_rows(gpu, xt):
    """Float rows give the bits of quantised ones."""
    rng = np.random.default_rng(11)
    experts, rows, cols, tokens, topk = 12, 200, 1000, 6, 5
    w, ws, _, st, sst = arena(rng, experts, rows, cols)
    x = dev(rng.standard_normal((tokens, cols + 4))).to(TYPES[xt])
    c, s = quant(gpu, x, xt, cols + 4, tokens, cols)
    eid = dev(rng.integers(0, experts, tokens * topk).astype(np.int32))
    y = torch.empty((2, tokens * topk, rows), device="cuda")
    for i, (a, b, t) in enumerate(((x, None, xt), (c, s, MX4))):
        q4mi.check(gpu.q4mi_mx4_mul_sel(w.data_ptr(), ws.data_ptr(), rows, cols, st, sst, experts,
                                        a.data_ptr(), q4mi.ptr(b), t, cols + 4, topk,
                                        eid.data_ptr(), tokens * topk, y[i].data_ptr(), 0, rows),
                   "sel")
    y = host(y)
    assert np.array_equal(y[0], y[1])


@pytest.mark.parametrize("n,experts,rows,cols,div", [
    (600, 3, 40, 96, 1), (40, 1, 50, 352, 1), (257, 2, 33, 32, 4), (300, 1000, 20, 64, 1),
    (17, 4, 64, 4096, 17), (256, 1, 16, 512, 8)])
def test_mul_sel_shared_experts(gpu, n, experts, rows, cols, div):
    """Lists past 256 rows, many rows of one expert, rows of none between
    them: codes give the 64-bit result, float rows the bits of their codes."""
    rng = np.random.default_rng(n + experts)
    w, ws, wv, st, sst = arena(rng, experts, rows, cols)
    xr = (n + div - 1) // div
    x, xs = ref.random_rows(rng, xr, cols, 126, 128)
    xv = ref.values(x, xs, cols)
    eid = rng.integers(0, experts, n).astype(np.int32)
    eid[::7] = -1
    eid[3] = experts
    want = np.full((n, rows + 1), -7.0)
    for p in range(n):
        if 0 <= eid[p] < experts:
            want[p, :rows] = wv[eid[p]] @ xv[p // div]
    de = dev(eid)
    f = dev(rng.standard_normal((xr, cols))).to(torch.bfloat16)
    c, s = quant(gpu, f, q4mi.T_BF16, cols, xr, cols)
    y = torch.full((3, n, rows + 1), -7.0, device="cuda")
    sides = ((dev(x), dev(xs), MX4), (f, None, q4mi.T_BF16), (c, s, MX4))
    for i, (a, b, t) in enumerate(sides):
        q4mi.check(gpu.q4mi_mx4_mul_sel(w.data_ptr(), ws.data_ptr(), rows, cols, st, sst, experts,
                                        a.data_ptr(), q4mi.ptr(b), t, cols, div, de.data_ptr(), n,
                                        y[i].data_ptr(), 0, rows + 1), "sel")
    y = host(y)
    assert np.array_equal(y[0], want)
    assert np.array_equal(y[1], y[2])


@pytest.mark.parametrize("counts,rows,cols,spare", [
    ([0, 5, 0, 17], 64, 96, 3), ([40], 33, 32, 0), ([1] * 20, 100, 640, 0), ([0, 0], 16, 32, 4),
    ([130, 0, 300, 7, 64, 65], 272, 288, 9), ([500, 1], 1024, 512, 0),
    ([33, 260, 31], 520, 2048, 1), ([3] * 64, 200, 1013, 2),
    ([32, 33, 31, 64, 16, 17], 90, 416, 0), ([1, 0, 2] * 341 + [5], 20, 64, 3),
    ([20, 150], 50, 9000, 0), ([129] * 3, 600, 1056, 0)])
@pytest.mark.parametrize("gather", [True, False])
def test_mul_id_exact(gpu, counts, rows, cols, spare, gather):
    """Ragged stretches, empty experts, rows that no stretch covers."""
    rng = np.random.default_rng(sum(counts) + rows)
    experts, total = len(counts), sum(counts)
    # long rows keep one scale, so that their sums stay exact
    w, ws, wv, st, sst = arena(rng, experts, rows, cols, 126 if cols <= 4096 else 127,
                               128 if cols <= 4096 else 127)
    n = total + spare
    xrows = max(1, total // 3) if gather else max(n, 1)
    x, xs = ref.random_rows(rng, xrows, cols, 126 if cols <= 4096 else 127,
                            128 if cols <= 4096 else 127)
    xv = ref.values(x, xs, cols)
    bounds = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    act = rng.integers(0, xrows, n).astype(np.int32) if gather else np.arange(n, dtype=np.int32)
    if gather and total > 4:
        act[1], act[total - 1] = -1, xrows
    want = np.full((n, rows + 5), -7.0)
    for e in range(experts):
        for p in range(bounds[e], bounds[e + 1]):
            if 0 <= act[p] < xrows:
                want[p, :rows] = wv[e] @ xv[act[p]]
    y = torch.full((n, rows + 5), -7.0, device="cuda")
    d = [dev(a) for a in (x, xs, act, bounds)]
    q4mi.check(gpu.q4mi_mx4_mul_id(w.data_ptr(), ws.data_ptr(), rows, cols, st, sst, experts,
                                   d[0].data_ptr(), d[1].data_ptr(), xrows,
                                   d[2].data_ptr() if gather else None, d[3].data_ptr(), n,
                                   y.data_ptr(), 0, rows + 5), "id")
    assert np.array_equal(host(y), want)


def test_mul_id_fewer_activations_than_rows(gpu):
    """Without a row list, packed rows past xrows are left as they were."""
    rng = np.random.default_rng(21)
    counts, rows, cols, xrows = [70, 90, 40], 40, 96, 100
    w, ws, wv, st, sst = arena(rng, 3, rows, cols)
    x, xs = ref.random_rows(rng, xrows, cols, 126, 128)
    xv = ref.values(x, xs, cols)
    bounds = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    n = sum(counts)
    e = np.repeat(np.arange(3), counts)
    want = np.full((n, rows), -7.0)
    for p in range(xrows):
        want[p] = wv[e[p]] @ xv[p]
    y = torch.full((n, rows), -7.0, device="cuda")
    d = [dev(a) for a in (x, xs, bounds)]
    q4mi.check(gpu.q4mi_mx4_mul_id(w.data_ptr(), ws.data_ptr(), rows, cols, st, sst, 3,
                                   d[0].data_ptr(), d[1].data_ptr(), xrows, None, d[2].data_ptr(),
                                   n, y.data_ptr(), 0, rows), "id")
    assert np.array_equal(host(y), want)


@pytest.mark.parametrize("yt", [q4mi.T_F16, q4mi.T_BF16])
def test_mul_id_types(gpu, yt):
    rng = np.random.default_rng(8)
    counts, rows, cols = [70, 0, 9, 200], 130, 320
    w, ws, wv, st, sst = arena(rng, 4, rows, cols)
    total = sum(counts)
    x, xs = ref.random_rows(rng, total, cols, 120, 124)
    xv = ref.values(x, xs, cols)
    bounds = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    y = torch.empty((total, rows), dtype=TYPES[yt], device="cuda")
    d = [dev(a) for a in (x, xs, bounds)]
    q4mi.check(gpu.q4mi_mx4_mul_id(w.data_ptr(), ws.data_ptr(), rows, cols, st, sst, 4,
                                   d[0].data_ptr(), d[1].data_ptr(), total, None, d[2].data_ptr(),
                                   total, y.data_ptr(), yt, rows), "id")
    e = np.repeat(np.arange(4), counts)
    want = np.einsum("prc,pc->pr", wv[e], xv)
    s = np.einsum("prc,pc->pr", np.abs(wv[e]), np.abs(xv))
    close(y, want, s, cols, TYPES[yt])


# ---------------------------------------------------- a layer and its logits

def test_layer_to_logits(gpu):
    """The operators as an engine runs them: router, pack, 4-bit experts of a
    prompt and of its last token alone, LM head, processed logits, top-k.  Each
    step is checked against 64 bits on what the step before it gave."""
    L, rng = gpu, np.random.default_rng(31)
    T, E, K, H, F, V = 150, 12, 3, 256, 96, 500
    t = lambda *n, dtype=torch.float32: torch.zeros(n, dtype=dtype, device="cuda")  # noqa: E731
    i32, u8 = torch.int32, torch.uint8
    x = dev(rng.standard_normal((T, H)).astype(np.float32))
    wr = dev(rng.standard_normal((E, H)).astype(np.float32) / 16)
    gu = [dev(a) for a in ref.quant(rng.standard_normal((E * 2 * F, H)) / 16)]
    dn = [dev(a) for a in ref.quant(rng.standard_normal((E * H, F)) / 10)]
    lm = [dev(a) for a in ref.quant(rng.standard_normal((V, H)) / 16)]
    guv = ref.values(*map(host, gu), H).reshape(E, 2 * F, H)
    dnv = ref.values(*map(host, dn), F).reshape(E, H, F)
    lmv = ref.values(*map(host, lm), H)

    def experts(w, rows, cols):
        return (w[0].data_ptr(), w[1].data_ptr(), rows, cols, rows * w[0].shape[1],
                rows * w[1].shape[1], E)

    logits, ids, wts = t(T, E), t(T, K, dtype=i32), t(T, K)
    q4mi.check(L.q4mi_moe_route(wr.data_ptr(), 0, None, x.data_ptr(), T, H, E, K,
                                logits.data_ptr(), ids.data_ptr(), wts.data_ptr(), None, K, -1,
                                None), "route")
    R = T * K
    atok, rsrc, rw, bounds = t(R, dtype=i32), t(R, dtype=i32), t(R), t(E + 1, dtype=i32)
    stg, stgn, ek = t(512, dtype=i32), t(1, dtype=i32), t(512, dtype=i32)
    q4mi.check(L.q4mi_assign(ids.data_ptr(), wts.data_ptr(), atok.data_ptr(), rsrc.data_ptr(),
                             rw.data_ptr(), stg.data_ptr(), stgn.data_ptr(), ek.data_ptr(),
                             bounds.data_ptr(), T, K, E, T), "pack")
    xq, xs = quant(L, x, 0, H, T, H)
    g, h, pd, y = t(R, 2 * F), t(R, F), t(R, H), t(T, H)
    q4mi.check(L.q4mi_mx4_mul_id(*experts(gu, 2 * F, H), xq.data_ptr(), xs.data_ptr(), T,
                                 atok.data_ptr(), bounds.data_ptr(), R, g.data_ptr(), 0, 2 * F),
               "gate/up")
    q4mi.check(L.q4_mmq_swiglu(g.data_ptr(), h.data_ptr(), R, F), "swiglu")
    hq, hs = quant(L, h, 0, F, R, F)
    q4mi.check(L.q4mi_mx4_mul_id(*experts(dn, H, F), hq.data_ptr(), hs.data_ptr(), R, None,
                                 bounds.data_ptr(), R, pd.data_ptr(), 0, H), "down")
    q4mi.check(L.q4_hip_expert_reduce(y.data_ptr(), pd.data_ptr(), rsrc.data_ptr(), rw.data_ptr(),
                                      T, K, H), "reduce")
    e = np.repeat(np.arange(E), np.diff(host(bounds)))
    xv = ref.values(*ref.quant(host(x)), H)[host(atok)]
    close(g, np.einsum("prc,pc->pr", guv[e], xv), np.einsum("prc,pc->pr", abs(guv[e]), abs(xv)), H,
          torch.float32)
    want = ref.quant(host(h))
    assert np.array_equal(host(hq), want[0]) and np.array_equal(host(hs), want[1])
    hv = ref.values(*want, F)
    close(pd, np.einsum("prc,pc->pr", dnv[e], hv), np.einsum("prc,pc->pr", abs(dnv[e]), abs(hv)),
          F, torch.float32)

    # the last token alone, as a decode step: float rows in, the router's list
    one = x[T - 1:]
    g1, h1, d1 = t(K, 2 * F), t(K, F), t(K, H)
    q4mi.check(L.q4mi_mx4_mul_sel(*experts(gu, 2 * F, H), one.data_ptr(), None, 0, H, K,
                                  ids[T - 1].data_ptr(), K, g1.data_ptr(), 0, 2 * F), "gate/up")
    q4mi.check(L.q4_mmq_swiglu(g1.data_ptr(), h1.data_ptr(), K, F), "swiglu")
    q4mi.check(L.q4mi_mx4_mul_sel(*experts(dn, H, F), h1.data_ptr(), None, 0, F, 1,
                                  ids[T - 1].data_ptr(), K, d1.data_ptr(), 0, H), "down")
    pick = host(ids)[T - 1]
    xv1 = ref.values(*ref.quant(host(one)), H)[0]
    close(g1, guv[pick] @ xv1, abs(guv[pick]) @ abs(xv1), H, torch.float32)
    hv1 = ref.values(*ref.quant(host(h1)), F)
    close(d1, np.einsum("prc,pc->pr", dnv[pick], hv1),
          np.einsum("prc,pc->pr", abs(dnv[pick]), abs(hv1)), F, torch.float32)
    at = host(rsrc).reshape(T, K)[T - 1]
    # the same rows of the prompt's pass, where no sum came out another way
    same = np.array_equal(host(g)[at], host(g1))
    if same:
        assert np.array_equal(ref.quant(host(h)[at])[0], ref.quant(host(h1))[0])

    # LM head on the last two tokens, penalties and a mask, then the best token
    z, out = t(2, V), t(2, V)
    q4mi.check(L.q4mi_mx4_mul(lm[0].data_ptr(), lm[1].data_ptr(), V, H, y[T - 2:].data_ptr(), None,
                              0, H, 2, z.data_ptr(), 0, V), "LM head")
    yv = ref.values(*ref.quant(host(y[T - 2:])), H)
    close(z, yv @ lmv.T, abs(yv) @ abs(lmv).T, H, torch.float32)
    best = host(z).argmax(1)
    hist, off = dev(best.astype(np.int32)), dev(np.array([0, 1, 2], np.int64))
    pen = dev(np.array([[1.0, 100.0, 0.0], [1.0, 0.0, 0.0]], np.float32))
    mask = np.full((1, (V + 31) // 32), 0xffffffff, np.uint32)
    mask[0, best[1] // 32] &= ~np.uint32(1 << (best[1] % 32))
    dm, dr = dev(mask.view(np.int32)), dev(np.array([-1, 0], np.int32))
    q4mi.check(L.q4mi_logits_process(z.data_ptr(), 0, V, 2, V, hist.data_ptr(), off.data_ptr(),
                                     None, pen.data_ptr(), None, None, None, dm.data_ptr(),
                                     mask.shape[1], 1, dr.data_ptr(), out.data_ptr(), V), "logits")
    zh, got = host(z), host(out)
    # tokens the model wrote count from the start of the history without gen
    want = zh.copy()
    want[0, best[0]] = np.float32(zh[0, best[0]] - np.float32(100))
    want[1, best[1]] = -np.inf
    assert np.array_equal(got, want)
    top, tw = t(2, 1, dtype=i32), t(2, 1)
    q4mi.check(L.q4_hip_route_pf(out.data_ptr(), top.data_ptr(), tw.data_ptr(), 2, V, 1), "top-k")
    assert np.array_equal(host(top)[:, 0], want.argmax(1))


# ---------------------------------------------------------- streams and graphs

def test_two_streams_and_graphs(gpu):
    """Two captured sequences replayed on two streams at once, over and over:
    each gives what it gives alone."""
    rng = np.random.default_rng(9)
    n, rows, cols, experts = 64, 500, 1056, 5
    w, ws, _, st, sst = arena(rng, experts, rows, cols)
    bounds = dev(np.array([0, 3, 40, 40, 41, 64], np.int32))
    eid = dev(rng.integers(0, experts, n).astype(np.int32))
    x = [dev(rng.standard_normal((n, cols)).astype(np.float32)) for _ in range(2)]
    c = torch.empty((2, n, ref.blocks(cols) * 16), dtype=torch.uint8, device="cuda")
    s = torch.empty((2, n, ref.scale_row(cols)), dtype=torch.uint8, device="cuda")
    y = torch.zeros((2, 3, n, rows), device="cuda")

    def calls(i):
        q4mi.use_torch_stream()
        q4mi.check(gpu.q4mi_mx4_quant(x[i].data_ptr(), 0, cols, None, n, cols, c[i].data_ptr(),
                                      s[i].data_ptr()), "quant")
        q4mi.check(gpu.q4mi_mx4_mul(w.data_ptr(), ws.data_ptr(), rows, cols, c[i].data_ptr(),
                                    s[i].data_ptr(), MX4, 0, n, y[i, 0].data_ptr(), 0, rows), "mul")
        q4mi.check(gpu.q4mi_mx4_mul_sel(w.data_ptr(), ws.data_ptr(), rows, cols, st, sst, experts,
                                        x[i].data_ptr(), None, 0, cols, 1, eid.data_ptr(), n,
                                        y[i, 1].data_ptr(), 0, rows), "sel")
        q4mi.check(gpu.q4mi_mx4_mul_id(w.data_ptr(), ws.data_ptr(), rows, cols, st, sst, experts,
                                       c[i].data_ptr(), s[i].data_ptr(), n, None,
                                       bounds.data_ptr(), n, y[i, 2].data_ptr(), 0, rows), "id")

    streams = [torch.cuda.Stream() for _ in range(2)]
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    calls(0), calls(1)
    torch.cuda.synchronize()
    want = y.clone()
    assert not torch.equal(want[0], want[1])
    try:
        for i in range(2):
            with torch.cuda.graph(graphs[i], stream=streams[i]):
                calls(i)
        for eager in (False, True, False):
            y.zero_()
            torch.cuda.synchronize()
            for _ in range(4):
                for i in range(2):
                    with torch.cuda.stream(streams[i]):
                        if eager:
                            calls(i)
                        else:
                            graphs[i].replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want), eager
    finally:
        q4mi.use_torch_stream()


def test_mx4_graph_and_stream(gpu):
    """Captured on a stream of its own and replayed with other inputs, eager
    calls between: every replay is the eager result."""
    rng = np.random.default_rng(4)
    n, rows, cols, experts = 40, 300, 640, 6
    w, ws, _, st, sst = arena(rng, experts, rows, cols)
    x = torch.empty((n, cols), device="cuda")
    c = torch.empty((n, ref.blocks(cols) * 16), dtype=torch.uint8, device="cuda")
    s = torch.empty((n, ref.scale_row(cols)), dtype=torch.uint8, device="cuda")
    bounds = dev(np.array([0, 1, 1, 20, 33, 33, 40], np.int32))
    eid = dev(rng.integers(0, experts, n).astype(np.int32))
    y = torch.zeros((3, n, rows), device="cuda")

    def calls():
        q4mi.check(gpu.q4mi_mx4_quant(x.data_ptr(), 0, cols, None, n, cols, c.data_ptr(),
                                      s.data_ptr()), "quant")
        q4mi.check(gpu.q4mi_mx4_mul(w.data_ptr(), ws.data_ptr(), rows, cols, c.data_ptr(),
                                    s.data_ptr(), MX4, 0, n, y[0].data_ptr(), 0, rows), "mul")
        q4mi.check(gpu.q4mi_mx4_mul_sel(w.data_ptr(), ws.data_ptr(), rows, cols, st, sst, experts,
                                        x.data_ptr(), None, 0, cols, 1, eid.data_ptr(), n,
                                        y[1].data_ptr(), 0, rows), "sel")
        q4mi.check(gpu.q4mi_mx4_mul_id(w.data_ptr(), ws.data_ptr(), rows, cols, st, sst, experts,
                                       c.data_ptr(), s.data_ptr(), n, None, bounds.data_ptr(), n,
                                       y[2].data_ptr(), 0, rows), "id")

    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    x.copy_(dev(rng.standard_normal((n, cols)).astype(np.float32)))
    torch.cuda.synchronize()
    try:
        with torch.cuda.stream(side):
            q4mi.use_torch_stream()
            calls()
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            q4mi.use_torch_stream()
            calls()
    finally:
        q4mi.use_torch_stream()
    for i in range(4):
        x.copy_(dev(rng.standard_normal((n, cols)).astype(np.float32)))
        calls()
        torch.cuda.synchronize()
        want = y.clone()
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want), i
        assert float(want.abs().sum()) > 0
