"""q4mi_rms_norm against its formula in 64 bits.

h is exact up to its one rounding.  i = fp32(1 / sqrt(..)) of a 64-bit sum is off
by 2^-24 relative (and some 2^-50), y = (h * i) * w by two more roundings: at
most 3.1 * 2^-24 |y| before the rounding to its type.  The 8-bit codes are those
of the fp32 y of the same call, exactly."""
import numpy as np
import pytest
import torch

import f8_ref as ref
import q4mi

pytestmark = pytest.mark.gpu

TYPES = {0: torch.float32, 1: torch.float16, 30: torch.bfloat16}
F8, Q8 = q4mi.T_F8, q4mi.T_Q8_0


def host(t):
    return t.cpu().numpy()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def norm(L, x, xt, ldx, res, sum_, rt, ldr, w, wt, eps, rows, cols, y, yt, ldy, qt=0, c=None,
         s=None):
    q4mi.check(L.q4mi_rms_norm(q4mi.ptr(x), xt, ldx, q4mi.ptr(res), q4mi.ptr(sum_), rt, ldr,
                               q4mi.ptr(w), wt, eps, rows, cols, q4mi.ptr(y), yt, ldy, qt,
                               q4mi.ptr(c), q4mi.ptr(s)), "norm")


def room(c, cols, qt, rows):
    """Codes and scales to be written over."""
    if qt == F8:
        nb = ref.blocks(cols)
        return (torch.full((rows, nb * 128), 0xcd, dtype=torch.uint8, device="cuda"),
                torch.full((rows, nb), -7.0, device="cuda"))
    return (torch.full((rows, cols), 0x5d, dtype=torch.int8, device="cuda"),
            torch.full((rows, cols // 32), -7.0, device="cuda"))


SHAPES = [(1, 1), (3, 31), (5, 128), (2, 129), (9, 512), (4, 513), (1, 2048), (33, 2560),
          (7, 2049), (3, 8192), (2, 8200), (2, 20000), (1, 32768), (3, 40000), (2, 32776)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("xt,rt,wt,yt", [(0, 0, 0, 0), (30, 30, 0, 30), (30, 0, 30, 0),
                                         (1, 30, 1, 1), (0, 1, 30, 30)])
@pytest.mark.parametrize("with_res", [True, False])
def test_norm(gpu, rows, cols, xt, rt, wt, yt, with_res):
    g = gen(rows * cols)
    rnd = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    ldx, ldr, ldy = cols + 3, cols + 1, cols + 2
    x, w = (3 * rnd(rows, ldx)).to(TYPES[xt]), (1 + 0.3 * rnd(cols)).to(TYPES[wt])
    h, res, sum_ = x[:, :cols].double(), None, None
    if with_res:
        res = rnd(rows, ldr).to(TYPES[rt])
        h = x[:, :cols].float() + res[:, :cols].float()
    if with_res or cols % 2:
        sum_ = torch.full((rows, ldr), 77.0, dtype=TYPES[rt], device="cuda")
        h = h.to(TYPES[rt]).double()
    eps = float(np.float32(1e-5))
    want = h / torch.sqrt((h * h).mean(1, keepdim=True) + eps) * w.double()
    y = torch.full((rows, ldy), 77.0, dtype=TYPES[yt], device="cuda")
    norm(gpu, x, xt, ldx, res, sum_, rt, ldr, w, wt, eps, rows, cols, y, yt, ldy)
    if sum_ is not None:
        assert torch.equal(sum_[:, :cols].double(), h)
        assert (sum_[:, cols:] == 77).all()
    off = 3.1 * 2.0 ** -24 * want.abs()
    off += (want.abs() + off) * torch.finfo(TYPES[yt]).eps / 2
    if yt == 1:
        off += 2.0 ** -25       # subnormals of fp16: half their step
    assert ((y[:, :cols].double() - want).abs() <= off).all()
    assert (y[:, cols:] == 77).all()
    # codes of the same fp32 y, with and without y beside them
    y32 = torch.empty((rows, cols), device="cuda")
    for qt in (F8, Q8) if cols % 32 == 0 else (F8,):
        c, s = room(None, cols, qt, rows)
        norm(gpu, x, xt, ldx, res, None, rt, ldr, w, wt, eps, rows, cols, y32, 0, cols, qt, c, s)
        if qt == F8 and (sum_ is None or with_res):
            wc, wsc = ref.quant(host(y32))
            assert np.array_equal(host(c), wc) and np.array_equal(host(s), wsc)
        elif qt == Q8:
            q, d = room(None, cols, Q8, rows)
            q4mi.check(gpu.q4mi_quant8(y32.data_ptr(), None, rows, cols, q.data_ptr(),
                                       d.data_ptr(), None), "quant8")
            assert torch.equal(c, q) and torch.equal(s, d)
        c2, s2 = room(None, cols, qt, rows)
        norm(gpu, x, xt, ldx, res, None, rt, ldr, w, wt, eps, rows, cols, None, 0, 0, qt, c2, s2)
        assert torch.equal(c, c2) and torch.equal(s, s2)


@pytest.mark.parametrize("cols", [100, 2048, 5000, 40000])
@pytest.mark.parametrize("t", sorted(TYPES))
def test_in_place(gpu, cols, t):
    """sum over the residual, y over x; without a residual sum over x."""
    g, rows = gen(cols), 5
    x = torch.randn((rows, cols), device="cuda", generator=g).to(TYPES[t])
    r = torch.randn((rows, cols), device="cuda", generator=g).to(TYPES[t])
    w = torch.randn(cols, device="cuda", generator=g)
    s, y = torch.empty_like(r), torch.empty_like(x)
    norm(gpu, x, t, cols, r, s, t, cols, w, 0, 1e-6, rows, cols, y, t, cols)
    x1, r1 = x.clone(), r.clone()
    norm(gpu, x1, t, cols, r1, r1, t, cols, w, 0, 1e-6, rows, cols, x1, t, cols)
    assert torch.equal(r1, s) and torch.equal(x1, y)
    x2 = x.clone()
    norm(gpu, x2, t, cols, r, x2, t, cols, w, 0, 1e-6, rows, cols, y, t, cols)
    assert torch.equal(x2, s) and torch.equal(x1, y)


@pytest.mark.parametrize("cols", [128, 2048, 40000])
def test_no_weight_zero_rows_and_non_finite(gpu, cols):
    x = torch.ones((4, cols), device="cuda")
    x[0] = 0
    x[1, 5], x[2, cols - 1] = float("inf"), float("nan")
    y = torch.empty_like(x)
    c, s = room(None, cols, F8, 4)
    norm(gpu, x, 0, cols, None, None, 0, 0, None, 0, 1e-6, 4, cols, y, 0, cols, F8, c, s)
    y, c, s = host(y), host(c), host(s)
    assert (y[0] == 0).all() and (c[0] == 0).all() and (s[0] == 2.0 ** -120).all()
    assert np.isnan(y[1, 5]) and (np.delete(y[1], 5) == 0).all()     # 1 / inf = 0
    assert np.isnan(s[1, 0]) and not np.isnan(s[1, 1:]).any() and (c[1] == 0).all()
    assert np.isnan(y[2]).all() and np.isnan(s[2]).all() and (c[2] == 0).all()
    assert np.abs(y[3] - 1 / np.sqrt(1 + 1e-6)).max() <= 3.1 * 2.0 ** -24
    # huge and tiny values: squares that no fp32 holds
    x = torch.tensor([1e30, 1e-30], device="cuda")[:, None].expand(2, cols).contiguous()
    y = torch.empty_like(x)
    norm(gpu, x, 0, cols, None, None, 0, 0, None, 0, 0.0, 2, cols, y, 0, cols)
    assert (y - 1).abs().max() <= 3.1 * 2.0 ** -24


def test_no_rows(gpu):
    norm(gpu, None, 0, 64, None, None, 0, 0, None, 0, 1e-6, 0, 64, None, 0, 64)


def test_many_rows(gpu):
    """Rows past the first launch dimension (2^20 workgroups of four)."""
    rows, cols = (1 << 22) + 7, 32
    x = torch.randn((rows, cols), device="cuda", generator=gen(1)).to(torch.bfloat16)
    y = torch.empty_like(x)
    norm(gpu, x, 30, cols, None, None, 0, 0, None, 0, 1e-6, rows, cols, y, 30, cols)
    v = x.double()
    want = v / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-6)
    assert ((y.double() - want).abs() <= (2.0 ** -8 + 4 * 2.0 ** -24) * want.abs()).all()


@pytest.mark.parametrize("cols", [512, 513, 1024, 1030, 1536, 2048, 2049, 2100, 3000, 4800, 5900,
                                  6400, 7168, 8190, 9000, 10240, 11000, 12289, 13000, 14336, 15400,
                                  16384, 16385, 20000, 32768, 32769])
def test_every_number_of_waves(gpu, cols):
    """Rows of one wave to sixteen, one to four chunks a lane, and beyond."""
    g, rows = gen(cols), 6
    x = torch.randn((rows, cols), device="cuda", generator=g).to(torch.bfloat16)
    r = torch.randn((rows, cols), device="cuda", generator=g)
    w = torch.randn(cols, device="cuda", generator=g)
    s, y = torch.empty_like(r), torch.empty_like(r)
    c, sc = room(None, cols, F8, rows)
    norm(gpu, x, 30, cols, r, s, 0, cols, w, 0, 1e-6, rows, cols, y, 0, cols, F8, c, sc)
    h = x.float() + r
    assert torch.equal(s, h)
    h = h.double()
    want = h / torch.sqrt((h * h).mean(1, keepdim=True) + float(np.float32(1e-6))) * w.double()
    assert ((y.double() - want).abs() <= 3.1 * 2.0 ** -24 * want.abs()).all()
    wc, wsc = ref.quant(host(y))
    assert np.array_equal(host(c), wc) and np.array_equal(host(sc), wsc)
