"""Refusals of the 4-bit and logits entry points (host checks, no GPU), and
the format's reference against its definition."""
import numpy as np
import pytest

import mx4_ref as ref
import q4mi

F32, F16, BF16, MX4 = q4mi.T_F32, q4mi.T_F16, q4mi.T_BF16, q4mi.T_MXFP4
A = 1 << 20     # an aligned address that no refused call touches


def refused(ok, text):
    assert not ok
    assert text in q4mi.last_error(), q4mi.last_error()


def test_sizes():
    L = q4mi.lib()
    for rows, cols in ((1, 1), (3, 32), (5, 33), (7, 129), (2, 2048)):
        assert L.q4mi_mx4_code_bytes(rows, cols) == rows * ref.blocks(cols) * 16
        assert L.q4mi_mx4_scale_bytes(rows, cols) == rows * ref.scale_row(cols)


def test_reference_format():
    """Every code's value, the ties, the cap and the scale of known blocks."""
    x = np.zeros((1, 32))
    x[0, :15] = [4, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 7.99, -0.25, -6, 0.2500001, 0.7499, 6.5,
                 -5]
    c, s = ref.quant(x)
    v = ref.values(c, s, 32)[0]
    assert s[0, 0] == 127
    assert v[:15].tolist() == [4, 0, 1, 1, 2, 2, 4, 4, 6, 0, -6, 0.5, 0.5, 6, -4]
    assert ref.quant(np.full((1, 32), 8.0))[1][0, 0] == 128
    assert ref.quant(np.full((1, 5), np.inf))[1][0, 0] == 255
    assert ref.quant(np.zeros((1, 5)))[1][0].tolist() == [0, 0, 0, 0]


def test_quant_refusals():
    L = q4mi.lib()
    for f, name in ((L.q4mi_mx4_quant, "quant"), (L.q4mi_mx4_dequant, "dequant")):
        def call(fl=A, ty=F32, ld=64, rows=2, cols=64, c=A, s=A, f=f, name=name):
            return f(fl, ty, ld, None, rows, cols, c, s) if name == "quant" else \
                f(c, s, None, rows, cols, fl, ty, ld)
        refused(call(fl=None), "bad arguments")
        refused(call(c=None), "bad arguments")
        refused(call(s=None), "bad arguments")
        refused(call(cols=0), "bad arguments")
        refused(call(ty=q4mi.T_Q8_0), "type 8")
        refused(call(ty=MX4), "type 39")
        refused(call(ld=63), "row stride")
        refused(call(fl=A + 2), "aligned")
        refused(call(fl=A + 1, ty=F16), "aligned")
        refused(call(c=A + 8), "aligned")
        refused(call(s=A + 2), "aligned")
        refused(call(cols=1 << 31, ld=1 << 31), "too large")
        refused(call(rows=1 << 33), "too large")
        assert call(rows=0)


@pytest.mark.parametrize("which", ["mul", "sel", "id"])
def test_product_refusals(which):
    L = q4mi.lib()

    def call(w=A, ws=A, rows=64, cols=64, wst=4096, wsst=256, ne=4, x=A, xs=A, xt=MX4, ldx=64,
             div=1, eid=A, n=4, xrows=4, bounds=A, y=A, yt=F32, ldy=64):
        if which == "mul":
            return L.q4mi_mx4_mul(w, ws, rows, cols, x, xs, xt, ldx, n, y, yt, ldy)
        if which == "sel":
            return L.q4mi_mx4_mul_sel(w, ws, rows, cols, wst, wsst, ne, x, xs, xt, ldx, div, eid,
                                      n, y, yt, ldy)
        return L.q4mi_mx4_mul_id(w, ws, rows, cols, wst, wsst, ne, x, xs, xrows, None, bounds, n,
                                 y, yt, ldy)

    for k in ("w", "ws", "x", "y"):
        refused(call(**{k: None}), "bad arguments")
    refused(call(rows=0, ldy=0), "bad arguments")
    refused(call(cols=0), "bad arguments")
    refused(call(cols=(1 << 24) + 32), "sizes")
    refused(call(rows=(1 << 30) + 1, ldy=1 << 31), "sizes")
    refused(call(n=(1 << 30) + 1), "sizes")
    refused(call(yt=MX4), "types")
    refused(call(yt=q4mi.T_Q8_0), "types")
    refused(call(w=A + 8), "aligned")
    refused(call(ws=A + 1), "aligned")
    refused(call(x=A + 4), "aligned")
    refused(call(xs=None), "scales")
    refused(call(y=A + 2), "aligned")
    refused(call(y=A + 1, yt=BF16), "aligned")
    refused(call(ldy=63), "stride")
    assert call(n=0)
    if which != "mul":
        refused(call(wst=4100), "aligned")
        refused(call(wsst=258), "aligned")
        refused(call(ne=0), "experts")
    if which == "sel":
        refused(call(eid=None), "list")
        refused(call(div=0), "x_div")
        refused(call(n=65536), "65535")
    if which == "id":
        refused(call(bounds=None), "bounds")
        refused(call(ne=1025), "bounds")
        assert call(xrows=0)
        return
    refused(call(xt=q4mi.T_Q8_0), "types")
    refused(call(xt=F32), "scales")                       # float rows with scales
    refused(call(xt=F32, xs=None, ldx=63), "stride")
    refused(call(xt=F32, xs=None, x=A + 2), "alignment")
    if which == "mul":
        refused(call(xt=F32, xs=None, n=9), "float rows")


def test_calls_without_rows():
    """An empty batch's pointers may be NULL, as an empty tensor's are."""
    L = q4mi.lib()
    assert L.q4mi_mx4_quant(None, F32, 64, None, 0, 64, None, None), q4mi.last_error()
    assert L.q4mi_mx4_dequant(None, None, None, 0, 64, None, F32, 64), q4mi.last_error()
    for x_type in (MX4, F32):
        assert L.q4mi_mx4_mul(A, A, 64, 64, None, None, x_type, 64, 0, None, F32, 64), \
            q4mi.last_error()
        assert L.q4mi_mx4_mul_sel(A, A, 64, 64, 4096, 256, 4, None, None, x_type, 64, 1, None, 0,
                                  None, F32, 64), q4mi.last_error()
    for n, xrows in ((0, 0), (0, 4), (4, 0)):
        assert L.q4mi_mx4_mul_id(A, A, 64, 64, 4096, 256, 4, None, None, xrows, None, A, n, None,
                                 F32, 64), q4mi.last_error()
    assert L.q4mi_logits_process(None, F32, 100, 0, 100, None, A, None, None, None, None, A, None,
                                 0, 0, None, None, 100), q4mi.last_error()


def test_logits_refusals():
    L = q4mi.lib()

    def call(x=A, ty=F32, ld=100, n=2, v=100, hist=A, hoff=A, gen=None, pen=A, bid=A, bias=A,
             boff=A, mask=A, mld=4, nm=2, mrow=None, out=2 * A, ldo=100):
        return L.q4mi_logits_process(x, ty, ld, n, v, hist, hoff, gen, pen, bid, bias, boff, mask,
                                     mld, nm, mrow, out, ldo)

    refused(call(x=None), "bad arguments")
    refused(call(out=None), "bad arguments")
    refused(call(v=0), "bad arguments")
    refused(call(v=(1 << 30) + 1), "bad arguments")
    refused(call(ty=MX4), "type 39")
    refused(call(ld=99), "strides")
    refused(call(ldo=99), "strides")
    refused(call(out=A, ldo=101), "strides")
    refused(call(x=A + 2), "aligned")
    refused(call(out=A + 1, ty=F16), "aligned")
    refused(call(pen=None), "penalties")
    refused(call(hoff=None), "penalties")
    refused(call(pen=None, hoff=None), "penalties")       # a history alone
    refused(call(pen=None, hoff=None, hist=None, gen=A), "penalties")
    refused(call(bid=None), "biases")
    refused(call(bias=None), "biases")
    refused(call(boff=None), "biases")
    refused(call(mld=3), "masks")
    refused(call(nm=0), "masks")
    refused(call(nm=1), "masks")                          # one mask for two rows, no rows named
    refused(call(mask=None, mrow=A), "masks")
    refused(call(n=(1 << 32) - 1, v=1 << 20, ld=1 << 20, ldo=1 << 20, mld=1 << 15, mrow=A),
            "too large")
    refused(call(n=1 << 24, mrow=A), "too large")         # 2^24 workgroups of 512 threads
    assert call(n=0)
