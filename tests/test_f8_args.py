"""Refusals of the 8-bit floating point, norm and scored routing entry points
(host checks, no GPU), and their reference against the definitions."""
import math

import numpy as np
import pytest

import f8_ref as ref
import q4mi

F32, F16, BF16, F8 = q4mi.T_F32, q4mi.T_F16, q4mi.T_BF16, q4mi.T_F8
A = 1 << 20     # an aligned address that no refused call touches


def refused(ok, text):
    assert not ok
    assert text in q4mi.last_error(), q4mi.last_error()


def test_sizes():
    L = q4mi.lib()
    for rows, cols in ((1, 1), (3, 128), (5, 129), (7, 2048), (300, 2500)):
        nb = ref.blocks(cols)
        assert L.q4mi_f8_code_bytes(rows, cols) == rows * nb * 128
        assert L.q4mi_f8_scale_bytes(rows, cols, 1) == rows * nb * 4
        assert L.q4mi_f8_scale_bytes(rows, cols, 128) == -(-rows // 128) * nb * 4
    assert L.q4mi_f8_scale_bytes(5, 5, 0) == 0


def test_reference_format():
    """Codes of known values, ties, the largest; scales at their borders."""
    assert ref.level([0, 1, 8, 0x38, 0x7e, 0xfe]).tolist() == [0, 2.0 ** -9, 2.0 ** -6, 1, 448,
                                                               -448]
    v = [1.0625, 1.1875, 2.0 ** -10, 3 * 2.0 ** -10, 17.0, 447.9, -1.1]
    assert ref.level(ref.encode(np.array(v))).tolist() == [1, 1.25, 0, 2.0 ** -8, 16, 448, -1.125]
    x = np.zeros((4, 128))
    x[0, 3], x[1, 3], x[2, 3] = 448, np.nextafter(np.float32(448), np.float32(449)), 3.5
    assert ref.quant(x)[1][:, 0].tolist() == [1, 2, 2.0 ** -7, 2.0 ** -120]
    c, s = ref.quant(x, 128)
    assert s.shape == (1, 1) and s[0, 0] == 2 and ref.level(c[0, 3]) == 224


def test_reference_routing():
    z = [[1.0, 3.0, 3.0, -math.inf, 0.0, math.nan, 2.0, -1.0]]
    ids, w = ref.route(z, 3)
    assert ids.tolist() == [[1, 2, 6]] and abs(w.sum() - 1) < 1e-15
    ids, _ = ref.route(z, 4, 1, groups=4, keep=2, group_top=2)
    assert ids.tolist() == [[1, 6, 0, 7]]       # groups 0 (1, 3) and 3 (2, -1)
    ids, w = ref.route(z, 8, 1, bias=[0, 0, 9, 0, -9, 0, 0, 0], renorm=False)
    assert ids.tolist() == [[2, 1, 6, 0, 7, 4, -1, -1]]
    assert abs(w[0, 0] - 1 / (1 + math.exp(-3))) < 1e-15 and w[0, 6] == 0


def test_quant_refusals():
    L = q4mi.lib()
    for f, name in ((L.q4mi_f8_quant, "quant"), (L.q4mi_f8_dequant, "dequant")):
        def call(fl=A, ty=F32, ld=64, rows=2, cols=64, br=1, c=A, s=A, f=f, name=name):
            return f(fl, ty, ld, None, rows, cols, br, c, s) if name == "quant" else \
                f(c, s, None, rows, cols, br, fl, ty, ld)
        refused(call(fl=None), "bad arguments")
        refused(call(c=None), "bad arguments")
        refused(call(s=None), "bad arguments")
        refused(call(cols=0), "bad arguments")
        refused(call(ty=q4mi.T_Q8_0), "type 8")
        refused(call(ty=F8), "type 248")
        for br in (0, 2, 64, 129):
            refused(call(br=br), "rows a scale")
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

    def call(w=A, ws=A, rows=64, cols=64, wst=8192, wsst=256, ne=4, x=A, xs=A, xt=F8, ldx=64,
             div=1, eid=A, n=4, xrows=4, bounds=A, y=A, yt=F32, ldy=64):
        if which == "mul":
            return L.q4mi_f8_mul(w, ws, rows, cols, x, xs, xt, ldx, n, y, yt, ldy)
        if which == "sel":
            return L.q4mi_f8_mul_sel(w, ws, rows, cols, wst, wsst, ne, x, xs, xt, ldx, div, eid,
                                     n, y, yt, ldy)
        return L.q4mi_f8_mul_id(w, ws, rows, cols, wst, wsst, ne, x, xs, xrows, None, bounds, n,
                                y, yt, ldy)

    for k in ("w", "ws", "x", "y"):
        refused(call(**{k: None}), "bad arguments")
    refused(call(rows=0, ldy=0), "bad arguments")
    refused(call(cols=0), "bad arguments")
    refused(call(cols=(1 << 24) + 32), "sizes")
    refused(call(rows=(1 << 30) + 1, ldy=1 << 31), "sizes")
    refused(call(n=(1 << 30) + 1), "sizes")
    refused(call(yt=F8), "types")
    refused(call(yt=q4mi.T_Q8_0), "types")
    refused(call(w=A + 8), "aligned")
    refused(call(ws=A + 1), "aligned")
    refused(call(x=A + 4), "aligned")
    refused(call(xs=None), "scales")
    refused(call(y=A + 2), "aligned")
    refused(call(y=A + 1, yt=BF16), "aligned")
    refused(call(ldy=63), "stride")
    if which != "id":
        refused(call(xt=q4mi.T_MXFP4), "types")
        refused(call(xt=F32), "float inputs")               # with scales
        refused(call(xt=F32, xs=None, ldx=63), "float inputs")
        refused(call(xt=F16, xs=None, x=A + 1), "float inputs")
    if which == "mul":
        refused(call(xt=F32, xs=None, n=17), "quantise")
    else:
        refused(call(wst=8), "aligned")
        refused(call(wsst=2), "aligned")
        refused(call(ne=0), "experts")
    if which == "sel":
        refused(call(eid=None), "list")
        refused(call(div=0), "x_div")
        refused(call(n=65536), "65535")
    if which == "id":
        refused(call(bounds=None), "bounds")
        refused(call(ne=1025), "1024")
        assert call(xrows=0)
    assert call(n=0)
    assert call(n=0, x=None, xs=None if which != "mul" else A, y=None)


def test_norm_refusals():
    L = q4mi.lib()

    def call(x=A, xt=F32, ldx=64, res=None, sum_=None, rt=F32, ldr=64, w=A, wt=F32, eps=1e-6,
             rows=2, cols=64, y=A, yt=F32, ldy=64, qt=0, c=None, s=None):
        return L.q4mi_rms_norm(x, xt, ldx, res, sum_, rt, ldr, w, wt, eps, rows, cols, y, yt, ldy,
                               qt, c, s)
    refused(call(x=None), "bad arguments")
    refused(call(y=None), "bad arguments")
    refused(call(cols=0), "bad arguments")
    refused(call(c=A, qt=F8), "bad arguments")
    refused(call(s=A, qt=F8), "bad arguments")
    for k in ("xt", "wt", "yt"):
        refused(call(**{k: F8}), "types")
    refused(call(res=A, rt=8), "types")
    refused(call(sum_=A, rt=8), "types")
    refused(call(c=A, s=A), "8-bit type 0")
    refused(call(c=A, s=A, qt=q4mi.T_MXFP4), "8-bit type 39")
    refused(call(c=A, s=A, qt=8, cols=63), "whole groups")
    refused(call(cols=(1 << 24) + 1, ldx=1 << 25, ldy=1 << 25), "too large")
    refused(call(rows=1 << 30), "too large")
    for eps in (-1e-6, math.inf, math.nan):
        refused(call(eps=eps), "eps")
    refused(call(ldx=63), "stride")
    refused(call(ldy=63), "stride")
    refused(call(res=A, ldr=63), "stride")
    refused(call(sum_=A, ldr=63), "stride")
    for k in ("x", "w", "y"):
        refused(call(**{k: A + 2}), "aligned")
    refused(call(res=A + 2), "aligned")
    refused(call(sum_=A + 1, rt=BF16), "aligned")
    refused(call(c=A + 8, s=A, qt=F8), "aligned")
    refused(call(c=A, s=A + 2, qt=F8), "aligned")
    assert call(rows=0)
    assert call(rows=0, x=None, y=None)


@pytest.mark.parametrize("front", [False, True])
def test_route_refusals(front):
    L = q4mi.lib()

    def call(lg=A, ty=F32, ld=64, T=2, E=64, bias=None, sig=1, ng=8, kg=4, gt=2, k=8, scale=1.0,
             ids=A, w=A, nh=None, os=9, shared=-1, sg=None, wr=A, wrt=F32, sgw=None, x=A, H=512):
        if front:
            return L.q4mi_moe_route_scored(wr, wrt, sgw, x, T, H, E, bias, sig, ng, kg, gt, k, True,
                                           scale, lg, ids, w, nh, os, shared, sg)
        return L.q4mi_route_scored(lg, ty, ld, T, E, bias, sig, ng, kg, gt, k, True, scale, ids, w,
                                   nh, os, shared, sg)
    for k in ("lg", "ids", "w"):
        refused(call(**{k: None}), "bad arguments")
    refused(call(E=0), "bad arguments")
    refused(call(k=0), "bad arguments")
    refused(call(E=1032, ld=2000), "sizes")
    refused(call(k=65, os=99), "sizes")
    refused(call(T=(1 << 24) + 1), "sizes")
    refused(call(sig=2), "score 2")
    for a in (dict(ng=0), dict(ng=7), dict(ng=128, E=128, ld=128), dict(kg=0), dict(kg=9),
              dict(gt=0), dict(gt=3)):
        refused(call(**a), "groups")
    refused(call(scale=math.inf), "scale")
    refused(call(scale=math.nan), "scale")
    refused(call(os=7), "ostride")
    refused(call(os=8, shared=3), "ostride")
    refused(call(lg=A + 2), "aligned")
    for k in ("bias", "ids", "w", "nh", "sg"):
        refused(call(**{k: A + 2}, **(dict(sgw=A) if k == "sg" else {})), "aligned")
    if front:
        refused(call(wr=None), "bad arguments")
        refused(call(x=None), "bad arguments")
        refused(call(T=0), "bad arguments")
        refused(call(E=520, ng=8), "bad arguments")
        refused(call(wrt=8), "router type")
        refused(call(H=100), "n_embd")
        refused(call(sgw=A), "d_sg")
        refused(call(x=A + 4), "aligned")
    else:
        refused(call(ty=8), "type 8")
        refused(call(lg=A + 1, ty=BF16), "aligned")
        refused(call(ld=63), "stride")
        assert call(T=0)
        assert call(T=0, lg=None, ids=None, w=None)
