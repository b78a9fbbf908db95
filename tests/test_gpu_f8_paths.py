"""The 8-bit products at sizes that reach each of their kernels, where 8-bit sums
cut off, on other streams and in captured graphs, and with the norm and the scored
routing as an engine runs them, against 64 bits (f8_ref)."""
import numpy as np
import pytest
import torch

import f8_ref as ref
import q4mi
from test_gpu_f8 import F8, TYPES, Output, dev, experts, host, quant, random_rows, room_of

pytestmark = pytest.mark.gpu


def mul(L, d, rows, cols, x, xs, xt, ld, n, y, yt, ldy):
    q4mi.check(L.q4mi_f8_mul(d[0].data_ptr(), d[1].data_ptr(), rows, cols, x.data_ptr(),
                             q4mi.ptr(xs), xt, ld, n, y.data_ptr(), yt, ldy), "mul")


def tall(rng, rows, cols):
    """Weights of whole numbers from four different blocks of 128 rows: codes and
    scales on the device, and X -> X . W^T."""
    nb, rb = ref.blocks(cols), -(-rows // 128)
    c, s, v = random_rows(rng, 512, cols, True, 128)
    pick = rng.integers(0, 4, rb)
    to = (pick[:, None] * 128 + np.arange(128)).reshape(-1)[:rows]
    return (dev(c)[dev(to)].contiguous(), dev(s[pick])), lambda x: (x @ v.T)[:, to]


# The sizes at which 64 x 64, 128 x 64, 128 x 128, 256 x 128 and the largest tiles
# begin on a chip of 256 units, and more tiles than it has at once of up to 32, 64
# and 128 rows; whole numbers, so that sums are exact.  Rows at odd addresses and at
# whole lines.
@pytest.mark.parametrize("yt", [0, 30])
@pytest.mark.parametrize("n,rows", [(64, 8200), (130, 8100), (300, 8100), (520, 8100), (1100, 8100),
                                    (257, 16300), (17, 17000),
                                    (32, 40001), (33, 17000), (64, 70000), (65, 17000), (128, 40003)])
@pytest.mark.parametrize("cols", [200, 1290])
def test_mul_every_tile(gpu, n, rows, cols, yt):
    rng = np.random.default_rng(n + cols)
    w, times = tall(rng, rows, cols)
    x, xs, xv = random_rows(rng, n, cols, True, 1)
    x, xs, want = dev(x), dev(xs), times(xv)
    for ld in (rows + 1, -(-rows // 64) * 64):
        out = Output(n, rows, yt, ld)
        out.set(slice(None), want, 0)
        mul(gpu, w, rows, cols, x, xs, F8, 0, n, out.y, yt, ld)
        out.check()


# Several rounds of weight tiles, K in parts, odd numbers of blocks, waves without
# a chunk, with each number of waves a tile.
@pytest.mark.parametrize("n,rows,cols", [
    (1, 40000, 1300), (3, 30000, 256), (16, 20000, 5000), (16, 70, 16384), (7, 9000, 9000),
    (2, 4100, 130), (16, 33000, 128), (5, 2000, 2000), (12, 4096, 6000)])
def test_mul_few_rows(gpu, n, rows, cols):
    rng = np.random.default_rng(n + cols)
    w, times = tall(rng, rows, cols)
    x, xs, xv = random_rows(rng, n, cols, True, 1)
    dx, dxs = dev(x), dev(xs)
    for yt in (0, 1):
        out = Output(n, rows, yt, rows + 1)
        out.set(slice(None), times(xv), 0)
        mul(gpu, w, rows, cols, dx, dxs, F8, 0, n, out.y, yt, out.ld)
        out.check()
    # float rows with the same codes: whole numbers of one scale a block
    f = dev(ref.values(x, xs, cols)).float()
    c, s = quant(gpu, f, 0, cols, n, cols)
    got = torch.empty((2, n, rows), device="cuda")
    mul(gpu, w, rows, cols, f, None, 0, cols, n, got[0], 0, rows)
    mul(gpu, w, rows, cols, c, s, F8, 0, n, got[1], 0, rows)
    assert torch.equal(got[0], got[1])
    assert np.array_equal(host(got[0].double()), times(xv))


@pytest.mark.parametrize("n", [4, 16, 17, 40, 300])
@pytest.mark.parametrize("yt", sorted(TYPES))
def test_sums_below_a_large_product(gpu, n, yt):
    """One product of an eight 2^14 times the others.  fp32 outputs, and all of up to
    sixteen rows, have the others whole.  The 8-bit matrix instruction, which 16-bit
    outputs of more rows come from, may lose of each of the seven what is less than
    2^-13 of the largest."""
    rng = np.random.default_rng(n)
    rows, cols = 96, 512
    v = np.full((n, cols), 448 * 2.0 ** -14)
    v[:, rng.integers(0, 8) + 8 * np.arange(cols // 8)] = 448
    x, xs = ref.encode(v), np.ones((n, 4), np.float32)
    xv = ref.values(x, xs, cols)
    assert np.array_equal(v, xv)
    w, ws = ref.encode(rng.choice([-1.0, 1.0], (rows, cols))), np.full((1, 4), 0.25, np.float32)
    wv = ref.values(w, ws, cols, 128)
    room = room_of(wv, xv, cols, False)
    if yt and n > 16:
        top = np.abs(xv[:, None, :] * wv[None]).reshape(n, rows, -1, 8).max(-1)
        room = room + 7 * 2.0 ** -13 * top.sum(-1)
    out = Output(n, rows, yt, rows)
    out.set(slice(None), xv @ wv.T, room)
    d = [dev(a) for a in (w, ws, x, xs)]
    mul(gpu, d, rows, cols, d[2], d[3], F8, 0, n, out.y, yt, rows)
    out.check()


# Stretches of each size a set can have, in sets of 32, 64, 128 and 256 rows (few of
# them in all; rows an expert), more sets than workgroups, 1024 experts.  Rows at any
# address and at whole lines.
@pytest.mark.parametrize("exact,lines", [(True, False), (True, True), (False, False)])
@pytest.mark.parametrize("counts,rows,cols,yt", [
    ([256, 1, 512, 64, 65, 128, 129, 300, 0, 257], 700, 900, 30),
    ([256, 1, 512, 64, 65, 128, 129, 300, 0, 257], 260, 900, 0),
    ([400, 600], 1030, 128, 1), ([130] * 9, 256, 1100, 30), ([32, 33, 64, 65, 96, 128, 1], 129, 130, 30),
    ([0, 2, 1, 0] * 256, 40, 256, 30), ([3000], 300, 300, 1), ([31, 95, 127] * 30, 2050, 128, 0),
    ([31, 95, 127, 0, 128, 200] * 15, 2050, 300, 30), ([700, 64, 65, 128, 129, 1, 256, 300], 6500, 300, 30),
    ([700, 64, 65, 128, 129, 1, 256, 300], 6500, 130, 0), ([33, 40, 32, 1, 70], 1030, 1100, 30),
    ([33, 40, 32, 1, 70], 1030, 1100, 0)])
def test_id_every_set(gpu, counts, rows, cols, yt, exact, lines):
    rng = np.random.default_rng(rows + len(counts))
    E, total = len(counts), sum(counts)
    nb, rb = ref.blocks(cols), -(-rows // 128)
    few = [random_rows(rng, rows, cols, exact, 128) for _ in range(min(E, 10))]
    pick = np.arange(E) % len(few)
    w = dev(np.stack([f[0].reshape(-1) for f in few]))[torch.from_numpy(pick).cuda()].contiguous()
    ws = dev(np.stack([f[1].reshape(-1) for f in few]))[torch.from_numpy(pick).cuda()].contiguous()
    xrows = total // 2 + 1
    x, xs, xv = random_rows(rng, xrows, cols, exact, 1)
    act = rng.integers(0, xrows, total)
    bounds = np.concatenate([[0], np.cumsum(counts)])
    out = Output(total, rows, yt, -(-rows // 64) * 64 if lines else rows)
    for e in range(E):
        v, wv = xv[act[bounds[e]:bounds[e + 1]]], few[pick[e]][2]
        room = room_of(wv, v, cols, exact)
        if yt and not exact:    # an eight's largest is no more than its sum
            room = room + 7 * 2.0 ** -13 * (np.abs(v) @ np.abs(wv).T)
        out.set(slice(bounds[e], bounds[e + 1]), v @ wv.T, room)
    d = [dev(a) for a in (x, xs, act.astype(np.int32), bounds.astype(np.int32))]
    q4mi.check(gpu.q4mi_f8_mul_id(w.data_ptr(), ws.data_ptr(), rows, cols, rows * nb * 128,
                                  4 * rb * nb, E, d[0].data_ptr(), d[1].data_ptr(), xrows,
                                  d[2].data_ptr(), d[3].data_ptr(), total, out.y.data_ptr(), yt,
                                  out.ld), "id")
    out.check()


def test_bounds_that_do_not_ascend(gpu):
    """Stretches that end before they begin have no rows; the others are as ever."""
    rng = np.random.default_rng(4)
    rows, cols, total = 130, 256, 600
    w, ws, wst, sst, wv = experts(rng, 4, rows, cols, True)
    x, xs, xv = random_rows(rng, total, cols, True, 1)
    for yt, bounds in ((0, [300, 0, 290, 290, 560]), (30, [600, 10, -5, 300, 600])):
        out = Output(total, rows, yt, rows)
        for e, (a, b) in enumerate(zip(bounds, bounds[1:])):
            if b > a:
                out.set(slice(max(a, 0), b), xv[max(a, 0):b] @ wv[e].T, 0)
        d = [dev(a) for a in (x, xs, np.array(bounds, np.int32))]
        q4mi.check(gpu.q4mi_f8_mul_id(w.data_ptr(), ws.data_ptr(), rows, cols, wst, sst, 4,
                                      d[0].data_ptr(), d[1].data_ptr(), total, None,
                                      d[2].data_ptr(), total, out.y.data_ptr(), yt, rows), "id")
        out.check()


class Layer:
    """A routed layer's calls on buffers of its own: norm with the residual, routing,
    the experts of a prompt and of a list, an LM head of few rows and of many."""
    T, E, K, H, F, V = 150, 10, 3, 256, 96, 500

    def __init__(self, rng):
        def t(*n, dtype=torch.float32):
            return torch.zeros(n, dtype=dtype, device="cuda")
        T, E, K, H, F, V = self.T, self.E, self.K, self.H, self.F, self.V
        R, i32, u8 = T * K, torch.int32, torch.uint8
        self.x, self.res = t(T, H, dtype=torch.bfloat16), t(T, H)
        self.o = dict(
            h=t(T, H), y=t(T, H), c=t(T, H, dtype=u8), s=t(T, H // 128), logits=t(T, E),
            ids=t(T, K, dtype=i32), wts=t(T, K), atok=t(R, dtype=i32), rsrc=t(R, dtype=i32),
            rw=t(R), bounds=t(E + 1, dtype=i32), stg=t(512, dtype=i32), stgn=t(1, dtype=i32),
            ek=t(512, dtype=i32), g=t(R, 2 * F), hid=t(R, F), hc=t(R, 128, dtype=u8), hs=t(R, 1),
            pd=t(R, H), z=t(T, H), g1=t(K, 2 * F), h1=t(K, F), d1=t(K, H), lm1=t(2, V),
            zc=t(T, H, dtype=u8), zs=t(T, H // 128), lm=t(T, V, dtype=torch.bfloat16),
            back=t(T, H), ids2=t(T, K, dtype=i32), wts2=t(T, K))

    @staticmethod
    def weights(rng):
        E, H, F, V = Layer.E, Layer.H, Layer.F, Layer.V
        # scales of blocks of 128 rows of each expert: gate and up have 192
        gu = [ref.quant(rng.standard_normal((2 * F, H)) / 16, 128) for _ in range(E)]
        q = [[np.concatenate(a) for a in zip(*gu)],
             ref.quant(rng.standard_normal((E * H, F)) / 10, 128),
             ref.quant(rng.standard_normal((V, H)) / 16, 128)]
        f = [rng.standard_normal((E, H)) / 16, rng.standard_normal(H) + 2, rng.random(E) / 10]
        return ([[dev(a) for a in p] for p in q], [dev(a.astype(np.float32)) for a in f])

    def pack(self, L):
        o = [self.o[k].data_ptr() for k in ("ids", "wts", "atok", "rsrc", "rw", "stg", "stgn", "ek",
                                            "bounds")]
        q4mi.check(L.q4mi_assign(*o, self.T, self.K, self.E, self.T), "pack", L)

    def run(self, L, wt):
        (gu, dn, lm), (wr, nw, bias) = wt
        T, E, K, H, F, V = self.T, self.E, self.K, self.H, self.F, self.V
        R, o = T * K, self.o
        p = {k: v.data_ptr() for k, v in o.items()}

        def ok(done, what):
            q4mi.check(done, what, L)

        def arena(w, rows, cols):
            nb, rb = ref.blocks(cols), -(-rows // 128)
            return (w[0].data_ptr(), w[1].data_ptr(), rows, cols, rows * nb * 128, rb * nb * 4, E)
        ok(L.q4mi_rms_norm(self.x.data_ptr(), 30, H, self.res.data_ptr(), p["h"], 0, H,
                           nw.data_ptr(), 0, 1e-6, T, H, p["y"], 0, H, F8, p["c"], p["s"]), "norm")
        ok(L.q4mi_moe_route_scored(wr.data_ptr(), 0, None, p["y"], T, H, E, bias.data_ptr(), 1, 5, 3,
                                   2, K, True, 2.5, p["logits"], p["ids"], p["wts"], None, K, -1,
                                   None), "route")
        ok(L.q4mi_route_scored(p["logits"], 0, E, T, E, None, 0, 1, 1, 1, K, False, 1.0, p["ids2"],
                               p["wts2"], None, K, -1, None), "route")
        self.pack(L)
        ok(L.q4mi_f8_mul_id(*arena(gu, 2 * F, H), p["c"], p["s"], T, p["atok"], p["bounds"], R,
                            p["g"], 0, 2 * F), "gate/up")
        ok(L.q4_mmq_swiglu(p["g"], p["hid"], R, F), "swiglu")
        ok(L.q4mi_f8_quant(p["hid"], 0, F, None, R, F, 1, p["hc"], p["hs"]), "quant")
        ok(L.q4mi_f8_mul_id(*arena(dn, H, F), p["hc"], p["hs"], R, None, p["bounds"], R, p["pd"], 0,
                            H), "down")
        torch.mul(o["h"], 1.0, out=o["z"])
        ok(L.q4_hip_expert_reduce(p["z"], p["pd"], p["rsrc"], p["rw"], T, K, H), "reduce")
        # the last token alone, as a decode step: float rows in, the router's list
        last = o["ids"][T - 1].data_ptr()
        ok(L.q4mi_f8_mul_sel(*arena(gu, 2 * F, H), o["y"][T - 1].data_ptr(), None, 0, H, K, last, K,
                             p["g1"], 0, 2 * F), "gate/up")
        ok(L.q4_mmq_swiglu(p["g1"], p["h1"], K, F), "swiglu")
        ok(L.q4mi_f8_mul_sel(*arena(dn, H, F), p["h1"], None, 0, F, 1, last, K, p["d1"], 0, H),
           "down")
        ok(L.q4mi_f8_mul(lm[0].data_ptr(), lm[1].data_ptr(), V, H, o["z"][T - 2:].data_ptr(), None,
                         0, H, 2, p["lm1"], 0, V), "LM head")
        ok(L.q4mi_f8_quant(p["z"], 0, H, None, T, H, 1, p["zc"], p["zs"]), "quant")
        ok(L.q4mi_f8_mul(lm[0].data_ptr(), lm[1].data_ptr(), V, H, p["zc"], p["zs"], F8, 0, T,
                         p["lm"], 30, V), "LM head")
        ok(L.q4mi_f8_dequant(p["zc"], p["zs"], None, T, H, 1, p["back"], 0, H), "dequant")

    def fill(self, rng):
        self.x.copy_(dev(rng.standard_normal((self.T, self.H))))
        self.res.copy_(dev(rng.standard_normal((self.T, self.H))))


def near(got, want, room):
    assert (np.abs(host(got.double()) - want) <= room + 2.0 ** -24 * np.abs(want)).all()


def test_layer(gpu):
    """Each step against 64 bits on what the step before it gave."""
    rng = np.random.default_rng(21)
    wt = Layer.weights(rng)
    a = Layer(rng)
    a.fill(rng)
    a.run(gpu, wt)
    T, E, K, H, F, V = a.T, a.E, a.K, a.H, a.F, a.V
    o = {k: host(v) for k, v in a.o.items() if v.dtype != torch.bfloat16}
    (gu, dn, lm), (wr, nw, bias) = wt
    h = host(a.x.float()) + host(a.res)
    assert np.array_equal(o["h"], h)
    h = h.astype(np.float64)
    y = h / np.sqrt((h ** 2).mean(1, keepdims=True) + 1e-6) * host(nw)
    # roundings of 1/sqrt, two products
    assert (np.abs(o["y"] - y) <= 3.1 * 2.0 ** -24 * np.abs(y)).all()
    c, s = ref.quant(o["y"])
    assert np.array_equal(o["c"], c) and np.array_equal(o["s"], s)
    yd, wd = o["y"].astype(np.float64), host(wr).astype(np.float64)
    near(a.o["logits"], yd @ wd.T, (H + 2) * 2.0 ** -24 * (np.abs(yd) @ np.abs(wd).T))
    ids, wts = ref.route(o["logits"], K, 1, host(bias), 5, 3, 2, True, 2.5)
    assert np.array_equal(o["ids"], ids)
    near(a.o["wts"], wts, 2.0 ** -40 * wts)
    ids2, wts2 = ref.route(o["logits"], K, renorm=False)
    assert np.array_equal(o["ids2"], ids2)
    near(a.o["wts2"], wts2, 2.0 ** -40 * wts2)
    # the experts' rows
    order = np.argsort(ids.reshape(-1), kind="stable")
    e = ids.reshape(-1)[order]
    assert np.array_equal(o["atok"], order // K)
    guv = [ref.values(host(gu[0])[i * 2 * F:(i + 1) * 2 * F], host(gu[1])[2 * i:2 * i + 2], H, 128)
           for i in range(E)]
    dnv = [ref.values(host(dn[0])[i * H:(i + 1) * H], host(dn[1])[2 * i:2 * i + 2], F, 128)
           for i in range(E)]

    def rows(got, w, x, e, cols):
        for i in range(len(x)):
            near(got[i], w[e[i]] @ x[i], room_of(w[e[i]], x[i:i + 1], cols, False)[0])
    yv = ref.values(c, s, H)
    rows(a.o["g"], guv, yv[o["atok"]], e, H)
    hc, hs = ref.quant(o["hid"])
    assert np.array_equal(o["hc"], hc) and np.array_equal(o["hs"], hs)
    rows(a.o["pd"], dnv, ref.values(hc, hs, F), e, F)
    pd = o["pd"].astype(np.float64)[o["rsrc"]].reshape(T, K, H) * o["wts"][:, :, None]
    near(a.o["z"], h + pd.sum(1), (2 * K + 1) * 2.0 ** -24 * (np.abs(h) + np.abs(pd).sum(1)) * 1.01)
    # the list's
    rows(a.o["g1"], guv, yv[[T - 1] * K], ids[T - 1], H)
    rows(a.o["d1"], dnv, ref.values(*ref.quant(o["h1"]), F), ids[T - 1], F)
    lmv = ref.values(host(lm[0]), host(lm[1]), H, 128)
    zc, zs = ref.quant(o["z"])
    zv = ref.values(zc, zs, H)
    near(a.o["lm1"], zv[T - 2:] @ lmv.T, room_of(lmv, zv[T - 2:], H, False))
    assert np.array_equal(o["zc"], zc) and np.array_equal(o["zs"], zs)
    assert np.array_equal(o["back"], zv)
    # bf16, off by half a step of 2^-8 and by what the 8-bit instruction cuts off
    want = zv @ lmv.T
    top = np.abs(zv[:, None, :] * lmv[None]).reshape(T, V, -1, 8).max(-1).sum(-1)
    room = room_of(lmv, zv, H, False) + 7 * 2.0 ** -13 * top
    off = np.abs(host(a.o["lm"].double()) - want)
    assert (off <= room + 2.0 ** -8 * (np.abs(want) + room)).all()


def test_layer_in_a_graph(gpu, gpu_meas):
    """Two captured graphs of the layer, on buffers of their own and of a library whose
    first calls they are, replayed in turn with eager work between: the bits that eager
    runs give."""
    rng = np.random.default_rng(22)
    wt = Layer.weights(rng)
    got, eager, graphs = [Layer(rng), Layer(rng)], Layer(rng), []
    eager.fill(rng)
    eager.run(gpu, wt)
    eager.pack(gpu_meas)        # has scratch of its own, allocated outside of captures
    torch.cuda.synchronize()
    try:
        for a in got:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                q4mi.use_torch_stream(gpu_meas)
                a.run(gpu_meas, wt)
            graphs.append(g)
    finally:
        q4mi.use_torch_stream(gpu_meas)
    for i in range(4):
        for a, g in zip(got, graphs):
            a.fill(rng)
            eager.x.copy_(a.x)
            eager.res.copy_(a.res)
            for v in a.o.values():
                v.zero_()
            g.replay()
            eager.run(gpu, wt)
            torch.cuda.synchronize()
            for k in a.o:
                assert torch.equal(a.o[k], eager.o[k]), (i, k)


def test_layer_on_two_streams(gpu):
    """The layer on two streams at once: nothing is shared between calls."""
    rng = np.random.default_rng(23)
    wt = Layer.weights(rng)
    layers, want = [Layer(rng), Layer(rng)], []
    for a in layers:
        a.fill(rng)
        a.run(gpu, wt)
        want.append({k: v.clone() for k, v in a.o.items()})
        for v in a.o.values():
            v.zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    try:
        for _ in range(5):
            for a, s in zip(layers, streams):
                with torch.cuda.stream(s):
                    q4mi.use_torch_stream()
                    a.run(gpu, wt)
    finally:
        q4mi.use_torch_stream()
    torch.cuda.synchronize()
    for a, w in zip(layers, want):
        for k in w:
            assert torch.equal(a.o[k], w[k]), k


@pytest.mark.parametrize("yt", sorted(TYPES))
@pytest.mark.parametrize("rows,cols,pad,block", [(5000, 4099, 2, 1), (4200, 4096, 0, 128)])
def test_dequant_large(gpu, yt, rows, cols, pad, block):
    """Outputs past 32 MiB."""
    rng = np.random.default_rng(rows)
    c, s, v = random_rows(rng, rows, cols, False, block)
    y = torch.full((rows, cols + pad), 77.0, dtype=TYPES[yt], device="cuda")
    d = [dev(a) for a in (c, s)]
    q4mi.check(gpu.q4mi_f8_dequant(d[0].data_ptr(), d[1].data_ptr(), None, rows, cols, block,
                                   y.data_ptr(), yt, cols + pad), "dequant")
    assert torch.equal(y[:, :cols], dev(v.astype(np.float32)).to(TYPES[yt]))
    assert (y[:, cols:] == 77).all()


@pytest.mark.parametrize("n,E", [(16, 2), (17, 16), (17, 17), (63, 64), (64, 64), (64, 512), (90, 64),
                                 (300, 40)])
def test_sel_alone_and_in_groups(gpu, n, E):
    """Rows each on its own and in groups of an expert's, also of one that most name."""
    rng = np.random.default_rng(n + E)
    rows, cols = 70, 300
    w, ws, wst, sst, wv = experts(rng, E, rows, cols, True)
    x, xs, xv = random_rows(rng, n, cols, True, 1)
    for even in (True, False):
        eid = rng.integers(0, E, n) if even else np.where(rng.random(n) < 0.8, E - 1, rng.integers(0, E, n))
        eid[n // 2] = -1
        out = Output(n, rows, 0, rows + 2)
        for p in range(n):
            if eid[p] >= 0:
                out.set(p, xv[p] @ wv[eid[p]].T, 0)
        d = [dev(a) for a in (x, xs, eid.astype(np.int32))]
        q4mi.check(gpu.q4mi_f8_mul_sel(w.data_ptr(), ws.data_ptr(), rows, cols, wst, sst, E,
                                       d[0].data_ptr(), d[1].data_ptr(), F8, 0, 1, d[2].data_ptr(),
                                       n, out.y.data_ptr(), 0, out.ld), "sel")
        out.check()
