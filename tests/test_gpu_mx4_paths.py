"""Every kernel that the 4-bit products choose from, in the forms that the
sizes of test_gpu_mx4 do not reach: large tiles of packed experts, 16-bit
outputs of every dense tile, long rows of the two-group kernel, places past
32-bit offsets, first calls inside a capture.

The choice is restated here and asserted, so that a rule that moves cannot
leave a kernel untested.  Inputs keep every partial sum exact in fp32 (codes
times codes are multiples of 1/4 up to 36; scales within a factor of 4 up to
4096 values, or one scale up to 16384), so an output is the 64-bit result
rounded once to its type: no tolerance anywhere.  Outputs start one element
past an aligned address, rows have odd strides, and everything around them
has to stay as it was."""
import numpy as np
import pytest
import torch

import mx4_ref as ref
import q4mi

pytestmark = pytest.mark.gpu

TYPES = {q4mi.T_F32: torch.float32, q4mi.T_F16: torch.float16, q4mi.T_BF16: torch.bfloat16}
MX4 = q4mi.T_MXFP4


def cus():
    return torch.cuda.get_device_properties(0).multi_processor_count


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def random_rows(gen, rows, cols, codes=None, scales=None):
    """Random codes (0 past cols) and scales, and their values in 64 bits."""
    nb, span = ref.blocks(cols), (126, 129) if cols <= 4096 else (127, 128)
    c = torch.randint(0, 16, (rows, nb * 32), dtype=torch.uint8, device="cuda", generator=gen)
    c[:, cols:] = 0
    s = torch.zeros((rows, ref.scale_row(cols)), dtype=torch.uint8, device="cuda")
    s[:, :nb] = torch.randint(*span, (rows, nb), dtype=torch.uint8, device="cuda", generator=gen)
    t = torch.tensor(np.concatenate([ref.LEVELS, -ref.LEVELS]), device="cuda")
    v = t[c.long()].view(rows, nb, 32) * torch.exp2(s[:, :nb].double() - 127)[..., None]
    packed = c[:, 0::2] | c[:, 1::2] << 4
    if codes is not None:
        codes.copy_(packed.reshape(-1)), scales.copy_(s.reshape(-1))
    return packed, s, v.view(rows, nb * 32)[:, :cols]


class Output:
    """Rows at an odd place: `shift` elements past the allocation, `ld` apart,
    one row more than the call has; all of it -7 before."""

    def __init__(self, rows, cols, yt, ld, shift=1):
        self.t, self.shape = TYPES[yt], (rows + 1, ld)
        self.flat = torch.full((shift + (rows + 1) * ld,), -7.0, dtype=self.t, device="cuda")
        self.want = self.flat.clone()
        self.shift, self.cols, self.ld = shift, cols, ld

    def ptr(self):
        return self.flat[self.shift:].data_ptr()

    def rows(self):
        return self.want[self.shift:].view(self.shape)[:, :self.cols]

    def check(self):
        assert torch.equal(self.flat, self.want)


# --------------------------------------------------------------------- dense

def dense_kernel(n, rows):
    """mul_pick's rule."""
    def tiles(bm, bn):
        return -(-n // bm) * -(-rows // bn)

    c = cus()
    if n <= 16 or tiles(16, 16) <= 2 * c:
        return "one group"
    if n <= 32:
        return "two groups"
    if 2 * tiles(64, 64) <= 5 * c:
        return "64x64"
    if tiles(64, 128) <= 2 * c:
        return "64x128"
    rounds128, rounds256 = -(-tiles(128, 128) // (2 * c)), -(-tiles(256, 256) // c)
    return "128x128" if 3 * rounds128 <= 5 * rounds256 else "256x256"


@pytest.mark.parametrize("yt", sorted(TYPES))
@pytest.mark.parametrize("kernel,n,rows,cols", [
    ("one group", 16, 5001, 352), ("one group", 100, 1030, 8224), ("two groups", 20, 20001, 608),
    ("two groups", 20, 20000, 4128), ("two groups", 32, 9001, 6176), ("two groups", 17, 9000, 12320),
    ("64x64", 65, 8190, 288), ("64x64", 333, 2333, 2080), ("64x128", 700, 5001, 352),
    ("64x128", 650, 5003, 2080), ("128x128", 1300, 5001, 256), ("128x128", 1301, 5000, 800),
    ("256x256", 2100, 5001, 96), ("256x256", 2101, 5002, 1056), ("256x256", 2304, 4608, 544)])
def test_dense_outputs(gpu, yt, kernel, n, rows, cols):
    assert dense_kernel(n, rows) == kernel
    g = generator(n + rows + cols)
    w, ws, wv = random_rows(g, rows, cols)
    x, xs, xv = random_rows(g, n, cols)
    out = Output(n, rows, yt, rows + 3 - rows % 2)
    out.rows()[:n] = (xv @ wv.t()).float().to(TYPES[yt])
    q4mi.check(gpu.q4mi_mx4_mul(w.data_ptr(), ws.data_ptr(), rows, cols, x.data_ptr(),
                                xs.data_ptr(), MX4, 0, n, out.ptr(), yt, out.ld), "mul")
    out.check()


# ------------------------------------------------------------ packed experts

ID_M, ID_N, ID_FEW, ID_COST = 128, 256, 32, 18


def id_tiles(counts, rows):
    """mx4_id_k's rule: (large tiles taken, 0 if everything is streamed;
    streamed 16-row tiles beside them)."""
    blocks, per = cus(), -(-rows // 16)
    items = sum(-(-c // ID_M) for c in counts if c > ID_FEW) * -(-rows // ID_N)
    few = sum(1 for c in counts if 0 < c <= ID_FEW) * per
    sets = sum(-(-c // ID_FEW) for c in counts) * per
    longest = max(-(-items // blocks) * ID_COST, (few + items * ID_COST) // blocks)
    return (items, few) if longest <= -(-sets // blocks) else (0, sets)


def experts_of(kind):
    """Packed rows of each expert."""
    rng = np.random.default_rng(len(kind))
    if kind == "one tile each":         # few tiles, streamed experts and empty ones among them
        c = np.concatenate([rng.integers(129, 300, 18), rng.integers(1, 33, 40), [0] * 9])
    elif kind == "several tiles each":      # every workgroup gets a tile, some two or three
        c = np.concatenate([rng.integers(129, 300, 50), [33, 128, 256, 257, 32, 1]])
    elif kind == "one heavy":           # an expert with most rows, many with one
        c = np.concatenate([[6000], [1] * 60, [0] * 3])
    else:                               # tiles alone
        c = np.concatenate([[128] * 30, [256] * 10])
    return rng.permutation(c).tolist()


@pytest.mark.parametrize("yt", sorted(TYPES))
@pytest.mark.parametrize("kind,rows,cols,gather", [
    ("one tile each", 1030, 96, True), ("one tile each", 1030, 1056, False),
    ("one tile each", 1030, 2080, True), ("several tiles each", 1030, 2080, True),
    ("several tiles each", 1290, 96, False), ("several tiles each", 1030, 32, True),
    ("one heavy", 1100, 1056, True), ("one heavy", 1100, 512, False),
    ("tiles alone", 1280, 256, True), ("tiles alone", 1270, 1000, False)])
def test_packed_experts_in_tiles(gpu, yt, kind, rows, cols, gather):
    """Stretches that begin past row 0 and end past the last row, activation
    rows that do not exist, experts at strides of their own."""
    counts = experts_of(kind)
    E, n = len(counts), sum(counts)
    first, spare = 2, 3
    bounds = np.concatenate([[0], np.cumsum(counts)]) + first
    total = int(bounds[-1]) + spare
    last = max(e for e in range(E) if counts[e])
    bounds[last + 1:] += spare + 5          # the last stretch says more than there is
    g, rng = generator(rows + cols), np.random.default_rng(n)
    nb = ref.blocks(cols)
    wst, sst = rows * nb * 16 + 48, rows * ref.scale_row(cols) + 12
    w = torch.full((E, wst), 0x77, dtype=torch.uint8, device="cuda")
    ws = torch.full((E, sst), 0xff, dtype=torch.uint8, device="cuda")
    xrows = total // 3 if gather else total - 7     # without a list, the last rows have none
    items, few = id_tiles(np.diff(bounds.clip(max=total if gather else xrows)).tolist(), rows)
    assert items and (few > 0) == (kind != "tiles alone")
    assert (items > cus()) == (kind == "several tiles each")
    x, xs, xv = random_rows(g, xrows, cols)
    act = rng.integers(0, xrows, total) if gather else np.arange(total)
    if gather:
        bad = rng.permutation(total)[:total // 20]
        act[bad] = rng.choice([-1, -(1 << 31), xrows, (1 << 31) - 1], len(bad))
    out = Output(total, rows, yt, rows + 5 - rows % 2)
    for e in range(E):
        v = random_rows(g, rows, cols, w[e, :rows * nb * 16], ws[e, :sst - 12])[2]
        p = np.arange(bounds[e], min(bounds[e + 1], total))
        p = p[(act[p] >= 0) & (act[p] < xrows)]
        if len(p):
            at, src = (torch.from_numpy(a.astype(np.int64)).cuda() for a in (p, act[p]))
            out.rows()[at] = (xv[src] @ v.t()).float().to(TYPES[yt])
    d = [torch.from_numpy(a.astype(np.int32)).cuda() for a in (act, bounds)]
    for _ in range(2):
        q4mi.check(gpu.q4mi_mx4_mul_id(w.data_ptr(), ws.data_ptr(), rows, cols, wst, sst, E,
                                       x.data_ptr(), xs.data_ptr(), xrows,
                                       d[0].data_ptr() if gather else None, d[1].data_ptr(), total,
                                       out.ptr(), yt, out.ld), "id")
        out.check()


# ------------------------------------------------------ float rows, both ways

def exact_rows(gen, rows, cols):
    """fp32 rows whose blocks are codes with a largest magnitude of 4 or 6:
    quantising gives the same codes back.  Codes, scales, values."""
    nb = ref.blocks(cols)
    c, s, _ = random_rows(gen, rows, cols)
    lead = torch.randint(6, 8, (rows, nb), dtype=torch.uint8, device="cuda", generator=gen)
    c.view(rows, nb, 16)[:, :, 0] = c.view(rows, nb, 16)[:, :, 0] & 0xf0 | lead
    v = ref.values(c.cpu().numpy(), s.cpu().numpy(), cols)
    return c, s, torch.from_numpy(v).cuda()


@pytest.mark.parametrize("tokens,topk,experts,rows,cols,div", [
    (1, 10, 16, 64, 256, 10), (4, 3, 8, 100, 96, 3), (8, 8, 512, 17, 33, 1),
    (5, 2, 4, 251, 640, 1), (37, 1, 2, 64, 1000, 1)])
def test_listed_experts_take_float_rows(gpu, tokens, topk, experts, rows, cols, div):
    g, rng = generator(rows + cols), np.random.default_rng(tokens * topk)
    n, nb = tokens * topk, ref.blocks(cols)
    wst, sst = rows * nb * 16 + 16, rows * ref.scale_row(cols) + 4
    w = torch.full((experts, wst), 0x77, dtype=torch.uint8, device="cuda")
    ws = torch.full((experts, sst), 0xff, dtype=torch.uint8, device="cuda")
    wv = [random_rows(g, rows, cols, w[e, :wst - 16], ws[e, :sst - 4])[2] for e in range(experts)]
    xr = -(-n // div)
    c, s, xv = exact_rows(g, xr, cols)
    eid = rng.integers(0, experts, n)
    eid[n // 2:n // 2 + 2] = [-1, experts]
    de = torch.from_numpy(eid.astype(np.int32)).cuda()
    f = xv.float()
    q, qs = torch.empty_like(c), torch.empty_like(s)
    q4mi.check(gpu.q4mi_mx4_quant(f.data_ptr(), 0, cols, None, xr, cols, q.data_ptr(),
                                  qs.data_ptr()), "quant")
    assert torch.equal(q, c) and torch.equal(qs, s)
    for a, b, t in ((f, None, q4mi.T_F32), (c, s, MX4)):
        out = Output(n, rows, q4mi.T_F32, rows + 2)
        for p in range(n):
            if 0 <= eid[p] < experts:
                out.rows()[p] = (wv[eid[p]] @ xv[p // div]).float()
        q4mi.check(gpu.q4mi_mx4_mul_sel(w.data_ptr(), ws.data_ptr(), rows, cols, wst, sst, experts,
                                        a.data_ptr(), q4mi.ptr(b), t, cols, div, de.data_ptr(), n,
                                        out.ptr(), 0, out.ld), "sel")
        out.check()


def test_prompt_and_decode_agree(gpu):
    """Sums that are exact do not depend on their order: a token's gate and up
    are the same bits packed with a prompt's rows and listed alone, and so are
    the codes of its activations."""
    g, rng = generator(8), np.random.default_rng(8)
    T, E, K, H, F = 900, 12, 3, 256, 520
    nb = ref.blocks(H)
    w, ws, _ = random_rows(g, E * 2 * F, H)
    ids = np.stack([rng.permutation(E)[:K] for _ in range(T)])
    order = np.argsort(ids.reshape(-1), kind="stable")
    bounds = np.concatenate([[0], np.cumsum(np.bincount(ids.reshape(-1), minlength=E))])
    assert id_tiles(np.diff(bounds).tolist(), 2 * F)[0]
    _, _, xv = exact_rows(g, T, H)
    x = xv.float()
    xq = torch.empty((T, nb * 16), dtype=torch.uint8, device="cuda")
    xs = torch.empty((T, ref.scale_row(H)), dtype=torch.uint8, device="cuda")
    q4mi.check(gpu.q4mi_mx4_quant(x.data_ptr(), 0, H, None, T, H, xq.data_ptr(), xs.data_ptr()),
               "quant")
    d = [torch.from_numpy(a.astype(np.int32)).cuda() for a in (order // K, bounds, ids)]
    arena = (w.data_ptr(), ws.data_ptr(), 2 * F, H, 2 * F * nb * 16, 2 * F * ref.scale_row(H), E)

    def codes(gu, rows):
        h = torch.empty((rows, F), device="cuda")
        q4mi.check(gpu.q4_mmq_swiglu(gu.data_ptr(), h.data_ptr(), rows, F), "swiglu")
        c = torch.empty((rows, ref.blocks(F) * 16), dtype=torch.uint8, device="cuda")
        s = torch.empty((rows, ref.scale_row(F)), dtype=torch.uint8, device="cuda")
        q4mi.check(gpu.q4mi_mx4_quant(h.data_ptr(), 0, F, None, rows, F, c.data_ptr(),
                                      s.data_ptr()), "quant")
        return c, s

    packed = torch.empty((T * K, 2 * F), device="cuda")
    q4mi.check(gpu.q4mi_mx4_mul_id(*arena, xq.data_ptr(), xs.data_ptr(), T, d[0].data_ptr(),
                                   d[1].data_ptr(), T * K, packed.data_ptr(), 0, 2 * F), "packed")
    pc, ps = codes(packed, T * K)
    place = np.argsort(order)       # of (token, pick) among the packed rows
    for t in (0, 1, T // 2, T - 1):
        one = torch.empty((K, 2 * F), device="cuda")
        q4mi.check(gpu.q4mi_mx4_mul_sel(*arena, x[t].data_ptr(), None, 0, H, K, d[2][t].data_ptr(),
                                        K, one.data_ptr(), 0, 2 * F), "listed")
        at = torch.from_numpy(place[t * K:t * K + K]).cuda()
        assert torch.equal(one, packed[at])
        c, s = codes(one, K)
        assert torch.equal(c, pc[at]) and torch.equal(s, ps[at])


# -------------------------------------------------------------- far places

def test_places_past_32_bits(gpu):
    """Experts 3 GiB apart, input and output rows that begin past 2^32
    elements."""
    g, F16 = generator(1), q4mi.T_F16
    E, rows, cols, far, n = 3, 40, 96, 3 << 30, 40
    nb, sr = ref.blocks(cols), ref.scale_row(cols)
    w = torch.empty(2 * far + rows * nb * 16, dtype=torch.uint8, device="cuda")
    ws = torch.empty(2 * far + rows * sr, dtype=torch.uint8, device="cuda")
    wv = [random_rows(g, rows, cols, w[e * far:][:rows * nb * 16], ws[e * far:][:rows * sr])[2]
          for e in range(E)]
    x, xs, xv = exact_rows(g, n, cols)
    near, ld = (1 << 27) + 1, (1 << 31) + 1
    flat = torch.zeros(n * near, dtype=torch.float16, device="cuda")

    y = torch.as_strided(flat, (E, rows), (ld, 1))
    want = torch.stack([wv[e] @ xv[e] for e in range(E)]).float().half()
    ids = torch.arange(E + 1, dtype=torch.int32, device="cuda")
    arena = (w.data_ptr(), ws.data_ptr(), rows, cols, far, far, E)
    q4mi.check(gpu.q4mi_mx4_mul_sel(*arena, x.data_ptr(), xs.data_ptr(), MX4, 0, 1, ids.data_ptr(),
                                    E, flat.data_ptr(), F16, ld), "sel")
    assert torch.equal(y, want)
    y.zero_()
    q4mi.check(gpu.q4mi_mx4_mul_id(*arena, x.data_ptr(), xs.data_ptr(), E, None, ids.data_ptr(), E,
                                   flat.data_ptr(), F16, ld), "id")
    assert torch.equal(y, want)
    del w, ws

    v = torch.as_strided(flat, (n, cols), (near, 1))
    q4mi.check(gpu.q4mi_mx4_dequant(x.data_ptr(), xs.data_ptr(), None, n, cols, flat.data_ptr(),
                                    F16, near), "dequant")
    assert torch.equal(v, xv.half())
    c, s = torch.empty_like(x), torch.empty_like(xs)
    q4mi.check(gpu.q4mi_mx4_quant(flat.data_ptr(), F16, near, None, n, cols, c.data_ptr(),
                                  s.data_ptr()), "quant")
    assert torch.equal(c, x) and torch.equal(s, xs)

    for rows, kernel in ((5000, "64x64"), (100, "one group")):
        assert dense_kernel(n, rows) == kernel
        a, b, av = random_rows(g, rows, cols)
        y = torch.as_strided(flat, (n, rows), (near, 1))
        q4mi.check(gpu.q4mi_mx4_mul(a.data_ptr(), b.data_ptr(), rows, cols, x.data_ptr(),
                                    xs.data_ptr(), MX4, 0, n, flat.data_ptr(), F16, near), "mul")
        assert torch.equal(y, (xv @ av.t()).float().half())
    del flat, y, v
    torch.cuda.empty_cache()


# ------------------------------------------------- first calls of a process

def test_first_calls_inside_a_capture(gpu, gpu_meas):
    """The measurement library is its own copy, and nothing else here calls
    its 4-bit and logits kernels: their first calls, of more than 64 KB of LDS
    among them, are captured, and every replay gives what the product library
    gives eagerly."""
    M, g, rng = gpu_meas, generator(12), np.random.default_rng(12)
    H, E, V, B = 1056, 5, 5000, 70
    sizes = [(1, 400), (20, 20000), (65, 8190), (700, 5001), (1300, 5001), (2100, 5001)]
    kinds = {dense_kernel(*a) for a in sizes}
    assert len(kinds) == 6
    w, ws, _ = random_rows(g, 20000, H)
    most = max(n for n, _ in sizes)
    x = torch.empty((most, H), device="cuda")
    logits = torch.empty((B, V), device="cuda")
    ids = torch.from_numpy(rng.integers(0, E, 64).astype(np.int32)).cuda()
    bounds = torch.tensor([0, 3, 40, 40, 41, 64], dtype=torch.int32, device="cuda")
    hist = torch.from_numpy(rng.integers(0, V, 300).astype(np.int32)).cuda()
    off = torch.from_numpy(np.minimum(np.arange(B + 1) * 5, 300)).cuda()
    pen = torch.tensor([[1.3, 0.1, 0.4]] * B, device="cuda")
    nb, sr, rows = ref.blocks(H), ref.scale_row(H), 500

    def outputs():
        u8 = dict(dtype=torch.uint8, device="cuda")
        return [torch.zeros((most, nb * 16), **u8), torch.zeros((most, sr), **u8),
                torch.zeros((most, H), device="cuda"), torch.zeros((64, rows), device="cuda"),
                torch.zeros((64, rows), device="cuda"), torch.zeros((B, V), device="cuda"),
                *[torch.zeros(a, device="cuda") for a in sizes]]

    def calls(L, o):
        def ok(done, what):
            q4mi.check(done, what, L)
        c, s, v, sel, pk, z, *ys = o
        ok(L.q4mi_mx4_quant(x.data_ptr(), 0, H, None, most, H, c.data_ptr(), s.data_ptr()), "quant")
        ok(L.q4mi_mx4_dequant(c.data_ptr(), s.data_ptr(), None, most, H, v.data_ptr(), 0, H),
           "dequant")
        for (n, r), y in zip(sizes, ys):
            ok(L.q4mi_mx4_mul(w.data_ptr(), ws.data_ptr(), r, H, c.data_ptr(), s.data_ptr(), MX4, 0,
                              n, y.data_ptr(), 0, r), "mul")
        arena = (w.data_ptr(), ws.data_ptr(), rows, H, rows * nb * 16, rows * sr, E)
        ok(L.q4mi_mx4_mul_sel(*arena, x.data_ptr(), None, 0, H, 1, ids.data_ptr(), 64,
                              sel.data_ptr(), 0, rows), "sel")
        ok(L.q4mi_mx4_mul_id(*arena, c.data_ptr(), s.data_ptr(), 64, None, bounds.data_ptr(), 64,
                             pk.data_ptr(), 0, rows), "id")
        ok(L.q4mi_logits_process(logits.data_ptr(), 0, V, B, V, hist.data_ptr(), off.data_ptr(),
                                 None, pen.data_ptr(), None, None, None, None, 0, 0, None,
                                 z.data_ptr(), V), "logits")

    got, want = outputs(), outputs()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    try:
        with torch.cuda.graph(graph):
            q4mi.use_torch_stream(M)
            calls(M, got)
    finally:
        q4mi.use_torch_stream(M)
    for i in range(4):
        x.normal_(generator=g), logits.normal_(generator=g)
        calls(gpu, want)
        for t in got:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for k, (a, b) in enumerate(zip(got, want)):
            assert torch.equal(a, b), (i, k)
            assert bool(a.any())
