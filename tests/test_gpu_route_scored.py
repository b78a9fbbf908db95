"""q4mi_route_scored against its definition in 64 bits: the same ids, weights to
one fp32 rounding (2^-24 relative, and 2^-40 for two 64-bit computations; where
the weight is less than fp32's least normal value, half of its step 2^-149)."""
import numpy as np
import pytest
import torch

import f8_ref as ref
import q4mi

pytestmark = pytest.mark.gpu

TYPES = {0: torch.float32, 1: torch.float16, 30: torch.bfloat16}


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def route(L, z, zt, topk, sigmoid=0, bias=None, groups=1, keep=1, group_top=1, renorm=True,
          scale=1.0, E=None, ostride=None, shared=-1, sg=None, nh=None):
    T, E = z.shape[0], E or z.shape[1]
    ostride = ostride or topk
    ids = torch.full((T, ostride), 777, dtype=torch.int32, device="cuda")
    w = torch.full((T, ostride), 777.0, device="cuda")
    q4mi.check(L.q4mi_route_scored(z.data_ptr(), zt, z.stride(0), T, E, q4mi.ptr(bias), sigmoid,
                                   groups, keep, group_top, topk, renorm, scale, ids.data_ptr(),
                                   w.data_ptr(), q4mi.ptr(nh), ostride, shared, q4mi.ptr(sg)),
               "route")
    return ids.cpu().numpy(), w.cpu().numpy()


def same(got, want):
    assert np.array_equal(got[0], want[0])
    room = (2.0 ** -24 + 2.0 ** -40) * np.abs(want[1]) + 2.0 ** -150
    bad = np.argwhere(np.abs(got[1] - want[1]) > room)
    assert not len(bad), bad[:5]


CASES = [   # experts, topk, groups, kept, group_top
    (1, 1, 1, 1, 1), (2, 2, 1, 1, 1), (63, 8, 1, 1, 1), (64, 64, 1, 1, 1), (128, 10, 1, 1, 1),
    (65, 3, 5, 2, 2), (256, 8, 8, 4, 2), (256, 6, 8, 3, 1), (512, 10, 1, 1, 1), (60, 5, 12, 5, 2),
    (512, 22, 16, 7, 2), (160, 6, 8, 3, 1), (1000, 17, 1, 1, 1), (1024, 10, 64, 9, 2),
    (1024, 64, 2, 1, 1), (48, 4, 48, 6, 2), (513, 12, 3, 2, 2)]


@pytest.mark.parametrize("E,topk,groups,keep,group_top", CASES)
@pytest.mark.parametrize("sigmoid", [0, 1])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("T,zt,renorm", [(1, 0, True), (7, 30, False), (203, 1, True),
                                         (1030, 0, False)])
def test_route(gpu, E, topk, groups, keep, group_top, sigmoid, with_bias, T, zt, renorm):
    rng = np.random.default_rng(E * 10 + T)
    ld = E + 3
    z = dev(rng.standard_normal((T, ld)) * 2).to(TYPES[zt])
    bias = (rng.standard_normal(E) * 0.1).astype(np.float32) if with_bias else None
    got = route(gpu, z, zt, topk, sigmoid, None if bias is None else dev(bias), groups, keep,
                group_top, renorm, 2.5, E)
    some = slice(0, T) if T < 300 else slice(0, T, 7)
    want = ref.route(z[:, :E].double().cpu().numpy()[some], topk, sigmoid, bias, groups, keep,
                     group_top, renorm, 2.5)
    same((got[0][some], got[1][some]), want)


@pytest.mark.parametrize("sigmoid", [0, 1])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("E,topk,groups,keep,group_top", [
    (16, 6, 1, 1, 1), (16, 6, 4, 2, 2), (300, 20, 1, 1, 1), (512, 20, 8, 3, 2)])
def test_masked_tied_and_non_finite(gpu, E, topk, groups, keep, group_top, sigmoid, with_bias):
    """Logits of -inf, the type's lowest value, NaN and +inf, rows with few or no
    experts left, equal logits, biases of -inf, +inf and NaN."""
    rng = np.random.default_rng(E)
    T = 64
    z = rng.integers(-3, 4, (T, E)).astype(np.float32)      # many ties
    z[rng.random((T, E)) < 0.3] = -np.inf
    z[rng.random((T, E)) < 0.05] = np.nan
    z[5] = -np.inf
    z[6] = np.nan
    z[7] = -np.inf
    z[7, E - 1] = 2
    z[8, :] = -np.finfo(np.float32).max
    z[9, 3], z[10, 3], z[10, 4] = np.inf, np.inf, np.inf
    z[11] = 0
    z[12] = np.finfo(np.float32).max
    z[13] = -200        # sigmoid scores of 1e-87
    z[14] = -80000      # of 0
    bias = None
    if with_bias:
        bias = (rng.integers(-2, 3, E) / 8).astype(np.float32)
        bias[1], bias[2], bias[5 % E] = -np.inf, np.nan, np.inf
    for renorm in (True, False):
        got = route(gpu, dev(z), 0, topk, sigmoid, None if bias is None else dev(bias), groups,
                    keep, group_top, renorm)
        same(got, ref.route(z, topk, sigmoid, bias, groups, keep, group_top, renorm))


@pytest.mark.parametrize("topk,shared", [(4, 99), (64, 7), (3, -1)])
def test_lists(gpu, topk, shared):
    """Rows apart, the shared expert after the picks that were found, counts."""
    rng = np.random.default_rng(3)
    T, E = 9, 80
    z = rng.standard_normal((T, E)).astype(np.float32)
    z[4, 2:] = -np.inf
    z[5] = -np.inf
    want = ref.route(z, topk, 1)
    sg = dev(rng.random(T).astype(np.float32))
    nh = torch.full((T,), 777, dtype=torch.int32, device="cuda")
    need = topk + (shared >= 0)
    for gate in (sg, None):
        ids, w = route(gpu, dev(z), 0, topk, 1, ostride=need + 2, shared=shared, sg=gate, nh=nh)
        assert (ids[:, need:] == 777).all() and (w[:, need:] == 777).all()
        for t in range(T):
            found = int((want[0][t] >= 0).sum())
            i, v = list(want[0][t][:found]), list(want[1][t][:found])
            if shared >= 0:
                i.append(shared)
                v.append(float(gate[t]) if gate is not None else 1.0)
            assert int(nh[t]) == len(i)
            rest = need - len(i)
            same((ids[t, :need], w[t, :need]), (np.array(i + [-1] * rest), np.array(v + [0] * rest)))


def test_agrees_with_the_softmax_router(gpu):
    """Without bias and groups the picks are q4_hip_route_pf's, its weights to
    fp32 sums of 512 terms."""
    g = torch.Generator(device="cuda").manual_seed(4)
    T, E, K = 500, 512, 10
    z = torch.randn((T, E), device="cuda", generator=g)
    ids, w = route(gpu, z, 0, K)
    i2 = torch.empty((T, K), dtype=torch.int32, device="cuda")
    w2 = torch.empty((T, K), device="cuda")
    q4mi.check(gpu.q4_hip_route_pf(z.data_ptr(), i2.data_ptr(), w2.data_ptr(), T, E, K), "pf")
    i2, w2 = i2.cpu().numpy(), w2.cpu().numpy()
    rows = (ids == i2).all(1)       # fp32 probabilities can tie
    assert rows.mean() > 0.98
    # expf and its arguments' rounding (|z| < 8: 2^-21), K sums and two divisions
    assert np.abs(w[rows] - w2[rows]).max() <= (8 + K + 4) * 2.0 ** -23


@pytest.mark.parametrize("wt", [0, 1, 30])
@pytest.mark.parametrize("T,gate", [(1, True), (5, False), (70, True)])
def test_router_front(gpu, wt, T, gate):
    """The GEMV's logits are q4mi_moe_route's, the rest the scored routing of
    them."""
    g = torch.Generator(device="cuda").manual_seed(T)
    E, H, K = 96, 512, 6
    rnd = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    wr, x, sgw, bias = (rnd(E, H) / 16).to(TYPES[wt]), rnd(T, H), rnd(H) / 16, rnd(E) * 0.1
    new = lambda *s: torch.zeros(s, device="cuda")  # noqa: E731
    lg, lg2, w, w2, sg, sg2 = new(T, E), new(T, E), new(T, 64), new(T, 64), new(T), new(T)
    ids, ids2 = (torch.zeros((T, 64), dtype=torch.int32, device="cuda") for _ in range(2))
    nh = torch.zeros(T, dtype=torch.int32, device="cuda")
    a = sgw.data_ptr() if gate else None
    q4mi.check(gpu.q4mi_moe_route_scored(
        wr.data_ptr(), wt, a, x.data_ptr(), T, H, E, bias.data_ptr(), 1, 8, 3, 2, K, True, 2.5,
        lg.data_ptr(), ids.data_ptr(), w.data_ptr(), nh.data_ptr(), 64, E, sg.data_ptr()), "front")
    q4mi.check(gpu.q4mi_moe_route(wr.data_ptr(), wt, a, x.data_ptr(), T, H, E, K, lg2.data_ptr(),
                                  ids2.data_ptr(), w2.data_ptr(), None, 64, E, sg2.data_ptr()),
               "route")
    assert torch.equal(lg, lg2) and torch.equal(sg, sg2)
    want = ref.route(lg.double().cpu().numpy(), K, 1, bias.double().cpu().numpy(), 8, 3, 2, True,
                     2.5)
    got = ids.cpu().numpy(), w.cpu().numpy()
    same((got[0][:, :K], got[1][:, :K]), want)
    assert (got[0][:, K] == E).all() and (nh == K + 1).all()
    assert torch.equal(w[:, K], sg if gate else torch.ones_like(sg))


def test_no_tokens(gpu):
    q4mi.check(gpu.q4mi_route_scored(None, 0, 8, 0, 8, None, 1, 1, 1, 1, 2, True, 1.0, None, None,
                                     None, 2, -1, None), "route")


GROUPS = [(1, 1, 1), (8, 4, 2), (8, 2, 1), (12, 5, 2)]


def bias_and_logits(E, T, seed):
    rng = np.random.default_rng(seed)
    z = rng.integers(-6, 7, (T, E)) / 4
    return rng, z.astype(np.float32)


@pytest.mark.parametrize("sigmoid", [0, 1])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("groups,keep,group_top", GROUPS)
@pytest.mark.parametrize("E,topk", [(48, 8), (480, 10), (480, 64), (960, 33)])
def test_many_ties(gpu, E, topk, groups, keep, group_top, with_bias, sigmoid):
    """Logits of 13 values and biases of 4: most keys have equals, also at the last
    pick and the last group, and more than 64 of them may be in question."""
    rng, z = bias_and_logits(E, 40, E + topk)
    z[3], z[4, ::2], z[5] = 0.25, -1.0, -np.inf
    # one bias a group: two of a group's sum with each other's biases would be a tie
    # of the mathematics, not of the rounded keys
    bias = rng.integers(0, 4, E) if groups == 1 else np.repeat(rng.integers(0, 4, groups),
                                                               E // groups)
    bias = (bias / 64).astype(np.float32) if with_bias else None
    got = route(gpu, dev(z), 0, topk, sigmoid, None if bias is None else dev(bias), groups, keep,
                group_top)
    same(got, ref.route(z, topk, sigmoid, bias, groups, keep, group_top))


@pytest.mark.parametrize("sigmoid", [0, 1])
@pytest.mark.parametrize("groups,keep,group_top", GROUPS)
def test_biases_that_cancel(gpu, groups, keep, group_top, sigmoid):
    """A group's two best keys of opposite signs and 10^4 times the scores, so that
    the groups differ in the last bits of an fp32 of either; biases next to one
    another in fp32."""
    rng, z = bias_and_logits(480, 60, 5)
    z += rng.standard_normal(z.shape).astype(np.float32) / 8
    bias = np.full(480, -2.0 ** 13, np.float32)
    bias[::480 // groups] = 2.0 ** 13
    for b in (bias, bias * 2.0 ** -11, bias + rng.integers(0, 2, 480).astype(np.float32) / 1024):
        got = route(gpu, dev(z), 0, 9, sigmoid, dev(b), groups, keep, group_top)
        same(got, ref.route(z, 9, sigmoid, b, groups, keep, group_top))


@pytest.mark.parametrize("sigmoid", [0, 1])
@pytest.mark.parametrize("groups,keep,group_top", GROUPS)
def test_largest_biases(gpu, groups, keep, group_top, sigmoid):
    """Biases of +-inf, NaN and the largest finite ones (two of which are no fp32)."""
    rng, z = bias_and_logits(480, 30, 6)
    z[2, 10:30] = np.finfo(np.float32).max
    z[3] = np.finfo(np.float32).min
    z[4, 5] = np.inf
    big = np.finfo(np.float32).max
    b = rng.choice(np.array([0, 1, big, -big, np.inf, -np.inf, np.nan], np.float32), 480,
                   p=[.3, .3, .1, .1, .05, .1, .05])
    got = route(gpu, dev(z), 0, 12, sigmoid, dev(b), groups, keep, group_top)
    same(got, ref.route(z, 12, sigmoid, b, groups, keep, group_top))


def test_nearest_keys(gpu):
    """Keys a few last bits of an fp32 apart, of which the hardware's exponential
    says nothing: the order of 64 bits."""
    rng = np.random.default_rng(8)
    E, T = 512, 200
    base = np.float32(1.5) + np.arange(E, dtype=np.float32) * np.float32(2.0 ** -23)
    z = np.stack([rng.permutation(base) for _ in range(T)])
    for sigmoid in (0, 1):
        for bias in (None, np.full(E, 2.0 ** -9, np.float32)):
            for g in ((1, 1, 1), (8, 4, 2)):
                got = route(gpu, dev(z), 0, 10, sigmoid, None if bias is None else dev(bias), *g)
                same(got, ref.route(z, 10, sigmoid, bias, *g))
