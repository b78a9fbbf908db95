"""8-bit products whose sums need every bit of fp32, in each kernel and output type.

Codes and scales of 1 where each eight of products holds one of +-448 * 448 and
seven of +-1, the large ones of two neighbouring eights cancelling: at most
2 * 128 * 200704 / 16 + cols in magnitude at any point, whole numbers below 2^24, so
that every order of additions in fp32 is exact.  A sum that keeps 14 bits below its
largest term would have the cancelled difference alone."""
import numpy as np
import pytest
import torch

import f8_ref as ref
import q4mi
from test_gpu_f8 import F8, TYPES, Output, dev, random_rows

pytestmark = pytest.mark.gpu


def rows_of(rng, n, cols, weights):
    """n rows of codes and their values: +-1, and at the first place of every eight
    448 (activations) or +448 and -448 in turn (weights)."""
    v = rng.choice([-1.0, 1.0], (n, cols))
    v[:, ::8] = 448
    if weights:
        v[:, 8::16] = -448
    nb = ref.blocks(cols)
    codes = np.zeros((n, nb * 128), np.uint8)
    codes[:, :cols] = ref.encode(v)
    return codes, np.ones((-(-n // (128 if weights else 1)), nb), np.float32), v


# a size for each tile on a chip of 256 units
@pytest.mark.parametrize("yt", sorted(TYPES))
@pytest.mark.parametrize("n,rows", [(3, 300), (17, 200), (64, 8200), (130, 8100), (300, 8100),
                                    (520, 8100), (1100, 8100), (17, 17000), (33, 17000), (65, 17000),
                                    (257, 16300)])
def test_mul(gpu, n, rows, yt):
    rng, cols = np.random.default_rng(n), 256
    w, ws, wv = rows_of(rng, 128, cols, True)
    x, xs, xv = rows_of(rng, n, cols, False)
    to = np.arange(rows) % 128      # the same 128 weight rows over and over
    d = [dev(a) for a in (w[to], np.repeat(ws, -(-rows // 128), 0), x, xs)]
    out = Output(n, rows, yt, rows)
    out.set(slice(None), (xv @ wv.T)[:, to], 0)
    q4mi.check(gpu.q4mi_f8_mul(d[0].data_ptr(), d[1].data_ptr(), rows, cols, d[2].data_ptr(),
                               d[3].data_ptr(), F8, 0, n, out.y.data_ptr(), yt, rows), "mul")
    out.check()


# sets of 32, 64, 128 rows, and as many rows an expert as any
@pytest.mark.parametrize("yt", sorted(TYPES))
@pytest.mark.parametrize("counts,rows", [([20, 0, 5], 100), ([64] * 8, 1030), ([100, 129, 3] * 8, 2050),
                                         ([700, 64, 128, 300], 6500)])
def test_id(gpu, counts, rows, yt):
    rng, cols, E, total = np.random.default_rng(rows), 256, len(counts), sum(counts)
    w, ws, wv = rows_of(rng, 128, cols, True)
    x, xs, xv = rows_of(rng, total, cols, False)
    to, rb = np.arange(rows) % 128, -(-rows // 128)
    d = [dev(a) for a in (np.tile(w[to], (E, 1)), np.repeat(ws, E * rb, 0), x, xs,
                          np.concatenate([[0], np.cumsum(counts)]).astype(np.int32))]
    out = Output(total, rows, yt, rows)
    out.set(slice(None), (xv @ wv.T)[:, to], 0)
    q4mi.check(gpu.q4mi_f8_mul_id(d[0].data_ptr(), d[1].data_ptr(), rows, cols, rows * cols,
                                  4 * rb * 2, E, d[2].data_ptr(), d[3].data_ptr(), total, None,
                                  d[4].data_ptr(), total, out.y.data_ptr(), yt, rows), "id")
    out.check()


@pytest.mark.parametrize("yt", [1, 30])
@pytest.mark.parametrize("n,rows,cols", [(5, 300, 900), (40, 2500, 1300), (500, 8200, 640),
                                         (1500, 9000, 300)])
def test_16_bits_are_fp32_rounded(gpu, n, rows, cols, yt):
    """One product, one order of its sums: 16-bit outputs are its fp32 ones rounded."""
    rng = np.random.default_rng(cols)
    w, ws, _ = random_rows(rng, rows, cols, False, 128)
    x, xs, _ = random_rows(rng, n, cols, False, 1)
    d = [dev(a) for a in (w, ws, x, xs, np.array([0, n // 3, n], np.int32))]
    w2, ws2 = (torch.stack([t, t]) for t in d[:2])
    got = {}
    for t in (0, yt):
        y = torch.empty((2, n, rows), dtype=TYPES[t], device="cuda")
        q4mi.check(gpu.q4mi_f8_mul(d[0].data_ptr(), d[1].data_ptr(), rows, cols, d[2].data_ptr(),
                                   d[3].data_ptr(), F8, 0, n, y[0].data_ptr(), t, rows), "mul")
        q4mi.check(gpu.q4mi_f8_mul_id(w2.data_ptr(), ws2.data_ptr(), rows, cols, w.size,
                                      4 * ws.size, 2, d[2].data_ptr(), d[3].data_ptr(), n, None,
                                      d[4].data_ptr(), n, y[1].data_ptr(), t, rows), "id")
        got[t] = y
    assert torch.equal(got[yt], got[0].to(TYPES[yt]))
