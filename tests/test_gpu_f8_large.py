"""8-bit products with outputs past 128 MiB, which go around the caches: rows at whole
lines and not, dense and packed.  Whole numbers, so that sums are exact."""
import numpy as np
import pytest
import torch

import f8_ref as ref
import q4mi
from test_gpu_f8 import F8, TYPES, dev, random_rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("yt,n,rows,ld,cols", [(30, 8300, 8200, 8256, 300), (1, 8300, 8200, 8203, 130),
                                               (0, 5000, 7000, 7008, 130), (0, 5000, 7008, 7008, 128)])
def test_large_outputs(gpu, packed, yt, n, rows, ld, cols):
    rng = np.random.default_rng(n + cols)
    c, s, v = random_rows(rng, 512, cols, True, 128)
    x, xs, xv = random_rows(rng, n, cols, True, 1)
    to = (128 * rng.integers(0, 4, -(-rows // 128))[:, None] + np.arange(128)).reshape(-1)
    d = [dev(a) for a in (c, s, x, xs, to, to[::128] // 128)]
    # the second expert has the blocks of 128 rows in another order
    back = torch.flip(d[4].view(-1, 128), (0,)).reshape(-1)
    nb, rb = ref.blocks(cols), -(-rows // 128)
    w = torch.stack([d[0][d[4]][:rows], d[0][back][:rows]]).contiguous()
    ws = torch.stack([d[1][d[5]], d[1][torch.flip(d[5], (0,))]]).contiguous()
    y = torch.full((n, ld), 77.0, dtype=TYPES[yt], device="cuda")
    half = n // 2 + 1
    if packed:
        bounds = dev(np.array([0, half, n], np.int32))
        q4mi.check(gpu.q4mi_f8_mul_id(w.data_ptr(), ws.data_ptr(), rows, cols, rows * nb * 128,
                                      4 * rb * nb, 2, d[2].data_ptr(), d[3].data_ptr(), n, None,
                                      bounds.data_ptr(), n, y.data_ptr(), yt, ld), "id")
    else:
        q4mi.check(gpu.q4mi_f8_mul(w.data_ptr(), ws.data_ptr(), rows, cols, d[2].data_ptr(),
                                   d[3].data_ptr(), F8, 0, n, y.data_ptr(), yt, ld), "mul")
    sums = torch.from_numpy(xv @ v.T).to(TYPES[yt]).cuda()      # exact in fp32, rounded once
    for i, j, place in ((0, half, d[4]), (half, n, back if packed else d[4])):
        assert torch.equal(y[i:j, :rows], sums[i:j, place[:rows]])
    assert (y[:, rows:] == 77).all()
