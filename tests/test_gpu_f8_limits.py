"""8-bit products at the largest number of weight rows (include/q4mi.h: 2^30)."""
import numpy as np
import pytest
import torch

import f8_ref as ref
import q4mi
from test_gpu_f8 import F8, dev, random_rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [17])
def test_most_weight_rows(gpu, n):
    """2^23 tiles of 128 weight rows: 137 GB of codes, the same 128 rows over and over
    with four scales in turn; whole numbers, so that sums are exact."""
    rows, cols = 1 << 30, 128
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 200 << 30:
        pytest.skip("needs 200 GiB of device memory")
    rng = np.random.default_rng(n)
    c, _, wv = random_rows(rng, 128, cols, True, 128)
    wv = ref.values(c, np.ones((1, 1)), cols, 128)
    x, xs, xv = random_rows(rng, n, cols, True, 1)
    w = torch.empty((rows // 128, 128 * 128), dtype=torch.uint8, device="cuda")
    w.copy_(dev(c).view(1, -1).expand_as(w))
    ws = torch.tensor([0.25, 0.5, 1.0, 2.0], device="cuda").repeat(rows // 512)
    y = torch.full((n, rows), 77.0, dtype=torch.bfloat16, device="cuda")
    d = [dev(a) for a in (x, xs)]
    q4mi.check(gpu.q4mi_f8_mul(w.data_ptr(), ws.data_ptr(), rows, cols, d[0].data_ptr(),
                               d[1].data_ptr(), F8, 0, n, y.data_ptr(), 30, rows), "mul")
    want = dev(xv @ wv.T)[:, None, :] * torch.tensor([0.25, 0.5, 1.0, 2.0], device="cuda")[:, None]
    want = want.reshape(n, 512).to(torch.bfloat16)
    for i in range(n):
        assert (y[i].view(-1, 512) == want[i]).all(), i
    del w, ws, y
    torch.cuda.empty_cache()
