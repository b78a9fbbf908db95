"""The 8-bit codes of rows that end inside a block, without a residual: those of the
fp32 y of the same call, exactly."""
import numpy as np
import pytest
import torch

import f8_ref as ref
from test_gpu_norm import F8, TYPES, gen, host, norm, room

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 31), (5, 127), (2, 129), (4, 513), (7, 2049),
                                       (3, 4095), (2, 16385), (2, 32769)])
@pytest.mark.parametrize("xt", sorted(TYPES))
@pytest.mark.parametrize("with_sum", [False, True])
def test_codes(gpu, rows, cols, xt, with_sum):
    x = (3 * torch.randn((rows, cols + 3), device="cuda", generator=gen(cols))).to(TYPES[xt])
    w = 1 + 0.3 * torch.randn(cols, device="cuda", generator=gen(rows))
    sum_ = torch.empty((rows, cols + 1), dtype=torch.bfloat16, device="cuda") if with_sum else None
    y = torch.empty((rows, cols), device="cuda")
    c, s = room(None, cols, F8, rows)
    norm(gpu, x, xt, cols + 3, None, sum_, 30, cols + 1, w, 0, 1e-6, rows, cols, y, 0, cols, F8, c, s)
    h = x[:, :cols]
    if with_sum:
        h = h.to(torch.bfloat16)
        assert torch.equal(sum_[:, :cols], h)
    h = h.double()
    want = h / torch.sqrt((h * h).mean(1, keepdim=True) + float(np.float32(1e-6))) * w.double()
    assert ((y.double() - want).abs() <= 3.1 * 2.0 ** -24 * want.abs()).all()
    wc, ws = ref.quant(host(y))
    assert np.array_equal(host(c), wc) and np.array_equal(host(s), ws)
