"""q4mi_logits_process where test_gpu_logits does not reach: every slice size
in every type, in place and out of place, at the most workgroups, past 32-bit
offsets; penalties without a bound.  The choice of slice is restated here and
asserted.  Formula and tolerance are test_gpu_logits'."""
import numpy as np
import pytest
import torch

import q4mi
from test_gpu_logits import TYPES, call, check, dev, formula, make

pytestmark = pytest.mark.gpu


def slice_tokens(b, v):
    """q4mi_logits_process' rule."""
    least, fill = -(-v // 2048) * b, 4 * torch.cuda.get_device_properties(0).multi_processor_count
    return 2048 * (1 if least <= fill else 2 if least <= 2 * fill else 4)


@pytest.mark.parametrize("xt", sorted(TYPES))
@pytest.mark.parametrize("tokens,b,v,pad,hmax,bmax", [
    (2048, 30, 50001, 3, 2500, 200), (4096, 37, 70001, 1, 2500, 150),
    (8192, 70, 70001, 5, 2500, 150), (8192, 260, 16391, 1, 700, 40),
    (8192, 2100, 100, 3, 60, 9), (8192, 700, 8193, 0, 0, 20), (8192, 1030, 4096, 1, 300, 0)])
def test_every_slice(gpu, xt, tokens, b, v, pad, hmax, bmax):
    assert slice_tokens(b, v) == tokens
    rng = np.random.default_rng(b + v)
    hist, gen, pen, bias, ms, rows = make(rng, b, v, hmax, bmax, 5)
    # the tokens on both sides of every slice's border, in histories and biases
    edge = np.arange(tokens, v, tokens)
    edge = np.concatenate([edge - 1, edge, [0, v - 1]])
    for i in range(0, b, 3):
        if len(hist[i]) >= len(edge):
            hist[i][:len(edge)] = edge
        if len(bias[i][0]) >= len(edge):
            bias[i][0][:len(edge)] = edge
    x = dev(4 * rng.standard_normal((b, v + pad)), TYPES[xt])
    want = formula(x[:, :v].double().cpu().numpy(), hist, gen, pen, bias, ms, rows)
    out = call(gpu, xt, x, v, hist, gen, pen, bias, ms, rows)
    check(out, x, v, want, TYPES[xt])
    y = x.clone()
    call(gpu, xt, y, v, hist, gen, pen, bias, ms, rows, out=y)
    assert torch.equal(y[:, :v], out[:, :v]) and torch.equal(y[:, v:], x[:, v:])


def test_most_workgroups(gpu):
    """2^23 - 1 rows of one workgroup each."""
    b = (1 << 23) - 1
    x = torch.randn((b, 1), device="cuda").half()
    out = torch.zeros_like(x)
    mask = torch.tensor([[1], [0]], dtype=torch.int32, device="cuda")
    row = torch.arange(b, dtype=torch.int32, device="cuda") % 3 - 1
    q4mi.check(gpu.q4mi_logits_process(x.data_ptr(), q4mi.T_F16, 1, b, 1, None, None, None, None,
                                       None, None, None, mask.data_ptr(), 1, 2, row.data_ptr(),
                                       out.data_ptr(), 1), "logits")
    want = torch.where(row[:, None] == 1, torch.full_like(x, -np.inf), x)
    assert torch.equal(out, want)


def test_rows_past_32_bits(gpu):
    """Rows, and the output's, that begin past 2^32 elements."""
    rng = np.random.default_rng(3)
    b, v, ld = 3, 5001, (1 << 31) + 3
    hist, gen, pen, bias, ms, rows = make(rng, b, v, 900, 40, 3)
    flat = torch.zeros(2 * ld + v, dtype=torch.bfloat16, device="cuda")
    x = torch.as_strided(flat, (b, v), (ld, 1))
    x.copy_(dev(4 * rng.standard_normal((b, v))))
    near = call(gpu, q4mi.T_BF16, x.contiguous(), v, hist, gen, pen, bias, ms, rows)
    ids = dev(np.concatenate(hist).astype(np.int32))
    off = dev(np.concatenate([[0], np.cumsum([len(h) for h in hist])]))
    bid = dev(np.concatenate([i for i, _ in bias]).astype(np.int32))
    bva = dev(np.concatenate([a for _, a in bias]))
    bof = dev(np.concatenate([[0], np.cumsum([len(i) for i, _ in bias])]))
    d = [dev(np.asarray(gen, np.int32)), dev(pen), dev(ms.view(np.int32)),
         dev(np.asarray(rows, np.int32))]
    q4mi.check(gpu.q4mi_logits_process(
        flat.data_ptr(), q4mi.T_BF16, ld, b, v, ids.data_ptr(), off.data_ptr(), d[0].data_ptr(),
        d[1].data_ptr(), bid.data_ptr(), bva.data_ptr(), bof.data_ptr(), d[2].data_ptr(),
        ms.shape[1], len(ms), d[3].data_ptr(), flat.data_ptr(), ld), "logits")
    assert torch.equal(x, near)
    del flat, x
    torch.cuda.empty_cache()


@pytest.mark.parametrize("xt", sorted(TYPES))
def test_penalties_without_a_bound(gpu, xt):
    """A token that the model has written may be forbidden by an infinite
    frequency or presence penalty, or forced by a negative one; the others,
    those of the prompt among them, keep their logits (no infinity times
    zero)."""
    v, inf = 3000, np.inf
    prompt, wrote = np.array([5, 6, 7, 2999, 0]), np.array([6, 8, 8, 2048, 0])
    hist = np.concatenate([prompt, wrote]).astype(np.int32)
    pen = np.array([[1, inf, 0], [1, 0, inf], [2, inf, inf], [1, -inf, 0], [1, 0, -inf]],
                   np.float32)
    b = len(pen)
    x = dev(np.random.default_rng(1).standard_normal((b, v)), TYPES[xt])
    out = call(gpu, xt, x, v, [hist] * b, [len(prompt)] * b, pen)
    want = x.clone()
    seen = dev(prompt.astype(np.int64))
    want[2, seen] = torch.where(x[2, seen] > 0, x[2, seen] / 2, x[2, seen] * 2)
    for i in range(b):
        want[i, dev(wrote.astype(np.int64))] = -inf if i < 3 else inf
    assert torch.equal(out, want)
