"""Microscaled 4-bit floating point and the logits of a decode step, as timing
cases.

Each case goes through the public C entry points the way an engine calls
them, or through the operators' plain forms:

  quant   rows to microscaled 4-bit blocks (q4mi_mx4_quant), read back as
          values (q4mi_mx4_dequant)
  mul     y[t] = W . x[t], weights and activations in 4 bits (q4mi_mx4_mul);
          up to eight float rows go in as they are, more are quantised first
  sel     every row through the expert that a list names (q4mi_mx4_mul_sel):
          routed experts of a decode step
  id      packed rows, each expert's in one stretch (q4mi_mx4_mul_id): routed
          experts of a prompt
  logits  penalties for repeated tokens, biases and grammar masks on a batch's
          logits (q4mi_logits_process)

A microscaled block is 32 values of a row: 4-bit codes (sign, two exponent
bits, one mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6) times one power of two,
kept as a byte s for 2^(s - 127).  A row of n values has nb = ceil(n / 32)
blocks, 16 * nb bytes of codes (two to a byte, the even value low) and its
scales padded to whole dwords.

Weights are N(0, 1/cols) in this format, activations N(0,1) with a few large
channels, prompts' routing Zipf; histories repeat few tokens often.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

TYPES = {"f32": (0, torch.float32), "f16": (1, torch.float16), "bf16": (30, torch.bfloat16)}
MX4 = 39
FLOAT_ROWS = 8      # rows of float activations that q4mi_mx4_mul takes as they are


def listed():
    return [
        # one token's hidden state ahead of a decode product
        {"name": "quant_token", "kind": "quant", "rows": 1, "cols": 2048, "pad": 0,
         "gather": False, "x": "f32", "y": "f32"},
        # a prompt chunk's activations
        {"name": "quant_prompt", "kind": "quant", "rows": 4096, "cols": 4096, "pad": 0,
         "gather": False, "x": "bf16", "y": "bf16"},
        # the smallest product of a decode step: one short projection
        {"name": "mul_token", "kind": "mul", "n": 1, "rows": 2048, "cols": 2048, "x": "f32",
         "y": "f32"},
        # the LM head of a decode step
        {"name": "mul_lm_head", "kind": "mul", "n": 1, "rows": 151936, "cols": 2048, "x": "f32",
         "y": "f32"},
        # a ragged batch through a projection of the reference model's width
        {"name": "mul_batch_77", "kind": "mul", "n": 77, "rows": 2560, "cols": 2560, "x": "bf16",
         "y": "bf16"},
        # a long prompt through a square projection
        {"name": "mul_prompt", "kind": "mul", "n": 8192, "rows": 8192, "cols": 8192, "x": "bf16",
         "y": "bf16"},
        # gate and up of one decode token's ten experts
        {"name": "sel_gate_up", "kind": "sel", "tokens": 1, "topk": 10, "experts": 128,
         "rows": 1024, "cols": 2048, "each": False, "x": "f32", "y": "f32"},
        # down of a four-token verify window's experts, each row its own input
        {"name": "sel_down_window", "kind": "sel", "tokens": 4, "topk": 10, "experts": 512,
         "rows": 2048, "cols": 512, "each": True, "x": "f32", "y": "f32"},
        # gate and up of a prompt chunk's routed experts
        {"name": "id_prompt", "kind": "id", "tokens": 2048, "topk": 10, "experts": 512,
         "rows": 1024, "cols": 2048, "spare": 0, "x": "f32", "y": "f32"},
        # the reference model's widths and a short ragged prompt: a handful of rows an expert
        {"name": "id_prompt_333", "kind": "id", "tokens": 333, "topk": 10, "experts": 256,
         "rows": 1280, "cols": 2560, "spare": 5, "x": "bf16", "y": "bf16"},
        # the logits of one decode token with a grammar
        {"name": "logits_token", "kind": "logits", "batch": 1, "vocab": 151936, "history": 2000,
         "biases": 20, "grammar": 1.0, "penalties": True, "x": "f32"},
        # a serving batch with long histories, some rows under a grammar
        {"name": "logits_batch", "kind": "logits", "batch": 64, "vocab": 151936,
         "history": 32768, "biases": 300, "grammar": 0.5, "penalties": True, "x": "f32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cols(rng):
    """Row lengths: mostly whole blocks, now and then any number."""
    if rng.random() < 0.3:
        return _log(rng, 1, 8192)
    return 32 * _log(rng, 1, 256)


def _draw(rng):
    kind = rng.choice(["quant", "mul", "mul", "sel", "id", "logits"])
    c = {"kind": kind, "x": rng.choice(sorted(TYPES))}
    if kind == "logits":
        c.update(batch=_log(rng, 1, 256), vocab=_log(rng, 100, 152000),
                 history=_log(rng, 1, 32768) if rng.random() < 0.9 else 0,
                 biases=_log(rng, 1, 2000) if rng.random() < 0.7 else 0,
                 grammar=rng.choice([0.0, 0.5, 1.0]), penalties=rng.random() < 0.8)
        return c
    c.update(y=rng.choice(sorted(TYPES)), cols=_cols(rng))
    if kind == "quant":
        c.update(rows=_log(rng, 1, 8192), pad=rng.choice([0, 0, 8, rng.randint(1, 70)]),
                 gather=rng.random() < 0.4)
    elif kind == "mul":
        c.update(n=_log(rng, 1, 8192), rows=_log(rng, 1, 152000))
    elif kind == "sel":
        c.update(tokens=rng.randint(1, 8), topk=rng.randint(1, 16), experts=_log(rng, 1, 512),
                 rows=_log(rng, 16, 4096), each=rng.random() < 0.5)
    else:
        c.update(tokens=_log(rng, 1, 2048), topk=rng.randint(1, 10), experts=_log(rng, 1, 512),
                 rows=_log(rng, 16, 4096), spare=rng.choice([0, 0, rng.randint(1, 40)]))
        c["topk"] = min(c["topk"], c["experts"])
    return c


def _cost(case):
    w = work(case)
    return w["bytes"] / 2e12 + w["flops"] / 1e15


def _weights_held(case):
    """Values of all weight matrices (the plain forms hold them at 32 bits)."""
    return case.get("experts", 1) * case.get("rows", 0) * case["cols"] if "cols" in case else 0


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        c = _draw(rng)
        if _cost(c) <= most and _weights_held(c) <= 1.1e9:
            return c


# ------------------------------------------------------------------ sizes

def _blocks(cols):
    return (cols + 31) // 32


def _scale_row(cols):
    return (_blocks(cols) + 3) // 4 * 4


def _size(name):
    return TYPES[name][1].itemsize


def work(case):
    """Each input once, each output once; a product's multiplications and
    additions over the values of its rows."""
    kind = case["kind"]
    if kind == "logits":
        n = case["batch"] * case["vocab"]
        lists = case["batch"] * (4 * case["history"] // 2 + 8 * case["biases"])
        mask = int(case["grammar"] * n) // 8
        return {"bytes": 2 * n * _size(case["x"]) + lists + mask, "flops": 4 * n}
    row = _blocks(case["cols"]) * 17
    if kind == "quant":
        n = case["rows"] * case["cols"]
        return {"bytes": n * (_size(case["x"]) + _size(case["y"])) + 2 * case["rows"] * row,
                "flops": 2 * n}
    if kind == "mul":
        n, xrows, held = case["n"], case["n"], 1
    else:
        n = case["tokens"] * case["topk"]
        xrows = n if case.get("each") else case["tokens"]
        held = min(n, case["experts"])
    return {"bytes": held * case["rows"] * row + xrows * case["cols"] * _size(case["x"]) +
            n * case["rows"] * _size(case["y"]),
            "flops": 2 * n * case["rows"] * case["cols"]}


# ------------------------------------------------------------- plain forms

LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _plain_quant(x, cols):
    """Rows of floats -> codes [rows][16 nb] and scales [rows][scale row]:
    exponent floor(log2(largest)) - 2, codes to nearest (ties to the even
    code), at most 6; a block with an infinity or a NaN has scale 255."""
    rows, nb = x.shape[0], _blocks(cols)
    v = torch.zeros((rows, nb * 32), dtype=torch.float32, device=x.device)
    v[:, :cols] = x.float()
    v = v.view(rows, nb, 32)
    top = v.abs().amax(2)
    bad = ~torch.isfinite(v).all(2)
    exp = (torch.frexp(torch.where(bad, torch.ones_like(top), top))[1] - 3).clamp(-127, 127)
    exp = torch.where(top == 0, torch.full_like(exp, -127), exp)
    a = torch.ldexp(v, -exp[..., None])
    s = torch.signbit(a).to(torch.uint8) * 8
    a = a.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) +
            (a >= 3.5) + (a > 5.0)).to(torch.uint8) + s
    code = torch.where(bad[..., None], torch.zeros_like(code), code).view(rows, nb * 32)
    scales = torch.zeros((rows, _scale_row(cols)), dtype=torch.uint8, device=x.device)
    scales[:, :nb] = torch.where(bad, torch.full_like(exp, 255), exp + 127).to(torch.uint8)
    return code[:, 0::2] + code[:, 1::2] * 16, scales


def _plain_values(codes, scales, cols):
    """What codes and scales stand for, in 32 bits."""
    rows, nb = codes.shape[0], _blocks(cols)
    table = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=codes.device)
    v = torch.stack([table[(codes & 15).int()], table[(codes >> 4).int()]], 2).view(rows, nb, 32)
    s = scales[:, :nb].int()
    f = torch.ldexp(torch.ones((), device=codes.device), s - 127)
    f = torch.where(s == 255, torch.full_like(f, math.nan), f)
    return (v * f[..., None]).reshape(rows, nb * 32)[:, :cols]


def _plain_x(s):
    return _plain_values(*_plain_quant(s["x"], s["case"]["cols"]), s["case"]["cols"])


def _plain_logits(s):
    c, b = s["case"], s["case"]["batch"]
    z = s["x"].float()
    if c["penalties"] and s["hist"].numel():
        row = torch.repeat_interleave(torch.arange(b, device="cuda"), s["lens"],
                                      output_size=s["hist"].numel())
        at = torch.arange(s["hist"].numel(), device="cuda")
        hist = s["hist"].long()
        ok = (hist >= 0) & (hist < c["vocab"])
        flat = torch.where(ok, row * c["vocab"] + hist, torch.zeros_like(row))
        late = at >= s["hist_off"][row] + s["gen"].long()[row]
        # the whole history, and the part that the model wrote
        every = torch.zeros(z.numel(), device="cuda").index_add_(0, flat, ok.float())
        wrote = torch.zeros(z.numel(), device="cuda").index_add_(0, flat, (ok & late).float())
        every, wrote = every.view_as(z), wrote.view_as(z)
        rep, freq, pres = (s["pen"][:, i:i + 1] for i in range(3))
        z = torch.where(every > 0, torch.where(z > 0, z / rep, z * rep), z)
        z = z - freq * wrote - pres * (wrote > 0)
    if s["bias"].numel():
        row = torch.repeat_interleave(torch.arange(b, device="cuda"), s["bias_lens"],
                                      output_size=s["bias"].numel())
        ids = s["bias_ids"].long()
        ok = (ids >= 0) & (ids < c["vocab"])
        flat = torch.where(ok, row * c["vocab"] + ids, torch.zeros_like(row))
        add = torch.zeros(z.numel(), dtype=torch.float64, device="cuda").index_add_(
            0, flat, torch.where(ok, s["bias"], torch.zeros_like(s["bias"])).double())
        z = z + add.float().view_as(z)
    if s["mask"] is not None:
        at = torch.arange(c["vocab"], device="cuda")
        words = s["mask"][s["mask_row"].clamp(min=0).long()]
        allowed = (words[:, at // 32] >> (at % 32)) & 1
        z = torch.where((allowed == 0) & (s["mask_row"][:, None] >= 0),
                        torch.full_like(z, -math.inf), z)
    return z.to(s["x"].dtype)


def _plain(s):
    c, kind = s["case"], s["case"]["kind"]
    if kind == "logits":
        return {"z": _plain_logits(s)}
    y = TYPES[c["y"]][1]
    if kind == "quant":
        x = s["x"] if s["ids"] is None else s["x"][s["ids"].long()]
        return {"v": _plain_values(*_plain_quant(x[:, :c["cols"]], c["cols"]), c["cols"]).to(y)}
    x = _plain_x(s)
    if kind == "mul":
        w = _plain_values(s["w"], s["ws"], c["cols"])
        return {"y": (x @ w.t()).to(y)}
    if kind == "sel":
        out = torch.empty((c["tokens"] * c["topk"], c["rows"]), dtype=torch.float32, device="cuda")
        w, ws = s["w"].view(c["experts"], c["rows"], -1), s["ws"].view(c["experts"], c["rows"], -1)
        for p in range(len(out)):
            e = s["eid"][p:p + 1].long()
            v = _plain_values(w[e][0], ws[e][0], c["cols"])
            out[p] = (v * x[p if c["each"] else p // c["topk"]]).sum(1)
        return {"y": out.to(y)}
    out = s["y"].float()
    w, ws = s["w"].view(c["experts"], c["rows"], -1), s["ws"].view(c["experts"], c["rows"], -1)
    x = x[s["act"].long()]
    for e in range(c["experts"]):
        lo, hi = s["stretch"][e], s["stretch"][e + 1]
        if hi > lo:
            out[lo:hi] = x[lo:hi] @ _plain_values(w[e], ws[e], c["cols"]).t()
    return {"y": out.to(y)}


# ----------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _matrix(rows, cols, gen):
    """Weights N(0, 1/cols) in 4 bits: codes [rows][16 nb], scales."""
    codes = torch.empty((rows, _blocks(cols) * 16), dtype=torch.uint8, device="cuda")
    scales = torch.empty((rows, _scale_row(cols)), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 26) // cols)
    for r in range(0, rows, step):
        v = torch.randn((min(step, rows - r), cols), device="cuda", generator=gen)
        codes[r:r + step], scales[r:r + step] = _plain_quant(v / math.sqrt(cols), cols)
    return codes, scales


def _activations(rows, cols, name, gen):
    """N(0,1) with about one channel in a hundred at twenty times the size."""
    x = torch.randn((rows, cols), device="cuda", generator=gen)
    x *= 1 + 19 * (torch.rand(cols, device="cuda", generator=gen) < 0.01)
    return x.to(TYPES[name][1])


def _new(rows, cols):
    """Room for the codes and scales of quantised rows."""
    return (torch.empty((rows, _blocks(cols) * 16), dtype=torch.uint8, device="cuda"),
            torch.empty((rows, _scale_row(cols)), dtype=torch.uint8, device="cuda"))


def _ragged(rng, batch, most):
    """Lengths of a batch's lists: about half of `most`, at most that, some
    rows empty."""
    n = rng.integers(0, most + 1, batch)
    n[0] = most
    return n


def _prepare_logits(case, seed, gen):
    rng = np.random.default_rng(seed)
    b, v = case["batch"], case["vocab"]
    cuda = lambda a, t: torch.from_numpy(np.ascontiguousarray(a)).to("cuda", t)  # noqa: E731
    s = {"x": (4 * torch.randn((b, v), device="cuda", generator=gen)).to(TYPES[case["x"]][1])}
    lens = _ragged(rng, b, case["history"])
    n = int(lens.sum())
    # a text's tokens: few of them often
    hist = (v * torch.rand(n, device="cuda", generator=gen) ** 4).int().clamp(max=v - 1)
    # now and then a place that no token stands for (an image's, say)
    s["hist"] = torch.where(torch.rand(n, device="cuda", generator=gen) < 0.001,
                            torch.full_like(hist, -1), hist)
    s["lens"] = cuda(lens, torch.int64)
    s["hist_off"] = cuda(np.concatenate([[0], np.cumsum(lens)]), torch.int64)
    s["gen"] = cuda(rng.integers(0, lens + 1), torch.int32)
    s["pen"] = cuda(np.stack([rng.uniform(0.8, 1.5, b), rng.uniform(-0.2, 0.5, b),
                              rng.uniform(-0.5, 1.0, b)], 1), torch.float32)
    blens = _ragged(rng, b, case["biases"])
    n = int(blens.sum())
    s["bias_ids"] = cuda(rng.integers(0, v, n), torch.int32)
    s["bias"] = cuda(rng.uniform(-10, 10, n), torch.float32)
    s["bias_lens"] = cuda(blens, torch.int64)
    s["bias_off"] = cuda(np.concatenate([[0], np.cumsum(blens)]), torch.int64)
    s["mask"] = s["mask_row"] = None
    if case["grammar"] > 0:
        # states of a grammar: how many tokens each allows differs widely; one of a batch's
        # allows none
        states, words = (b + 1) // 2, (v + 31) // 32
        share = torch.rand((states, 1, 1), device="cuda", generator=gen) ** 6
        share[1:2] = 0
        share[0] += 0.01
        bits = (torch.rand((states, words, 32), device="cuda", generator=gen) < share).int()
        s["mask"] = (bits << torch.arange(32, device="cuda", dtype=torch.int32)).sum(
            2, dtype=torch.int32)
        row = rng.integers(0, states, b)
        row[rng.random(b) >= case["grammar"]] = -1
        s["mask_row"] = cuda(row, torch.int32)
    s["z"] = torch.empty_like(s["x"])
    return s


def _zipf(rng, tokens, topk, experts):
    """Each token's distinct experts, by Zipf popularity (exponent 1.1)."""
    popular = rng.permutation(experts)
    key = rng.gumbel(size=(tokens, experts)) - 1.1 * np.log1p(popular)[None]
    return np.argsort(-key, axis=1, kind="stable")[:, :topk]


def prepare(case, seed):
    """What an engine has in hand: weights in 4 bits, activations, lists and
    room for the outputs."""
    gen, kind = _gen(seed), case["kind"]
    if kind == "logits":
        s = _prepare_logits(case, seed, gen)
    elif kind == "quant":
        rows, cols = case["rows"], case["cols"]
        s = {"x": _activations(rows, cols + case["pad"], case["x"], gen), "ids": None,
             "v": torch.empty((rows, cols), dtype=TYPES[case["y"]][1], device="cuda")}
        if case["gather"]:
            s["ids"] = torch.randint(0, rows, (rows,), device="cuda", generator=gen,
                                     dtype=torch.int32)
        s["xq"], s["xs"] = _new(rows, cols)
    else:
        rng = np.random.default_rng(seed)
        n = case["n"] if kind == "mul" else case["tokens"] * case["topk"]
        xrows = n if kind == "mul" or case.get("each") else case["tokens"]
        s = {"x": _activations(xrows, case["cols"], case["x"], gen)}
        s["xq"], s["xs"] = _new(xrows, case["cols"])
        s["w"], s["ws"] = _matrix(case.get("experts", 1) * case["rows"], case["cols"], gen)
        if kind == "sel":
            e = np.stack([rng.permutation(max(case["experts"], case["topk"]))[:case["topk"]]
                          for _ in range(case["tokens"])]) % case["experts"]
            s["eid"] = torch.from_numpy(e.reshape(-1).astype(np.int32)).cuda()
        elif kind == "id":
            ids = _zipf(rng, case["tokens"], case["topk"], case["experts"]).reshape(-1)
            order = np.argsort(ids, kind="stable")
            stretch = np.concatenate([[0], np.cumsum(np.bincount(ids, minlength=case["experts"]))])
            act = np.concatenate([order // case["topk"], np.zeros(case["spare"], np.int64)])
            s["act"] = torch.from_numpy(act.astype(np.int32)).cuda()
            s["bounds"] = torch.from_numpy(stretch.astype(np.int32)).cuda()
            s["stretch"] = stretch.tolist()
            n += case["spare"]      # rows past the last expert's stay as they are
        s["y"] = torch.zeros((n, case["rows"]), dtype=TYPES[case["y"]][1], device="cuda")
    s["case"] = case
    if own:
        _q4mi().use_torch_stream()
    return s


# ------------------------------------------------------------ one pass

def _q4mi():
    path = os.path.join(os.getcwd(), "suzuku-engine-q4_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import q4mi
    return q4mi


def _p(t):
    return None if t is None else t.data_ptr()


def _quantise(q, s):
    c, x = s["case"], s["x"]
    q.check(q.lib().q4mi_mx4_quant(x.data_ptr(), TYPES[c["x"]][0], x.shape[1], None, x.shape[0],
                                   c["cols"], s["xq"].data_ptr(), s["xs"].data_ptr()), "quantise")


def _run_logits(q, s):
    c, v = s["case"], s["case"]["vocab"]
    pen = c["penalties"]
    q.check(q.lib().q4mi_logits_process(
        s["x"].data_ptr(), TYPES[c["x"]][0], v, c["batch"], v,
        _p(s["hist"]) if pen else None, _p(s["hist_off"]) if pen else None,
        _p(s["gen"]) if pen else None, _p(s["pen"]) if pen else None, _p(s["bias_ids"]),
        _p(s["bias"]), _p(s["bias_off"]), _p(s["mask"]),
        0 if s["mask"] is None else s["mask"].shape[1],
        0 if s["mask"] is None else s["mask"].shape[0], _p(s["mask_row"]), s["z"].data_ptr(), v),
        "logits")
    return {"z": s["z"]}


def run(s):
    if not own:
        return _plain(s)
    q, c, kind = _q4mi(), s["case"], s["case"]["kind"]
    if kind == "logits":
        return _run_logits(q, s)
    lib, xt, yt = q.lib(), TYPES[c["x"]][0], TYPES[c["y"]][0]
    if kind == "quant":
        x = s["x"]
        q.check(lib.q4mi_mx4_quant(x.data_ptr(), xt, x.shape[1], _p(s["ids"]), c["rows"],
                                   c["cols"], s["xq"].data_ptr(), s["xs"].data_ptr()), "quantise")
        q.check(lib.q4mi_mx4_dequant(s["xq"].data_ptr(), s["xs"].data_ptr(), None, c["rows"],
                                     c["cols"], s["v"].data_ptr(), yt, c["cols"]), "values")
        return {"v": s["v"]}
    w, ws, rows, cols, y = s["w"], s["ws"], c["rows"], c["cols"], s["y"]
    if kind == "mul":
        x, xs = s["x"], None
        if c["n"] > FLOAT_ROWS:
            _quantise(q, s)
            x, xs, xt = s["xq"], s["xs"], MX4
        q.check(lib.q4mi_mx4_mul(w.data_ptr(), ws.data_ptr(), rows, cols, x.data_ptr(), _p(xs),
                                 xt, cols, c["n"], y.data_ptr(), yt, rows), "product")
    elif kind == "sel":
        q.check(lib.q4mi_mx4_mul_sel(
            w.data_ptr(), ws.data_ptr(), rows, cols, rows * w.shape[1], rows * ws.shape[1],
            c["experts"], s["x"].data_ptr(), None, xt, cols, 1 if c["each"] else c["topk"],
            s["eid"].data_ptr(), c["tokens"] * c["topk"], y.data_ptr(), yt, rows), "experts")
    else:
        _quantise(q, s)
        q.check(lib.q4mi_mx4_mul_id(
            w.data_ptr(), ws.data_ptr(), rows, cols, rows * w.shape[1], rows * ws.shape[1],
            c["experts"], s["xq"].data_ptr(), s["xs"].data_ptr(), c["tokens"],
            s["act"].data_ptr(), s["bounds"].data_ptr(), len(y), y.data_ptr(), yt, rows),
            "experts")
    return {"y": y}


# --------------------------------------------------------- in 64 bits

def _exact_round(x, cols):
    """Rows as the 4-bit format holds them, from its definition: the block's
    exponent, then the nearest multiple of the step at each size, ties to
    even."""
    rows, nb = x.shape[0], _blocks(cols)
    v = torch.nn.functional.pad(x.double(), (0, nb * 32 - cols)).reshape(rows, nb, 32)
    top = v.abs().max(2, keepdim=True).values
    unit = torch.exp2(torch.floor(torch.log2(top)).clamp(min=-125) - 2)
    a = torch.where(top > 0, v / unit, torch.zeros_like(v))
    m = a.abs()
    step = torch.where(m < 2, 0.5, torch.where(m < 4, 1.0, 2.0)).double()
    m = torch.minimum(torch.round(m / step) * step, torch.full_like(m, 6.0))
    return (torch.copysign(m, a) * unit).reshape(rows, nb * 32)[:, :cols]


def _exact_weights(codes, scales, cols):
    """Weights from their bits: sign, two exponent bits, one mantissa bit."""
    q = torch.stack([codes % 16, codes // 16], 2).reshape(codes.shape[0], -1).double()
    sign = torch.where(q >= 8, -1.0, 1.0).double()
    q = q % 8
    e, m = torch.floor(q / 2), q % 2
    mag = torch.where(e == 0, m / 2, torch.exp2(e - 1) * (1 + m / 2))
    unit = torch.exp2(scales[:, :_blocks(cols)].double() - 127)
    return (sign * mag * torch.repeat_interleave(unit, 32, 1))[:, :cols]


def _exact_logits(s):
    c, b, v = s["case"], s["case"]["batch"], s["case"]["vocab"]
    x = s["x"].double().cpu().numpy()
    hist, off = s["hist"].cpu().numpy(), s["hist_off"].cpu().numpy()
    gen, pen = s["gen"].cpu().numpy(), s["pen"].double().cpu().numpy()
    bid, bias = s["bias_ids"].cpu().numpy(), s["bias"].double().cpu().numpy()
    boff = s["bias_off"].cpu().numpy()
    mask = None if s["mask"] is None else s["mask"].cpu().numpy().view(np.uint32)
    for i in range(b):
        z = x[i]
        if c["penalties"]:
            h = hist[off[i]:off[i + 1]]
            seen = np.unique(h[(h >= 0) & (h < v)])
            z[seen] = np.where(z[seen] > 0, z[seen] / pen[i, 0], z[seen] * pen[i, 0])
            h = h[gen[i]:]
            tok, count = np.unique(h[(h >= 0) & (h < v)], return_counts=True)
            z[tok] -= pen[i, 1] * count + pen[i, 2]
        np.add.at(z, bid[boff[i]:boff[i + 1]], bias[boff[i]:boff[i + 1]])
        if mask is not None and s["mask_row"][i] >= 0:
            bits = np.unpackbits(mask[int(s["mask_row"][i])].view(np.uint8), bitorder="little")
            z[bits[:v] == 0] = -math.inf
    return x


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "logits":
        return {"z": torch.from_numpy(_exact_logits(s))}
    cols = case["cols"]
    if kind == "quant":
        x = s["x"] if s["ids"] is None else s["x"].index_select(0, s["ids"])
        return {"v": _exact_round(x[:, :cols], cols)}
    x = _exact_round(s["x"], cols)
    if kind == "mul":
        out = torch.empty((case["n"], case["rows"]), dtype=torch.float64, device="cuda")
        for r in range(0, case["rows"], 16384):
            out[:, r:r + 16384] = x @ _exact_weights(s["w"][r:r + 16384], s["ws"][r:r + 16384],
                                                     cols).t()
        return {"y": out}
    out = torch.zeros(s["y"].shape, dtype=torch.float64, device="cuda")
    if kind == "sel":
        who = s["eid"].tolist()
        src = list(range(len(who))) if case["each"] else [p // case["topk"]
                                                          for p in range(len(who))]
    else:
        who = np.repeat(np.arange(case["experts"]), np.diff(s["stretch"])).tolist()
        src = s["act"].tolist()
    at = {}
    for p, e in enumerate(who):
        at.setdefault(e, []).append(p)
    for e, ps in at.items():
        w = _exact_weights(s["w"][e * case["rows"]:(e + 1) * case["rows"]],
                           s["ws"][e * case["rows"]:(e + 1) * case["rows"]], cols)
        out[torch.tensor(ps, device="cuda")] = x[torch.tensor([src[p] for p in ps],
                                                              device="cuda")] @ w.t()
    return {"y": out}
