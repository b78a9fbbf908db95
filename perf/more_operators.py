"""A layer's operators in 8-bit floating point, as timing cases: the norm ahead
of it, routing with scores, biases and groups, and products whose blocks of 128
have a scale each.

Each case goes through the public C entry points the way an engine calls
them, or through the operators' plain forms:

  norm    residual addition, root-mean-square norm, floats and / or 8 bits with
          scales out (q4mi_rms_norm)
  route   logits to experts and weights: softmax or sigmoid scores, a bias for
          the choice, groups, top-k, renormalised, scaled (q4mi_route_scored)
  quant   rows (a scale for each 128 values) or weights (for each 128 x 128) to
          8-bit floating point (q4mi_f8_quant), read back as values
          (q4mi_f8_dequant)
  mul     y[t] = W . x[t], both sides in 8 bits (q4mi_f8_mul); up to sixteen
          float rows go in as they are, more are quantised first
  sel     every row through the expert that a list names (q4mi_f8_mul_sel):
          routed experts of a decode step
  id      packed rows, each expert's in one stretch (q4mi_f8_mul_id): routed
          experts of a prompt

A block's values are e4m3 codes times one fp32 scale.  Products take any scale;
the quantiser writes the least power of two that takes the block's largest
magnitude to at most 448 (at least 2^-120), so that the scaling is exact.  A row
of n values has nb = ceil(n / 128) blocks and 128 * nb bytes of codes, those past
n are 0.

Weights are N(0, 1/cols) in this format with scales of any size, activations
N(0,1) with a few large channels, prompts' routing Zipf.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

TYPES = {"f32": (0, torch.float32), "f16": (1, torch.float16), "bf16": (30, torch.bfloat16)}
F8, Q8 = 248, 8
FLOAT_ROWS = 16     # rows of float activations that q4mi_f8_mul takes as they are
EPS = 1e-6


def listed():
    return [
        # one decode token's hidden state: floats for the router, 8 bits for the experts
        {"name": "norm_token", "kind": "norm", "rows": 1, "cols": 2048, "x": "f32", "res": "f32",
         "y": "f32", "q": "f8"},
        # a prompt chunk ahead of its projections
        {"name": "norm_prompt", "kind": "norm", "rows": 8192, "cols": 4096, "x": "bf16",
         "res": "bf16", "y": "", "q": "f8"},
        # a decode token, plain softmax over the experts
        {"name": "route_token", "kind": "route", "tokens": 1, "experts": 128, "groups": 1,
         "topk_group": 1, "group_top": 1, "topk": 10, "sigmoid": False, "bias": False,
         "renorm": True, "scale": 1.0, "off": 0.0, "x": "f32"},
        # a prompt chunk, scores with a bias for balance and experts in groups
        {"name": "route_prompt", "kind": "route", "tokens": 8192, "experts": 512, "groups": 8,
         "topk_group": 4, "group_top": 2, "topk": 10, "sigmoid": True, "bias": True,
         "renorm": True, "scale": 2.5, "off": 0.0, "x": "f32"},
        # a four-token verify window's hidden states
        {"name": "quant_window", "kind": "quant", "rows": 4, "cols": 2048, "pad": 0,
         "block": 1, "x": "f32", "y": "f32"},
        # a projection's weights when a model is loaded
        {"name": "quant_weights", "kind": "quant", "rows": 16384, "cols": 4096, "pad": 0,
         "block": 128, "x": "bf16", "y": "bf16"},
        # the smallest product of a decode step: one short projection
        {"name": "mul_token", "kind": "mul", "n": 1, "rows": 2048, "cols": 2048, "x": "f32",
         "y": "f32"},
        # the LM head of a four-token verify window
        {"name": "mul_lm_head", "kind": "mul", "n": 4, "rows": 151936, "cols": 2048, "x": "f32",
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
        # gate and up of a prompt chunk's routed experts
        {"name": "id_prompt", "kind": "id", "tokens": 2048, "topk": 10, "experts": 512,
         "rows": 1024, "cols": 2048, "spare": 0, "x": "bf16", "y": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cols(rng):
    """Row lengths: mostly whole blocks, now and then any number."""
    if rng.random() < 0.3:
        return _log(rng, 1, 8192)
    return 128 * _log(rng, 1, 64)


def _draw(rng):
    kind = rng.choice(["norm", "route", "quant", "mul", "mul", "sel", "id"])
    c = {"kind": kind, "x": rng.choice(sorted(TYPES))}
    if kind == "route":
        groups = rng.choice([1, 1, 2, 4, 8, 16])
        each = _log(rng, 1, 1024 // groups)
        keep = rng.randint(1, groups)
        c.update(tokens=_log(rng, 1, 16384), experts=groups * each, groups=groups,
                 topk_group=keep, group_top=rng.choice([1, 2]),
                 topk=rng.randint(1, min(16, keep * each)), sigmoid=rng.random() < 0.6,
                 bias=rng.random() < 0.6, renorm=rng.random() < 0.7,
                 scale=rng.choice([1.0, 2.5]), off=rng.choice([0.0, 0.0, 0.3]))
        return c
    if kind == "norm":
        c.update(rows=_log(rng, 1, 16384), cols=_log(rng, 1, 256) * 32
                 if rng.random() < 0.7 else _log(rng, 1, 16384),
                 res=rng.choice(["", "f32", c["x"]]), y=rng.choice(["", "f32", c["x"]]),
                 q=rng.choice(["f8", "f8", "q8", ""]))
        if c["q"] == "q8" and c["cols"] % 32:
            c["q"] = "f8"
        if not c["y"] and not c["q"]:
            c["y"] = c["x"]
        return c
    c.update(y=rng.choice(sorted(TYPES)), cols=_cols(rng))
    if kind == "quant":
        c.update(rows=_log(rng, 1, 16384), pad=rng.choice([0, 0, 8, rng.randint(1, 70)]),
                 block=rng.choice([1, 1, 128]))
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
    if case["kind"] not in ("mul", "sel", "id"):
        return 0
    held = case.get("experts", 1)
    if case["kind"] == "sel":
        held = max(held, case["tokens"] * case["topk"])
    return held * case["rows"] * case["cols"]


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        c = _draw(rng)
        if _cost(c) <= most and _weights_held(c) <= 1.1e9:
            return c


# ------------------------------------------------------------------ sizes

def _blocks(cols):
    return (cols + 127) // 128


def _size(name):
    return TYPES[name][1].itemsize if name else 0


def work(case):
    """Each input once, each output once; a product's multiplications and
    additions over the values of its rows."""
    kind = case["kind"]
    if kind == "route":
        n = case["tokens"] * case["experts"]
        return {"bytes": n * _size(case["x"]) + 8 * case["tokens"] * case["topk"] +
                (4 * case["experts"] if case["bias"] else 0), "flops": 4 * n}
    if kind == "norm":
        n = case["rows"] * case["cols"]
        q = {"f8": 1 + 4 / 128, "q8": 1 + 4 / 32, "": 0}[case["q"]]
        return {"bytes": n * (_size(case["x"]) + 2 * _size(case["res"]) + _size(case["y"]) + q) +
                4 * case["cols"], "flops": 5 * n}
    nb = _blocks(case["cols"])
    if kind == "quant":
        n = case["rows"] * case["cols"]
        scales = 4 * nb * -(-case["rows"] // case["block"])
        return {"bytes": n * (_size(case["x"]) + 2 + _size(case["y"])) + 2 * scales,
                "flops": 2 * n}
    if kind == "mul":
        n, xrows, held = case["n"], case["n"], 1
    else:
        n = case["tokens"] * case["topk"]
        xrows = n if case.get("each") else case["tokens"]
        held = min(n, case["experts"])
    w = case["rows"] * case["cols"] + 4 * nb * -(-case["rows"] // 128)
    return {"bytes": held * w + xrows * case["cols"] * _size(case["x"]) +
            n * case["rows"] * _size(case["y"]),
            "flops": 2 * n * case["rows"] * case["cols"]}


# ------------------------------------------------------------- plain forms

def _plain_quant(x, block):
    """Rows of 32-bit floats -> codes [rows][128 nb] and scales
    [ceil(rows / block)][nb]."""
    rows, cols = x.shape
    nb, rb = _blocks(cols), -(-rows // block)
    v = torch.zeros((rb * block, nb * 128), dtype=torch.float32, device=x.device)
    v[:rows, :cols] = x
    v = v.view(rb, block, nb, 128)
    top = v.abs().amax((1, 3))
    bad = ~torch.isfinite(v).all(3).all(1)
    part, exp = torch.frexp(torch.where(bad, torch.ones_like(top), top))
    exp = (exp - 9 + (part > 0.875).int()).clamp(min=-120)      # 448 = 0.875 * 2^9
    q = torch.ldexp(v, -exp[:, None, :, None]).to(torch.float8_e4m3fn)
    q = torch.where(bad[:, None, :, None], 0, q.view(torch.uint8)).to(torch.uint8)
    s = torch.ldexp(torch.ones_like(top), exp)
    s = torch.where(bad, torch.full_like(s, math.nan), s)
    return q.view(rb * block, nb * 128)[:rows].contiguous(), s


def _plain_values(codes, scales, cols, block):
    """What codes and scales stand for, in 32 bits."""
    v = codes.view(torch.float8_e4m3fn).float()
    s = scales.repeat_interleave(block, 0)[:v.shape[0]].repeat_interleave(128, 1)
    return (v * s)[:, :cols]


def _plain_norm(s):
    c = s["case"]
    h = s["x"].float()
    out = {}
    if c["res"]:
        out["sum"] = (h + s["res"].float()).to(TYPES[c["res"]][1])
        h = out["sum"].float()
    mean = h.double().square().sum(1, keepdim=True) / c["cols"]
    y = h * (1 / torch.sqrt(mean + EPS)).float() * s["w"]
    if c["y"]:
        out["y"] = y.to(TYPES[c["y"]][1])
    if c["q"] == "f8":
        codes, out["scales"] = _plain_quant(y, 1)
        out["codes"] = codes.view(torch.float8_e4m3fn)
    elif c["q"] == "q8":
        g = y.view(c["rows"], -1, 32)
        top = g.abs().amax(2)
        inv = torch.where(top > 0, (127 / top.double()).float(), torch.zeros_like(top))
        out["codes"] = torch.round(g * inv[..., None]).to(torch.int8).view(c["rows"], -1)
        out["scales"] = (top.double() / 127).float()
    return out


def _plain_route(s):
    """Scores in 64 bits (two close ones must not change places); the sorts
    keep equal values in order."""
    c = s["case"]
    z = s["x"].double()
    if c["sigmoid"]:
        score = 1 / (1 + torch.exp(-z))
    else:
        e = torch.exp(z - z.amax(1, keepdim=True))
        score = e / e.sum(1, keepdim=True)
    key = score + s["bias"].double() if c["bias"] else score
    key = torch.where(torch.isneginf(z), torch.full_like(key, -math.inf), key)
    if c["groups"] > 1:
        g = key.view(c["tokens"], c["groups"], -1)
        best = torch.sort(g, dim=2, descending=True).values[:, :, :c["group_top"]]
        best = torch.where(torch.isneginf(best), torch.zeros_like(best), best).sum(2)
        best = torch.where(torch.isneginf(g.amax(2)), torch.full_like(best, -math.inf), best)
        first = torch.sort(best, dim=1, descending=True, stable=True).indices[:, :c["topk_group"]]
        keep = torch.zeros_like(best, dtype=torch.bool).scatter_(1, first, True)
        key = torch.where(keep[..., None], g, torch.full_like(g, -math.inf)).view_as(key)
    order = torch.sort(key, dim=1, descending=True, stable=True)
    ids = order.indices[:, :c["topk"]]
    none = torch.isneginf(order.values[:, :c["topk"]])
    w = torch.where(none, torch.zeros_like(score[:, :1]), score.gather(1, ids))
    if c["renorm"]:
        total = w.sum(1, keepdim=True)
        w = torch.where(total > 0, w / total, torch.zeros_like(w))
    return {"ids": torch.where(none, torch.full_like(ids, -1), ids).int(),
            "wts": (w * c["scale"]).float()}


def _plain(s):
    c, kind = s["case"], s["case"]["kind"]
    if kind == "norm":
        return _plain_norm(s)
    if kind == "route":
        return _plain_route(s)
    y, cols = TYPES[c["y"]][1], c["cols"]
    codes, scales = _plain_quant(s["x"][:, :cols].float(), c.get("block", 1))
    x = _plain_values(codes, scales, cols, c.get("block", 1))
    if kind == "quant":
        return {"v": x.to(y)}
    if kind == "mul":
        return {"y": (x @ _plain_values(s["w"][0], s["ws"][0], cols, 128).t()).to(y)}
    if kind == "sel":
        e = s["eid"].long()
        w = s["w"][e].view(torch.float8_e4m3fn)[:, :, :cols].float()
        ws = s["ws"][e].repeat_interleave(128, 1)[:, :c["rows"]]
        w *= ws.repeat_interleave(128, 2)[:, :, :cols]
        x = x if c["each"] else x.repeat_interleave(c["topk"], 0)
        return {"y": torch.matmul(w, x[..., None])[..., 0].to(y)}
    out = s["y"].float()
    x = x[s["act"].long()]
    for e in range(c["experts"]):
        lo, hi = s["stretch"][e], s["stretch"][e + 1]
        if hi > lo:
            out[lo:hi] = x[lo:hi] @ _plain_values(s["w"][e], s["ws"][e], cols, 128).t()
    return {"y": out.to(y)}


# ----------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _weights(experts, rows, cols, gen):
    """Matrices about N(0, 1/cols) in 8 bits: codes [experts][rows][128 nb], scales
    [experts][ceil(rows / 128)][nb] of any mantissa, as another quantiser's."""
    nb, rb = _blocks(cols), -(-rows // 128)
    codes = torch.empty((experts, rows, nb * 128), dtype=torch.uint8, device="cuda")
    scales = torch.empty((experts, rb, nb), dtype=torch.float32, device="cuda")
    step = max(1, (1 << 26) // cols // 128) * 128
    for e in range(experts):
        for r in range(0, rows, step):
            n = min(step, rows - r)
            v = torch.randn((n, cols), device="cuda", generator=gen) / math.sqrt(cols)
            codes[e, r:r + n], scales[e, r // 128:(r + n + 127) // 128] = _plain_quant(v, 128)
    scales *= 0.75 + 0.5 * torch.rand(scales.shape, device="cuda", generator=gen)
    return codes, scales


def _activations(rows, cols, name, gen):
    """N(0,1) with about one channel in a hundred at twenty times the size."""
    x = torch.randn((rows, cols), device="cuda", generator=gen)
    x *= 1 + 19 * (torch.rand(cols, device="cuda", generator=gen) < 0.01)
    return x.to(TYPES[name][1])


def _new(rows, cols, block=1):
    """Room for the codes and scales of quantised rows."""
    nb = _blocks(cols)
    return (torch.empty((rows, nb * 128), dtype=torch.uint8, device="cuda"),
            torch.empty((-(-rows // block), nb), dtype=torch.float32, device="cuda"))


def _zipf(rng, tokens, topk, experts):
    """Each token's distinct experts, by Zipf popularity (exponent 1.1)."""
    popular = rng.permutation(experts)
    key = rng.gumbel(size=(tokens, experts)) - 1.1 * np.log1p(popular)[None]
    return np.argsort(-key, axis=1, kind="stable")[:, :topk]


def _prepare_norm(case, gen):
    rows, cols = case["rows"], case["cols"]
    s = {"x": _activations(rows, cols, case["x"], gen)}
    s["w"] = 1 + 0.2 * torch.randn(cols, device="cuda", generator=gen)
    s["res"] = s["sum"] = s["y"] = s["codes"] = s["scales"] = None
    if case["res"]:
        s["res"] = _activations(rows, cols, case["res"], gen)
        s["sum"] = torch.empty_like(s["res"])
    if case["y"]:
        s["y"] = torch.empty((rows, cols), dtype=TYPES[case["y"]][1], device="cuda")
    if case["q"] == "f8":
        s["codes"], s["scales"] = _new(rows, cols)
    elif case["q"] == "q8":
        s["codes"] = torch.empty((rows, cols), dtype=torch.int8, device="cuda")
        s["scales"] = torch.empty((rows, cols // 32), dtype=torch.float32, device="cuda")
    return s


def _prepare_route(case, gen):
    t, e = case["tokens"], case["experts"]
    # some experts are liked by most tokens
    z = torch.randn((t, e), device="cuda", generator=gen)
    z += torch.randn(e, device="cuda", generator=gen)
    s = {"x": z.to(TYPES[case["x"]][1]), "bias": None}
    if case["off"]:
        # experts that this engine does not hold
        gone = torch.rand(e, device="cuda", generator=gen) < case["off"]
        s["x"][:, gone] = -math.inf
        s["x"][:, 0] = 0
    if case["bias"]:
        s["bias"] = 0.1 * torch.randn(e, device="cuda", generator=gen)
    s["ids"] = torch.empty((t, case["topk"]), dtype=torch.int32, device="cuda")
    s["wts"] = torch.empty((t, case["topk"]), dtype=torch.float32, device="cuda")
    return s


def prepare(case, seed):
    """What an engine has in hand: weights in 8 bits, activations, lists and
    room for the outputs."""
    gen, kind = _gen(seed), case["kind"]
    if kind == "norm":
        s = _prepare_norm(case, gen)
    elif kind == "route":
        s = _prepare_route(case, gen)
    elif kind == "quant":
        rows, cols = case["rows"], case["cols"]
        s = {"x": _activations(rows, cols + case["pad"], case["x"], gen),
             "v": torch.empty((rows, cols), dtype=TYPES[case["y"]][1], device="cuda")}
        s["xq"], s["xs"] = _new(rows, cols, case["block"])
    else:
        rng = np.random.default_rng(seed)
        n = case["n"] if kind == "mul" else case["tokens"] * case["topk"]
        xrows = n if kind == "mul" or case.get("each") else case["tokens"]
        s = {"x": _activations(xrows, case["cols"], case["x"], gen)}
        s["xq"], s["xs"] = _new(xrows, case["cols"])
        s["w"], s["ws"] = _weights(case.get("experts", 1), case["rows"], case["cols"], gen)
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
    return s


# ------------------------------------------------------------ one pass

_loaded = None


def _q4mi():
    """The package, its library launching on torch's stream."""
    global _loaded
    if _loaded is None:
        path = os.path.join(os.getcwd(), "suzuku-engine-q4_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        import q4mi
        q4mi.use_torch_stream()
        _loaded = q4mi
    return _loaded


def _p(t):
    return None if t is None else t.data_ptr()


def _quantise(q, s, block=1):
    c, x = s["case"], s["x"]
    q.check(q.lib().q4mi_f8_quant(x.data_ptr(), TYPES[c["x"]][0], x.shape[1], None, x.shape[0],
                                  c["cols"], block, s["xq"].data_ptr(), s["xs"].data_ptr()),
            "quantise")


def _run_norm(q, s):
    c, cols = s["case"], s["case"]["cols"]
    res = c["res"] or "f32"
    q.check(q.lib().q4mi_rms_norm(
        s["x"].data_ptr(), TYPES[c["x"]][0], cols, _p(s["res"]), _p(s["sum"]), TYPES[res][0],
        cols, s["w"].data_ptr(), 0, EPS, c["rows"], cols, _p(s["y"]),
        TYPES[c["y"] or "f32"][0], cols, {"f8": F8, "q8": Q8, "": 0}[c["q"]], _p(s["codes"]),
        _p(s["scales"])), "norm")
    out = {k: s[k] for k in ("sum", "y", "codes", "scales") if s[k] is not None}
    if c["q"] == "f8":
        out["codes"] = s["codes"].view(torch.float8_e4m3fn)
    return out


def run(s):
    if not own:
        return _plain(s)
    q, c, kind = _q4mi(), s["case"], s["case"]["kind"]
    lib = q.lib()
    if kind == "norm":
        return _run_norm(q, s)
    xt = TYPES[c["x"]][0]
    if kind == "route":
        q.check(lib.q4mi_route_scored(
            s["x"].data_ptr(), xt, c["experts"], c["tokens"], c["experts"], _p(s["bias"]),
            int(c["sigmoid"]), c["groups"], c["topk_group"], c["group_top"], c["topk"],
            c["renorm"], c["scale"], s["ids"].data_ptr(), s["wts"].data_ptr(), None, c["topk"],
            -1, None), "route")
        return {"ids": s["ids"], "wts": s["wts"]}
    yt = TYPES[c["y"]][0]
    if kind == "quant":
        _quantise(q, s, c["block"])
        q.check(lib.q4mi_f8_dequant(s["xq"].data_ptr(), s["xs"].data_ptr(), None, c["rows"],
                                    c["cols"], c["block"], s["v"].data_ptr(), yt, c["cols"]),
                "values")
        return {"v": s["v"]}
    w, ws, rows, cols, y = s["w"], s["ws"], c["rows"], c["cols"], s["y"]
    if kind == "mul":
        x, xs = s["x"], None
        if c["n"] > FLOAT_ROWS:
            _quantise(q, s)
            x, xs, xt = s["xq"], s["xs"], F8
        q.check(lib.q4mi_f8_mul(w.data_ptr(), ws.data_ptr(), rows, cols, x.data_ptr(), _p(xs), xt,
                                cols, c["n"], y.data_ptr(), yt, rows), "product")
    elif kind == "sel":
        q.check(lib.q4mi_f8_mul_sel(
            w.data_ptr(), ws.data_ptr(), rows, cols, w.stride(0), 4 * ws.stride(0), c["experts"],
            s["x"].data_ptr(), None, xt, cols, 1 if c["each"] else c["topk"],
            s["eid"].data_ptr(), c["tokens"] * c["topk"], y.data_ptr(), yt, rows), "experts")
    else:
        _quantise(q, s)
        q.check(lib.q4mi_f8_mul_id(
            w.data_ptr(), ws.data_ptr(), rows, cols, w.stride(0), 4 * ws.stride(0), c["experts"],
            s["xq"].data_ptr(), s["xs"].data_ptr(), c["tokens"], s["act"].data_ptr(),
            s["bounds"].data_ptr(), len(y), y.data_ptr(), yt, rows), "experts")
    return {"y": y}


# --------------------------------------------------------- in 64 bits

def _grid(a):
    """The nearest values of sign, four exponent bits (bias 7) and three
    mantissa bits, ties to even: multiples of an eighth of the power of two
    below, of 2^-9 under 2^-6."""
    e = torch.floor(torch.log2(a.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(e - 3)
    return (torch.round(a / step) * step).clamp(-448.0, 448.0)


def _exact_round(x, block):
    """Rows as the 8-bit format holds them: codes' values [rows][128 nb] and
    scales [ceil(rows / block)][nb]."""
    rows, cols = x.shape
    nb, rb = _blocks(cols), (rows + block - 1) // block
    v = torch.nn.functional.pad(x.double(), (0, nb * 128 - cols, 0, rb * block - rows))
    v = v.reshape(rb, block, nb, 128).transpose(1, 2)       # [row block][column block][128..]
    most = torch.clamp(v.abs().flatten(2).max(2).values / 448, min=2.0 ** -120)
    scale = torch.exp2(torch.ceil(torch.log2(most)))
    code = _grid(v / scale[:, :, None, None]).transpose(1, 2).reshape(rb * block, nb * 128)
    return code[:rows], scale


def _exact_values(x, block):
    code, scale = _exact_round(x, block)
    nb = scale.shape[1]
    per = torch.repeat_interleave(scale, block, 0)[:len(code)]
    return (code.reshape(-1, nb, 128) * per[:, :, None]).reshape(len(code), -1)[:, :x.shape[1]]


def _exact_weights(codes, scales, cols):
    """Weights from their bits: sign, four exponent bits, three mantissa bits."""
    q = codes.to(torch.int64)
    e, m = (q >> 3) & 15, (q & 7).double()
    mag = torch.where(e == 0, m / 512, torch.exp2(e.double() - 7) * (1 + m / 8))
    mag = torch.where(q >= 128, -mag, mag)
    rows = torch.arange(codes.shape[0], device=codes.device) // 128
    per = scales.double()[rows]
    return (mag.reshape(len(rows), -1, 128) * per[:, :, None]).reshape(len(rows), -1)[:, :cols]


def _exact_norm(s):
    c = s["case"]
    h = s["x"].double()
    out = {}
    if c["res"]:
        out["sum"] = h + s["res"].double()
        h = out["sum"].to(TYPES[c["res"]][1]).double()      # the norm is of what is kept
    y = h / torch.sqrt((h * h).mean(1, keepdim=True) + EPS) * s["w"].double()
    if c["y"]:
        out["y"] = y
    if c["q"] == "f8":
        out["codes"], out["scales"] = _exact_round(y, 1)
    elif c["q"] == "q8":
        out["codes"] = None
        out["scales"] = y.abs().reshape(c["rows"], -1, 32).max(2).values / 127
    return out


def _exact_route(s):
    c = s["case"]
    z = s["x"].double().cpu().numpy()
    with np.errstate(over="ignore"):
        if c["sigmoid"]:
            score = 1 / (1 + np.exp(-z))
        else:
            score = np.exp(z - z.max(1, keepdims=True))
            score /= score.sum(1, keepdims=True)
    key = score.copy()
    if c["bias"]:
        key += s["bias"].double().cpu().numpy()
    key[np.isneginf(z)] = -np.inf
    t, g = c["tokens"], c["groups"]
    if g > 1:
        v = key.reshape(t, g, -1)
        best = -np.sort(-v, 2)[:, :, :c["group_top"]]
        some = best[:, :, 0] > -np.inf
        best = np.where(np.isneginf(best), 0, best).sum(2)
        best[~some] = -np.inf
        rank = np.argsort(np.argsort(-best, 1, kind="stable"), 1)
        key = np.where((rank < c["topk_group"])[:, :, None], v, -np.inf).reshape(t, -1)
    ids = np.argsort(-key, 1, kind="stable")[:, :c["topk"]]
    none = np.isneginf(np.take_along_axis(key, ids, 1))
    w = np.where(none, 0, np.take_along_axis(score, ids, 1))
    if c["renorm"]:
        total = w.sum(1, keepdims=True)
        w = np.divide(w, total, out=np.zeros_like(w), where=total > 0)
    return {"ids": torch.from_numpy(np.where(none, -1, ids).astype(np.int32)),
            "wts": torch.from_numpy(w * c["scale"])}


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "norm":
        return _exact_norm(s)
    if kind == "route":
        return _exact_route(s)
    cols = case["cols"]
    x = _exact_values(s["x"][:, :cols], case.get("block", 1))
    if kind == "quant":
        return {"v": x}
    if kind == "mul":
        out = torch.empty((case["n"], case["rows"]), dtype=torch.float64, device="cuda")
        for r in range(0, case["rows"], 16384):
            out[:, r:r + 16384] = x @ _exact_weights(
                s["w"][0, r:r + 16384], s["ws"][0, r // 128:r // 128 + 128], cols).t()
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
        w = _exact_weights(s["w"][e], s["ws"][e], cols)
        out[torch.tensor(ps, device="cuda")] = x[torch.tensor([src[p] for p in ps],
                                                              device="cuda")] @ w.t()
    return {"y": out}
