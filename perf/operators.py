"""The 8-bit head of a model and what is read from its logits, as cases that can be timed and compared.

A case is one call of one operator: a tensor rounded to 8 bits with a scale for each block of 128, a product of two such
tensors, the log probabilities of given tokens with the entropy and the best alternatives, or the gradient of
these. Inputs are drawn on the GPU from a seed. `run` computes a case in its plain form, from elementary torch
operations in 32 bits (64 for float64 tensors), or, where `own` is set, by the framework's calls. These run on the
engine's stream, which nothing orders with torch's: a state's first run waits for its inputs, and whoever reads the
outputs, or gives the state's memory back, waits for the device first.
"""
import math

import torch

own = False

BLOCK = 128
F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
F8_MAX = {"e4m3": 448.0, "e5m2": 57344.0}
DT = {"f32": torch.float32, "f64": torch.float64, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f64": 8, "bf16": 2}


# ------------------------------------------------------------------------------------------
# the cases
# ------------------------------------------------------------------------------------------

def listed():
    return [
        # a large batch of activations on its way into an 8-bit product
        {"name": "quantize_row_8192x4096", "kind": "quantize", "rows": 8192, "cols": 4096, "dtype": "bf16",
         "format": "e4m3", "block": "row"},
        # a training batch of the convolutional net's dense layer, for the gradient of its weights
        {"name": "quantize_col_1000x1152", "kind": "quantize", "rows": 1000, "cols": 1152, "dtype": "f32",
         "format": "e5m2", "block": "col"},
        # one token through a square layer: the weights are read, nothing else counts
        {"name": "matmul_1x4096x4096", "kind": "matmul", "m": 1, "n": 4096, "k": 4096, "ta": False, "tb": True,
         "a_block": "row", "b_block": "tile", "a_format": "e4m3", "b_format": "e4m3", "out": "bf16", "layer": False},
        # a batch of tokens that are served together
        {"name": "matmul_64x8192x4096", "kind": "matmul", "m": 64, "n": 8192, "k": 4096, "ta": False, "tb": True,
         "a_block": "row", "b_block": "tile", "a_format": "e4m3", "b_format": "e4m3", "out": "bf16", "layer": False},
        # dense layer with bias and rectifier, weights stored as the graphs store them, sizes that no tile divides
        {"name": "matmul_layer_1000x625x1152", "kind": "matmul", "m": 1000, "n": 625, "k": 1152, "ta": False,
         "tb": False, "a_block": "row", "b_block": "tile", "a_format": "e4m3", "b_format": "e4m3", "out": "f32",
         "layer": True},
        # the gradient of a layer's weights: both operands are summed down their columns
        {"name": "matmul_dw_4096x4096x8192", "kind": "matmul", "m": 4096, "n": 4096, "k": 8192, "ta": True, "tb": False,
         "a_block": "col", "b_block": "col", "a_format": "e4m3", "b_format": "e5m2", "out": "f32", "layer": False},
        # the largest square product of the linear algebra sweep
        {"name": "matmul_8192", "kind": "matmul", "m": 8192, "n": 8192, "k": 8192, "ta": False, "tb": True,
         "a_block": "row", "b_block": "tile", "a_format": "e4m3", "b_format": "e4m3", "out": "bf16", "layer": False},
        # a classifier's batch: the smallest call
        {"name": "logprobs_256x10", "kind": "logprobs", "rows": 256, "vocab": 10, "dtype": "f32", "top": 1,
         "masked": 0.0, "padded": 0.0},
        # one step of a few sequences that are served together, some of the vocabulary not allowed
        {"name": "logprobs_8x131072", "kind": "logprobs", "rows": 8, "vocab": 131072, "dtype": "bf16", "top": 20,
         "masked": 0.25, "padded": 0.0},
        # scoring of whole texts, padded at their ends
        {"name": "logprobs_4096x32000", "kind": "logprobs", "rows": 4096, "vocab": 32000, "dtype": "f32", "top": 5,
         "masked": 0.0, "padded": 0.1},
        # the classifier's loss in the default type of the graphs
        {"name": "logprobs_diff_256x10", "kind": "diff", "rows": 256, "vocab": 10, "dtype": "f64", "entropy": False,
         "masked": 0.0, "padded": 0.0},
        # the gradient of a language model's loss with an entropy bonus
        {"name": "logprobs_diff_4096x32000", "kind": "diff", "rows": 4096, "vocab": 32000, "dtype": "bf16",
         "entropy": True, "masked": 0.0, "padded": 0.1},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["quantize", "quantize", "matmul", "matmul", "matmul", "matmul", "logprobs", "logprobs",
                       "logprobs", "diff", "diff"])
    if kind == "quantize":
        cols = _log(rng, 16, 16384)
        return {"kind": kind, "rows": _log(rng, 1, min(16384, (1 << 26) // cols)), "cols": cols,
                "dtype": rng.choice(["f32", "bf16"]), "format": rng.choice(["e4m3", "e4m3", "e5m2"]),
                "block": rng.choice(["row", "col", "tile"])}
    if kind == "matmul":
        # forward, gradient of the input, gradient of the weights; a layer's extents are often, not always, even
        step = rng.choice([1, 16, 64])
        m, n, k = (max(step, _log(rng, lo, 8192) // step * step) for lo in (1, 64, 64))
        use = rng.choice(["forward", "forward", "serve", "dx", "dw"])
        if use == "serve":
            m = _log(rng, 1, 64)
        c = {"kind": kind, "m": m, "n": n, "k": k, "ta": use == "dw", "tb": use in ("serve", "dx") or
             (use == "forward" and rng.random() < 0.5), "a_block": "col" if use == "dw" else rng.choice(["row", "row", "tile"])}
        c["b_block"] = "col" if use == "dw" else rng.choice(["tile", "tile", "row" if c["tb"] else "col"])
        return {**c, "a_format": rng.choice(["e4m3", "e4m3", "e5m2"]) if use == "dx" else "e4m3",
                "b_format": rng.choice(["e4m3", "e5m2"]) if use == "dw" else "e4m3",
                "out": "f32" if use == "dw" else rng.choice(["bf16", "f32"]),
                "layer": use == "forward" and rng.random() < 0.5}
    dtype = rng.choice(["f32", "bf16", "bf16", "f64"])
    vocab = _log(rng, 2, 200000)
    rows = _log(rng, 1, min(16384, (1 << 27) // vocab))
    c = {"kind": kind, "rows": rows, "vocab": vocab, "dtype": dtype}
    if kind == "logprobs":
        c["top"] = min(vocab, rng.choice([0, 1, 5, 20, 32]))
    else:
        c["entropy"] = rng.random() < 0.5
    return {**c, "masked": rng.choice([0.0, 0.0, 0.3]), "padded": rng.choice([0.0, 0.1])}


# ------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------

def _blocks_of(block):
    return {"row": (1, BLOCK), "col": (BLOCK, 1), "tile": (BLOCK, BLOCK)}[block]


def _up(n, d):
    return -(-n // d)


def _scale_shape(rows, cols, block):
    br, bc = _blocks_of(block)
    return _up(rows, br), _up(cols, bc)


def _over_blocks(x, block):
    """(row blocks, rows of one, column blocks, columns of one), padded with zeros."""
    br, bc = _blocks_of(block)
    rows, cols = x.shape
    x = torch.nn.functional.pad(x, (0, -cols % bc, 0, -rows % br))
    return x.view(x.shape[0] // br, br, x.shape[1] // bc, bc)


def _plain_quantize(x, fmt, block):
    rows, cols = x.shape
    b = _over_blocks(x.float(), block)
    amax = torch.where(torch.isfinite(b), b.abs(), 0.0).amax(dim=(1, 3), keepdim=True)
    part, e = torch.frexp(amax)  # part in [1/2, 1)
    e = e - {"e4m3": 9, "e5m2": 16}[fmt] + (part > 0.875).int()
    scale = torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), e.clamp(min=-126)), 1.0)
    q = (b / scale).view(b.shape[0] * b.shape[1], -1)[:rows, :cols].to(F8[fmt])
    return q.contiguous(), scale[:, 0, :, 0].contiguous()


def _values(rows, cols, g):
    """Values as layers hold them: normal, each row at a magnitude of its own, a few columns far above the rest."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    x *= torch.exp(torch.randn(rows, 1, generator=g, device="cuda"))
    return x.mul_(1.0 + 15.0 * (torch.rand(1, cols, generator=g, device="cuda") < 0.01).float())


def _logits(case, g):
    """Logits (fewer allowed classes in some cases: the others hold -Inf) and the tokens that are asked for."""
    rows, vocab, dt = case["rows"], case["vocab"], DT[case["dtype"]]
    x = torch.randn(rows, vocab, generator=g, device="cuda", dtype=torch.float64 if dt == torch.float64 else torch.float32)
    x = x.mul_(2.5)
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    if case["masked"]:
        gone = torch.rand(rows, vocab, generator=g, device="cuda") < case["masked"]
        gone.scatter_(1, t[:, None], False)
        x = x.masked_fill_(gone, -math.inf)
    if case["padded"]:
        t = torch.where(torch.rand(rows, generator=g, device="cuda") < case["padded"], -1, t)
    return x.to(dt), t


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": case}
    kind = case["kind"]

    def room(shape, dtype):
        return torch.empty(shape, device="cuda", dtype=dtype)

    if kind == "quantize":
        s["x"] = _values(case["rows"], case["cols"], g).to(DT[case["dtype"]])
        s["q"] = room((case["rows"], case["cols"]), F8[case["format"]])
        s["scales"] = room(_scale_shape(case["rows"], case["cols"], case["block"]), torch.float32)
    elif kind == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        s["a"], s["a_scales"] = _plain_quantize(_values(*((k, m) if case["ta"] else (m, k)), g), case["a_format"], case["a_block"])
        s["b"], s["b_scales"] = _plain_quantize(_values(*((n, k) if case["tb"] else (k, n)), g).mul_(k ** -0.5),
                                                case["b_format"], case["b_block"])
        s["bias"] = torch.randn(n, generator=g, device="cuda") if case["layer"] else None
        s["c"] = room((m, n), DT[case["out"]])
    else:
        s["x"], s["targets"] = _logits(case, g)
        rows, vocab = case["rows"], case["vocab"]
        stat = torch.float64 if case["dtype"] == "f64" else torch.float32
        if kind == "logprobs":
            for name in ("logp", "entropy", "lse"):
                s[name] = room((rows,), stat)
            s["top_logp"] = room((rows, case["top"]), stat) if case["top"] else None
            s["top_index"] = room((rows, case["top"]), torch.int64) if case["top"] else None
        else:
            # what the forward call has left, and the gradients that come down to it
            s["lse"], s["entropy"] = _statistics(s["x"].to(stat))
            on = s["targets"] >= 0
            s["grad_logp"] = torch.where(on, -torch.rand(rows, generator=g, device="cuda", dtype=stat), 0.0)
            s["grad_entropy"] = torch.where(on, -0.01 * torch.rand(rows, generator=g, device="cuda", dtype=stat), 0.0) \
                if case["entropy"] else None
            s["dx"] = room((rows, vocab), DT[case["dtype"]])
    return s


# ------------------------------------------------------------------------------------------
# the plain forms
# ------------------------------------------------------------------------------------------

def _statistics(x):
    """The log of the sum of exponentials of each row, and its entropy."""
    top = x.amax(dim=1, keepdim=True)
    d = x - top
    e = torch.exp(d)
    total = e.sum(dim=1)
    log_total = torch.log(total)
    return top[:, 0] + log_total, log_total - torch.where(e > 0, e * d, 0.0).sum(dim=1) / total


def _spread(scales, shape, block):
    """A scale for each value, from one for each block."""
    br, bc = _blocks_of(block)
    rows, cols = shape
    r = torch.arange(rows, device=scales.device) // br
    c = torch.arange(cols, device=scales.device) // bc
    return scales[r][:, c]


def _plain_matmul(s):
    case = s["case"]
    a = s["a"].float() * _spread(s["a_scales"], s["a"].shape, case["a_block"])
    b = s["b"].float() * _spread(s["b_scales"], s["b"].shape, case["b_block"])
    c = (a.T if case["ta"] else a) @ (b.T if case["tb"] else b)
    if case["layer"]:
        c = torch.clamp(c + s["bias"], min=0.0)
    return {"c": c.to(DT[case["out"]])}


def _plain_logprobs(s):
    case = s["case"]
    x = s["x"].to(torch.float64 if case["dtype"] == "f64" else torch.float32)
    lse, entropy = _statistics(x)
    t = s["targets"]
    logp = torch.where(t >= 0, x.gather(1, t.clamp(min=0)[:, None])[:, 0] - lse, 0.0)
    out = {"logp": logp, "entropy": entropy, "lse": lse}
    if case["top"]:
        if case["dtype"] == "f64":
            v, i = torch.sort(x, dim=1, descending=True, stable=True)
            v, i = v[:, :case["top"]], i[:, :case["top"]]
        else:
            # ties go to the lowest index: the value's order in the upper half of a key, the index in the lower
            bits = (x + 0.0).view(torch.int32)
            order = torch.where(bits >= 0, bits, bits ^ 0x7fffffff).long()
            key = order * (1 << 32) + ((1 << 32) - 1 - torch.arange(case["vocab"], device="cuda"))
            i = (1 << 32) - 1 - (torch.topk(key, case["top"], dim=1).values & 0xffffffff)
            v = x.gather(1, i)
        out["top_logp"], out["top_index"] = v - lse[:, None], i
    return out


def _plain_diff(s):
    case = s["case"]
    stat = torch.float64 if case["dtype"] == "f64" else torch.float32
    x, t, g = s["x"].to(stat), s["targets"], s["grad_logp"]
    d = x - s["lse"][:, None]
    p = torch.exp(d)
    dx = -g[:, None] * p
    if s["grad_entropy"] is not None:
        dx = dx - torch.where(p > 0, s["grad_entropy"][:, None] * p * (d + s["entropy"][:, None]), 0.0)
    dx.scatter_add_(1, t.clamp(min=0)[:, None], torch.where(t >= 0, g, 0.0)[:, None])
    return {"dx": dx.to(s["x"].dtype)}


# ------------------------------------------------------------------------------------------
# the framework's calls
# ------------------------------------------------------------------------------------------

_engine = None


def _handles(s):
    """The engine's handles of a state's tensors, which a program makes once beside the tensors, and after them: what
    torch's stream has still to write there, or to read from memory that came to the outputs, is waited for."""
    global _engine
    import numpy as np
    from gorgonia_b200 import BlockTensor, Engine, Tensor
    torch.cuda.current_stream().synchronize()
    if _engine is None:
        _engine = Engine(arena_bytes=1 << 30)
    case = s["case"]
    kind = {torch.float32: np.float32, torch.float64: np.float64, torch.int64: np.int64, torch.bfloat16: np.uint16,
            F8["e4m3"]: np.uint8, F8["e5m2"]: np.uint8}

    def handle(t):
        if t is None:
            return None
        h = Tensor(_engine, t.data_ptr(), t.shape, kind[t.dtype], owned=False)
        if t.dtype == torch.bfloat16:
            h.is_bf16 = True
        return h

    h = {name: handle(t) for name, t in s.items() if t is None or isinstance(t, torch.Tensor)}
    if case["kind"] == "quantize":
        h["blocks"] = BlockTensor(h["q"], h["scales"], case["format"], case["block"])
    if case["kind"] == "matmul":
        h["a"] = BlockTensor(h["a"], h["a_scales"], case["a_format"], case["a_block"])
        h["b"] = BlockTensor(h["b"], h["b_scales"], case["b_format"], case["b_block"])
    s["handles"] = h
    return h


def _own_run(s):
    h = s.get("handles") or _handles(s)
    case, e = s["case"], _engine
    if case["kind"] == "quantize":
        e.QuantizeBlocks(h["x"], h["blocks"])
        return {"q": s["q"], "scales": s["scales"]}
    if case["kind"] == "matmul":
        e.MatMulBlocks(h["a"], h["b"], h["c"], transA=case["ta"], transB=case["tb"], bias=h["bias"],
                       act="rectify" if case["layer"] else None)
        return {"c": s["c"]}
    if case["kind"] == "logprobs":
        e.TokenLogProbs(h["x"], h["targets"], h["logp"], entropy=h["entropy"], lse=h["lse"], top_logp=h["top_logp"],
                        top_index=h["top_index"])
        return {n: s[n] for n in ("logp", "entropy", "lse", "top_logp", "top_index") if s[n] is not None}
    e.TokenLogProbsDiff(h["x"], h["targets"], h["lse"], h["entropy"], h["grad_logp"], h["dx"],
                        grad_entropy=h["grad_entropy"])
    return {"dx": s["dx"]}


def run(s):
    if own:
        return _own_run(s)
    kind = s["case"]["kind"]
    if kind == "quantize":
        q, scales = _plain_quantize(s["x"], s["case"]["format"], s["case"]["block"])
        return {"q": q, "scales": scales}
    return {"matmul": _plain_matmul, "logprobs": _plain_logprobs, "diff": _plain_diff}[kind](s)


# ------------------------------------------------------------------------------------------
# what a case cannot do without, and its value in 64 bits
# ------------------------------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "quantize":
        n = case["rows"] * case["cols"]
        blocks = math.prod(_scale_shape(case["rows"], case["cols"], case["block"]))
        return {"bytes": n * (SIZE[case["dtype"]] + 1) + 4 * blocks, "flops": 2 * n}
    if kind == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        scales = math.prod(_scale_shape(*((k, m) if case["ta"] else (m, k)), case["a_block"])) + \
            math.prod(_scale_shape(*((n, k) if case["tb"] else (k, n)), case["b_block"]))
        return {"bytes": m * k + n * k + 4 * scales + m * n * SIZE[case["out"]] + (4 * n if case["layer"] else 0),
                "flops": 2 * m * n * k}
    n, stat = case["rows"] * case["vocab"], 8 if case["dtype"] == "f64" else 4
    if kind == "logprobs":
        return {"bytes": n * SIZE[case["dtype"]] + case["rows"] * (8 + 3 * stat + case["top"] * (8 + stat)), "flops": 6 * n}
    return {"bytes": 2 * n * SIZE[case["dtype"]] + case["rows"] * (8 + 4 * stat), "flops": (8 if case["entropy"] else 4) * n}


def _exact_quantize(s):
    case = s["case"]
    x = s["x"].double()
    rows, cols = x.shape
    br, bc = _blocks_of(case["block"])
    rb, cb = _up(rows, br), _up(cols, bc)
    whole = torch.zeros(rb * br, cb * bc, dtype=torch.float64, device="cuda")
    whole[:rows, :cols] = x
    tiles = whole.view(rb, br, cb, bc).transpose(1, 2)
    most = tiles.abs().flatten(2).max(dim=2).values
    # the least power of two that brings the largest magnitude inside the format
    power = torch.ceil(torch.log2(most / F8_MAX[case["format"]])).nan_to_num(0.0, 0.0, 0.0)
    power = torch.where(most > F8_MAX[case["format"]] * torch.exp2(power), power + 1, power)
    power = torch.where(most <= F8_MAX[case["format"]] * torch.exp2(power - 1), power - 1, power)
    scales = torch.where(most > 0, torch.exp2(power.clamp(min=-126)), 1.0)
    v = (tiles / scales[:, :, None, None]).transpose(1, 2).reshape(rb * br, cb * bc)[:rows, :cols]
    digits, low = {"e4m3": (3, -6), "e5m2": (2, -14)}[case["format"]]
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -40))).clamp(min=low) - digits)
    return {"q": torch.round(v / step) * step, "scales": scales}


def _exact_matmul(s):
    case = s["case"]

    def wide(q, scales, block):
        br, bc = _blocks_of(block)
        w = scales.double().repeat_interleave(br, 0)[:q.shape[0]].repeat_interleave(bc, 1)[:, :q.shape[1]]
        return w.mul_(q.float().double())

    a, b = wide(s["a"], s["a_scales"], case["a_block"]), wide(s["b"], s["b_scales"], case["b_block"])
    c = torch.matmul(a.t() if case["ta"] else a, b.t() if case["tb"] else b)
    if case["layer"]:
        c = torch.relu(c.add_(s["bias"].double()))
    return {"c": c}


def _exact_logprobs(s):
    case = s["case"]
    x = s["x"].double()
    lse = torch.logsumexp(x, dim=1)
    p = torch.exp(x - lse[:, None])
    entropy = -torch.special.xlogy(p, p).sum(dim=1)
    t = s["targets"]
    rows = torch.arange(case["rows"], device="cuda")
    logp = (x[rows, t.clamp(min=0)] - lse).masked_fill(t < 0, 0.0)
    out = {"logp": logp, "entropy": entropy, "lse": lse}
    if case["top"]:
        out["top_logp"] = torch.topk(x, case["top"], dim=1).values - lse[:, None]
        out["top_index"] = None
    return out


def _exact_diff(s):
    x, t = s["x"].double(), s["targets"]
    lse, g = s["lse"].double()[:, None], s["grad_logp"].double()[:, None]
    p = torch.exp(x - lse)
    hit = torch.zeros_like(p)
    rows = torch.nonzero(t >= 0)[:, 0]
    hit[rows, t[rows]] = 1.0
    dx = (hit - p) * g
    if s["grad_entropy"] is not None:
        h = s["grad_entropy"].double()[:, None]
        dx -= h * (torch.special.xlogy(p, p) + p * s["entropy"].double()[:, None])
    return {"dx": dx}


def exact(case, seed):
    s = prepare(case, seed)
    return {"quantize": _exact_quantize, "matmul": _exact_matmul, "logprobs": _exact_logprobs, "diff": _exact_diff}[case["kind"]](s)
