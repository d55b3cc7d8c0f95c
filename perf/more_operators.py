"""The operators of a layer whose projections run in 8-bit integers, as they are timed.

norm     the residual's addition, RMSNorm, and the row in 8 bits with its scale
swiglu   silu(gate) * up, and the row in 8 bits with its scale
quant    rows (tokens, or a weight's channels) in 8 bits with their scales
product  the product of 8-bit rows and 8-bit channels, scaled, with a bias

`run` computes them in plain torch (own = False) or with myos.dev (own = True).
8-bit values come back as what they stand for, q * scale. A row's scale and the
border between two of its 256 steps are places where 32 bits would decide by
their rounding, so the plain forms of the first three compute in 64.
"""
import math
import sys

import torch

own = False

PKG = "an-operating-system-for-ai-models-and-tensor-inference_b200"
SMALLEST = 2.0**-126  # the smallest scale: that of a row of zeros
EPS = 1e-6


def _dev():
    if PKG not in sys.path:
        sys.path.insert(0, PKG)
    from myos import dev

    return dev


# ---------------------------------------------------------------- cases
def listed():
    return [
        # one chat request in decode: the launch is what counts
        {"name": "norm 1 x 1536", "op": "norm", "rows": 1, "width": 1536, "x": "f32", "add": True},
        # a decode step of 64 sequences, 14B width, the projection's rows in bf16
        {"name": "norm 64 x 5120 bf16", "op": "norm", "rows": 64, "width": 5120, "x": "bf16", "add": True},
        # prompts of many requests in one chunk
        {"name": "norm 8191 x 5120", "op": "norm", "rows": 8191, "width": 5120, "x": "f32", "add": True},
        # one token between the 1.5B MLP's two products
        {"name": "swiglu 1 x 8960", "op": "swiglu", "rows": 1, "width": 8960, "x": "f32"},
        # the same for prompts, 14B width
        {"name": "swiglu 4099 x 13824 bf16", "op": "swiglu", "rows": 4099, "width": 13824, "x": "bf16"},
        # the attention's output before its projection, 61 sequences in decode
        {"name": "quant 61 x 1536", "op": "quant", "rows": 61, "width": 1536, "x": "f32"},
        # a weight at load time: a scale for each of the 14B gate and up channels
        {"name": "quant 27648 x 5120 bf16", "op": "quant", "rows": 27648, "width": 5120, "x": "bf16"},
        # q, k and v of one 1.5B token
        {"name": "product 1 x 1536 x 2048", "op": "product", "rows": 1, "k": 1536, "n": 2048, "bias": True, "out": "f32"},
        # one token's logits: 233 MB of weights
        {"name": "product 1 x 1536 x 151936", "op": "product", "rows": 1, "k": 1536, "n": 151936, "bias": False, "out": "f32"},
        # down_proj of 64 sequences in decode, 14B sizes
        {"name": "product 64 x 13824 x 5120", "op": "product", "rows": 64, "k": 13824, "n": 5120, "bias": False, "out": "f32"},
        # q, k and v of a short chunk of prompts
        {"name": "product 333 x 5120 x 7168", "op": "product", "rows": 333, "k": 5120, "n": 7168, "bias": True, "out": "f32"},
        # gate and up of a long chunk
        {"name": "product 4097 x 5120 x 27648", "op": "product", "rows": 4097, "k": 5120, "n": 27648, "bias": False, "out": "bf16"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["norm", "swiglu", "quant", "product", "product"])
    x = rng.choice(["f32", "bf16"])
    if op == "product":
        rows, k = _log(rng, 1, 4097), _log(rng, 64, 13824)
        most = min(151936, 4097 * 5120 * 27648 // (rows * k), 151936 * 1536 // k, 4097 * 27648 // rows // (2 if x == "f32" else 1))
        return {"op": op, "rows": rows, "k": k, "n": _log(rng, 64, max(64, most)), "bias": rng.random() < 0.5, "out": x}
    width = rng.choice([8960, 13824] if op == "swiglu" else [1536, 5120, 8960, 13824])
    width = rng.choice([width, width, width, _log(rng, 100, 16384)])
    case = {"op": op, "rows": _log(rng, 1, 8191 * 5120 // width), "width": width, "x": x}
    return {**case, "add": rng.random() < 0.7} if op == "norm" else case


# ---------------------------------------------------------------- inputs
_T = {"f32": torch.float32, "bf16": torch.bfloat16}


def _rows(rows, width, dtype):
    """Rows that begin at multiples of 16 bytes, whatever the width."""
    per = 16 // torch.empty(0, dtype=dtype).element_size()
    return torch.zeros(rows, -(-width // per) * per, dtype=dtype, device="cuda")[:, :width]


def _values(gen, rows, width, dtype, size):
    """Activations: each channel with a size of its own, a few of them far above the others."""
    channel = torch.exp(0.5 * torch.randn(width, device="cuda", generator=gen)) * size
    channel[torch.randint(width, (max(1, width // 1000),), device="cuda", generator=gen)] *= 12
    x = _rows(rows, width, dtype)
    x.copy_(torch.randn(rows, width, device="cuda", generator=gen) * channel)
    return x


def _bytes(gen, rows, width):
    """Rows as a scale for each row leaves them: the largest values near 127, most of them small."""
    x = _rows(rows, width, torch.int8)
    x.copy_((torch.randn(rows, width, device="cuda", generator=gen) * 30).round_().clamp_(-127, 127))
    return x


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, t, s = case["op"], case["rows"], {"case": case}
    if op == "product":
        k, n = case["k"], case["n"]
        s.update(a=_bytes(gen, t, k), w=_bytes(gen, n, k), bias=torch.randn(n, device="cuda", generator=gen) if case["bias"] else None)
        s["a_scales"] = torch.rand(t, device="cuda", generator=gen) * 0.05 + 0.01
        s["w_scales"] = (torch.rand(n, device="cuda", generator=gen) + 0.2) * (0.03 / math.sqrt(k))
        s["out"] = torch.zeros(t, n, dtype=_T[case["out"]], device="cuda")
        return s
    width, dtype = case["width"], _T[case["x"]]
    s["x"] = _values(gen, t, 2 * width if op == "swiglu" else width, dtype, 0.02 if op == "quant" else 1.0)
    s.update(q=_rows(t, width, torch.int8), scales=torch.zeros(t, device="cuda"))
    if op == "norm":
        s["gamma"] = (1 + 0.3 * torch.randn(width, device="cuda", generator=gen)).bfloat16()
        s["residual"] = _values(gen, t, width, torch.float32, 3.0) if case["add"] else None
        s["total"] = _rows(t, width, torch.float32) if case["add"] else None
    return s


# ---------------------------------------------------------------- one pass
def run(s):
    op = s["case"]["op"]
    if own:
        return _run_own(s, op)
    return {"norm": _norm, "swiglu": _swiglu, "quant": _quant, "product": _product}[op](s)


def _run_own(s, op):
    dev = _dev()
    if op == "product":
        dev.matmul_i8(s["out"], s["a"], s["a_scales"], s["w"], s["w_scales"], bias=s["bias"])
        return {"out": s["out"]}
    if op == "norm":
        dev.add_norm_quant(s["q"], s["scales"], s["x"], s["gamma"], residual=s["residual"], total=s["total"], eps=EPS)
    elif op == "swiglu":
        dev.swiglu_quant(s["q"], s["scales"], s["x"])
    else:
        dev.quant_rows(s["q"], s["scales"], s["x"])
    out = {"y": s["q"] * s["scales"][:, None], "scales": s["scales"]}
    return {**out, "total": s["total"]} if op == "norm" and s["total"] is not None else out


def _stepped(y):
    """y [rows, width] f64 -> the values that its 8 bits stand for, and the scales."""
    scales = (y.abs().amax(1) / 127).float().clamp(min=SMALLEST)
    steps = (y / scales.double()[:, None]).round()
    return {"y": steps.float() * scales[:, None], "scales": scales}


def _norm(s):
    x = s["x"].float()
    if s["residual"] is not None:
        x = x + s["residual"]
    y = x.double()
    inv = 1.0 / torch.sqrt((y * y).mean(1, keepdim=True) + EPS)
    out = _stepped(s["gamma"].double() * (y * inv))
    return {**out, "total": x} if s["residual"] is not None else out


def _swiglu(s):
    gate, up = s["x"].double().split(s["case"]["width"], 1)
    return _stepped(gate / (1.0 + torch.exp(-gate)) * up)


def _quant(s):
    return _stepped(s["x"].double())


def _product(s):
    x = torch.matmul(s["a"].float(), s["w"].float().T) * s["a_scales"][:, None] * s["w_scales"]
    if s["bias"] is not None:
        x = x + s["bias"]
    return {"out": x.to(s["out"].dtype)}


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    t = case["rows"]
    if case["op"] == "product":
        k, n = case["k"], case["n"]
        return {"bytes": t * k + n * k + t * n * (4 if case["out"] == "f32" else 2) + 4 * t + 4 * n * (2 if case["bias"] else 1), "flops": 2 * t * n * k}
    each = 4 if case["x"] == "f32" else 2  # read; the 8-bit row and its f32 values are written
    if case["op"] == "norm":
        return {"bytes": t * case["width"] * (each + 5 + (8 if case["add"] else 0)) + 2 * case["width"] + 4 * t, "flops": 8 * t * case["width"]}
    if case["op"] == "swiglu":
        return {"bytes": t * case["width"] * (2 * each + 5) + 4 * t, "flops": 10 * t * case["width"]}
    return {"bytes": t * case["width"] * (each + 5) + 4 * t, "flops": 4 * t * case["width"]}


# ---------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "product":
        parts = []
        for rows in range(0, case["n"], 16384):  # a block of channels at a time
            w = s["w"][rows : rows + 16384].double() * s["w_scales"][rows : rows + 16384].double()[:, None]
            parts.append(torch.einsum("tk,nk->tn", s["a"].double(), w))
        x = torch.cat(parts, 1) * s["a_scales"].double()[:, None]
        return {"out": x if s["bias"] is None else x + s["bias"].double()}
    parts = []
    for rows in range(0, case["rows"], 4096):
        x = s["x"][rows : rows + 4096].double()
        total = None
        if case["op"] == "norm":
            if s["residual"] is not None:
                # the residual stream is kept in 32 bits: what is normed is the sum as it is kept
                total = x + s["residual"][rows : rows + 4096].double()
                x = total.float().double()
            x = x * torch.pow(x.pow(2).sum(1, keepdim=True) / case["width"] + EPS, -0.5) * s["gamma"].double()
        elif case["op"] == "swiglu":
            x = x[:, : case["width"]] * torch.sigmoid(x[:, : case["width"]]) * x[:, case["width"] :]
        # a scale is a 32-bit number, and the steps are taken with that number
        scale = torch.maximum(x.max(1).values, -x.min(1).values).div(127.0).float().double().clamp_(min=SMALLEST)
        steps = torch.div(x, scale[:, None])
        low = torch.floor(steps)
        even = torch.remainder(low, 2) == 0
        up = (steps - low > 0.5) | ((steps - low == 0.5) & ~even)
        parts.append({"y": (low + up) * scale[:, None], "scales": scale, "total": total})
    return {n: torch.cat([p[n] for p in parts]) if parts[0][n] is not None else None for n in (("y", "scales", "total") if s.get("residual") is not None else ("y", "scales"))}
