"""The operators of a dense layer in 8-bit floating point as measurable cases.

A case is one call that a host of this library makes around its MoE blocks: the
residual addition with the RMSNorm behind it, a tensor put into 8-bit floats
(e4m3, largest value 448) with FP32 scales, the gated activation between two
projections, or one projection with 8-bit activations and weights. Sizes are
those of the layers that the benchmark and the tests use (hidden 2048, expert
widths 1408, 1024 and 768, shared width 5632 with gate and up in one matrix of
11264 rows) and others between and around them.

Groups of 128 neighbouring columns of one row share a scale; weights share it
over 128 rows as well: d = max|v| / 448, at least 2^-126, 1 for a group of
zeros; code = e4m3(v / d).
"""

from __future__ import annotations

import functools
import math
import sys
from pathlib import Path

import torch

own = False

DEVICE = "cuda:0"
GROUP = 128
FP8_MAX = 448.0
TINY = 2.0 ** -126
EPS = 1e-6
STD = 0.02


def listed():
    return [
        # One token through a decoder layer: the attention's output joins the
        # residual and the shared expert reads the norm in 8 bits. Latency counts.
        {"name": "norm_t1", "op": "norm", "rows": 1, "cols": 2048, "residual": True, "bf16": False, "fp8": True},
        # A short prompt through a model of odd width: the last group of a row
        # has 120 columns.
        {"name": "norm_t137_ragged", "op": "norm", "rows": 137, "cols": 1400, "residual": False, "bf16": False,
         "fp8": True},
        # A prefill chunk where the router reads the norm in BF16 and the
        # shared expert in 8 bits.
        {"name": "norm_t4095_both", "op": "norm", "rows": 4095, "cols": 2048, "residual": True, "bf16": True,
         "fp8": True},
        # Attention outputs of a short chat prompt, before their projection.
        {"name": "quantize_t77", "op": "quantize", "rows": 77, "cols": 2048, "block": 1},
        # A shared expert's gate and up matrices as a loader puts them into 8 bits.
        {"name": "quantize_weight", "op": "quantize", "rows": 11264, "cols": 2048, "block": 128},
        # A few sequences decoded together, between the shared expert's projections.
        {"name": "silu_t6", "op": "silu", "rows": 6, "cols": 5632, "bf16": False, "fp8": True},
        # The same of a prefill chunk.
        {"name": "silu_t4095", "op": "silu", "rows": 4095, "cols": 5632, "bf16": False, "fp8": True},
        # Decode of one sequence: the shared expert's gate and up.
        {"name": "linear_t1", "op": "linear", "rows": 1, "out": 11264, "cols": 2048, "bias": False},
        # The benchmark's batch-32 decode: the shared expert's down projection.
        {"name": "linear_t32", "op": "linear", "rows": 32, "out": 2048, "cols": 5632, "bias": False},
        # A short prompt through a projection of odd sizes with a bias (the
        # attention's query, key and value have one).
        {"name": "linear_t137_ragged", "op": "linear", "rows": 137, "out": 1400, "cols": 2000, "bias": True},
        # The benchmark's 512-token prefill: the down projection.
        {"name": "linear_t512", "op": "linear", "rows": 512, "out": 2048, "cols": 5632, "bias": False},
        # Long prompts of a batch together: gate and up.
        {"name": "linear_t8191", "op": "linear", "rows": 8191, "out": 11264, "cols": 2048, "bias": False},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, evenly over their logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["norm", "quantize", "silu", "linear", "linear"])
    if op == "linear":
        most = 8191 * 11264 * 2048
        while True:
            case = {"op": op, "rows": _spread(rng, 1, 8191), "out": _spread(rng, 128, 11264),
                    "cols": 16 * _spread(rng, 8, 512), "bias": rng.random() < 0.5}
            if case["rows"] * case["out"] * case["cols"] <= most:
                return case
    rows, cols = _spread(rng, 1, 4095), _spread(rng, 128, 5632)
    if rng.random() < 0.75:
        cols = -(-cols // 8) * 8
    if op == "quantize":
        return {"op": op, "rows": rows, "cols": cols, "block": rng.choice([1, 128])}
    bf16, fp8 = rng.choice([(False, True), (True, False), (True, True)])
    case = {"op": op, "rows": rows, "cols": cols, "bf16": bf16, "fp8": fp8}
    if op == "norm":
        case["residual"] = rng.random() < 0.7
    return case


def work(case):
    rows, cols = case["rows"], case["cols"]
    groups = -(-cols // GROUP)
    if case["op"] == "linear":
        out = case["out"]
        blocks = -(-out // GROUP) * groups
        nbytes = rows * cols + 4 * rows * groups + out * cols + 4 * blocks + 2 * out * case["bias"] + 2 * rows * out
        return {"bytes": nbytes, "flops": 2 * rows * out * cols}
    if case["op"] == "quantize":
        return {"bytes": 3 * rows * cols + 4 * -(-rows // case["block"]) * groups, "flops": 3 * rows * cols}
    written = 2 * rows * cols * case["bf16"] + (rows * cols + 4 * rows * groups) * case["fp8"]
    if case["op"] == "silu":
        return {"bytes": 4 * rows * cols + written, "flops": 8 * rows * cols}
    more = 4 * rows * cols if case["residual"] else 0
    return {"bytes": 2 * rows * cols + 2 * cols + more + written, "flops": 8 * rows * cols}


# ------------------------------------------------------------- plain form --
def _groups(v, block):
    """v [rows, cols] as [row blocks, block, column groups, 128], zeros behind its edges."""
    rows, cols = v.shape
    v = torch.nn.functional.pad(v, (0, -cols % GROUP, 0, -rows % block))
    return v.view(v.shape[0] // block, block, v.shape[1] // GROUP, GROUP)


def _steps(v, block):
    """The scale of every group of v [rows, cols] (float)."""
    most = _groups(v.abs(), block).amax((1, 3))
    return torch.where(most == 0, torch.ones_like(most), (most / FP8_MAX).clamp_min(TINY))


def _spread_steps(steps, block, rows, cols):
    """The scale of every element."""
    return steps.repeat_interleave(block, 0)[:rows].repeat_interleave(GROUP, 1)[:, :cols]


def _quantized(v, block):
    steps = _steps(v, block)
    return (v / _spread_steps(steps, block, *v.shape)).to(torch.float8_e4m3fn), steps


# ----------------------------------------------------------------- inputs --
def prepare(case, seed):
    """What a host holds before the call: BF16 activations (of a norm's input or
    a projection's output, with the few large channels that they have in
    earnest), norm weights near 1, and for a projection the 8-bit codes and
    scales of activations and weight."""
    g = torch.Generator(device=DEVICE).manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device=DEVICE) * std

    def activations(rows, cols):
        channel = torch.exp(0.5 * normal(cols))
        return normal(rows, cols) * torch.where(torch.rand(cols, generator=g, device=DEVICE) < 0.01, 20 * channel,
                                                channel)

    rows, cols = case["rows"], case["cols"]
    state = dict(case)
    if case["op"] == "linear":
        state["x"], state["x_scales"] = _quantized(activations(rows, cols).to(torch.bfloat16).float(), 1)
        state["w"], state["w_scales"] = _quantized(normal(case["out"], cols, std=STD).to(torch.bfloat16).float(), GROUP)
        state["b"] = normal(case["out"]).to(torch.bfloat16) if case["bias"] else None
    elif case["op"] == "quantize":
        v = activations(rows, cols) if case["block"] == 1 else normal(rows, cols, std=STD)
        state["x"] = v.to(torch.bfloat16)
    elif case["op"] == "silu":
        state["x"] = (3 * normal(rows, 2 * cols)).to(torch.bfloat16)
    else:
        state["x"] = activations(rows, cols).to(torch.bfloat16)
        state["r"] = (4 * activations(rows, cols)).to(torch.bfloat16) if case["residual"] else None
        state["w"] = (1 + 0.1 * normal(cols)).to(torch.bfloat16)
    return state


# ------------------------------------------------------------------- runs --
@functools.lru_cache(maxsize=None)
def _extension():
    """The library's operators, as a host loads them once."""
    package = str(Path.cwd() / "uma-qmoe_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from uma_qmoe_amd.native_backend import load_native_extension

    return load_native_extension()[1]


@functools.lru_cache(maxsize=None)
def _matrix():
    from uma_qmoe_amd.native_backend import Fp8Matrix

    return Fp8Matrix


def _run_own(s):
    ext = _extension()
    if s["op"] == "linear":
        fp8 = _matrix()
        return ext.fp8_linear(fp8(s["x"], s["x_scales"], 1), fp8(s["w"], s["w_scales"], GROUP), s["b"])
    if s["op"] == "quantize":
        q = ext.fp8_quantize(s["x"], block_rows=s["block"])
        return q.codes, q.scales
    if s["op"] == "silu":
        y, q = ext.silu_mul(s["x"], bf16=s["bf16"], fp8=s["fp8"])
        return _norm_outputs(None, y, q and (q.codes, q.scales))
    total, y, q = ext.add_rmsnorm(s["x"], s["r"], EPS, s["w"], bf16=s["bf16"], fp8=s["fp8"])
    return _norm_outputs(total if s["residual"] else None, y, q and (q.codes, q.scales))


def _norm_outputs(total, y, q):
    out = {} if total is None else {"sum": total}
    if y is not None:
        out["bf16"] = y
    if q is not None:
        out["codes"], out["scales"] = q
    return out


def run(s):
    if own:
        return _run_own(s)
    if s["op"] == "linear":
        rows, cols = s["x"].shape
        x = s["x"].float() * _spread_steps(s["x_scales"], 1, rows, cols)
        w = s["w"].float() * _spread_steps(s["w_scales"], GROUP, s["out"], cols)
        y = x @ w.t()
        return (y if s["b"] is None else y + s["b"].float()).to(torch.bfloat16)
    if s["op"] == "quantize":
        return _quantized(s["x"].float(), s["block"])
    total = None
    if s["op"] == "silu":
        gate, up = s["x"].float().chunk(2, 1)
        y = gate / (1 + torch.exp(-gate)) * up
    else:
        v = s["x"]
        if s["residual"]:
            v = total = (s["x"].float() + s["r"].float()).to(torch.bfloat16)
        v = v.float()
        y = v * torch.rsqrt((v * v).mean(1, keepdim=True) + EPS) * s["w"].float()
    return _norm_outputs(total, y.to(torch.bfloat16) if s["bf16"] else None, _quantized(y, 1) if s["fp8"] else None)


# ------------------------------------------------------- 64-bit definition --
def _exact_quantized(v, block):
    """v / d before its rounding to 8 bits, and d, for every group in 64 bits."""
    rows, cols = v.shape
    at_row = torch.arange(rows, device=v.device) // block
    at_col = torch.arange(cols, device=v.device) // GROUP
    most = torch.zeros(rows, -(-cols // GROUP), dtype=v.dtype, device=v.device)
    most.scatter_reduce_(1, at_col.expand(rows, cols), v.abs(), "amax")
    d = torch.zeros(-(-rows // block), most.shape[1], dtype=v.dtype, device=v.device)
    d.scatter_reduce_(0, at_row[:, None].expand_as(most), most, "amax")
    d = d / FP8_MAX
    d[d == 0] = 1.0
    d = d.clamp(min=TINY)
    return v / d[at_row][:, at_col], d


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        rows, out, cols = case["rows"], case["out"], case["cols"]
        y = torch.zeros(rows, out, dtype=torch.float64, device=DEVICE)
        for k in range(0, cols, GROUP):
            part = s["x"][:, k:k + GROUP].double() @ s["w"][:, k:k + GROUP].double().t()
            part *= s["x_scales"][:, k // GROUP, None].double()
            part *= s["w_scales"][torch.arange(out, device=DEVICE) // GROUP, k // GROUP].double()
            y += part
        return y if s["b"] is None else y + s["b"].double()
    x = s["x"].double()
    if case["op"] == "quantize":
        return _exact_quantized(x, case["block"])
    total = None
    if case["op"] == "silu":
        n = case["cols"]
        y = x[:, :n] * torch.sigmoid(x[:, :n]) * x[:, n:]
    else:
        if case["residual"]:
            total = x + s["r"].double()
            x = total.to(torch.bfloat16).double()  # the norm is that of the sum as it is kept
        y = x / torch.sqrt(x.pow(2).sum(1, keepdim=True) / case["cols"] + EPS) * s["w"].double()
    return _norm_outputs(total, y if case["bf16"] else None, _exact_quantized(y, 1) if case["fp8"] else None)
