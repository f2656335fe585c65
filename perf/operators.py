"""Cases of the 8-bit linear layer's operators: what is computed, on what, and how much of it.

Three operators, as a serving step strings them together:

quantize  rows of x, or of silu(gate) * up, to e4m3 with one power-of-two scale per 128 columns
norm      residual addition, root-mean-square norm, and the same 8-bit output
matmul    out[m, n] = sum over k of (lhs[m, k] * its scale) * (rhs[n, k] * its scale)

A group is 128 consecutive columns of a row (the last one of a row may be shorter). Its scale is the
least power of two s, at least 2^-127, with max |v| <= 448 s (1 where the group is all zeros); its
values are v / s rounded to nearest even in e4m3. Scales are held in one byte (e8m0).
"""

from __future__ import annotations

import math

import torch

own = False

GROUP = 128
_DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}
EPSILON = 1e-5


def listed():
    return [
        # The attention output of one decode step of 64 sequences, before its projection.
        {"name": "quantize 64x8192 bf16", "op": "quantize", "rows": 64, "cols": 8192, "dtype": "bf16", "gate": False, "pad": 0},
        # A projection's weights, laid out once when a model is loaded.
        {"name": "quantize 16384x8192 bf16", "op": "quantize", "rows": 16384, "cols": 8192, "dtype": "bf16", "gate": False, "pad": 0},
        # The gated activation of an MLP in a decode step of 16 sequences.
        {"name": "gate 16x16384 bf16", "op": "quantize", "rows": 16, "cols": 16384, "dtype": "bf16", "gate": True, "pad": 0},
        # The same over the ragged token count of a prefill step, with half-precision inputs.
        {"name": "gate 4001x11008 f16", "op": "quantize", "rows": 4001, "cols": 11008, "dtype": "f16", "gate": True, "pad": 0},
        # One token's hidden state between two layers.
        {"name": "norm 1x8192 bf16 residual", "op": "norm", "rows": 1, "cols": 8192, "dtype": "bf16", "residual": True, "pad": 0},
        # The first layer's norm (no residual yet) of a width that ends inside a group.
        {"name": "norm 777x5000 f32", "op": "norm", "rows": 777, "cols": 5000, "dtype": "f32", "residual": False, "pad": 0},
        # A prefill step's hidden states between two layers.
        {"name": "norm 8192x8192 bf16 residual", "op": "norm", "rows": 8192, "cols": 8192, "dtype": "bf16", "residual": True, "pad": 0},
        # A square projection of one decode token: latency, and the weights' bytes.
        {"name": "matmul 1x8192x8192", "op": "matmul", "m": 1, "k": 8192, "n": 8192, "out": "bf16"},
        # The smallest distributed-matmul shape of the run command, with f32 output.
        {"name": "matmul 128x1024x1024 f32", "op": "matmul", "m": 128, "k": 1024, "n": 1024, "out": "f32"},
        # An up-projection of a decode step of 64 sequences.
        {"name": "matmul 64x8192x16384", "op": "matmul", "m": 64, "k": 8192, "n": 16384, "out": "bf16"},
        # Odd extents everywhere: ragged tokens, a contraction that ends inside a group, odd output rows.
        {"name": "matmul 1001x5000x4099", "op": "matmul", "m": 1001, "k": 5000, "n": 4099, "out": "bf16"},
        # The benchmark's matmul shape: a prefill step.
        {"name": "matmul 8192x16384x8192", "op": "matmul", "m": 8192, "k": 16384, "n": 8192, "out": "bf16"},
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("quantize", "norm", "matmul"))
    if op == "matmul":
        while True:
            m, k, n = _log_uniform(rng, 1, 8192), _log_uniform(rng, 64, 16384), _log_uniform(rng, 64, 16384)
            if rng.random() < 0.5:  # whole groups, as most models have; the rest is odd
                k, n = -(-k // GROUP) * GROUP, -(-n // GROUP) * GROUP
            if m * k * n <= 8192 * 16384 * 8192:
                return {"op": op, "m": m, "k": k, "n": n, "out": rng.choice(("bf16", "bf16", "f32"))}
    rows, cols = _log_uniform(rng, 1, 16384), _log_uniform(rng, 64, 16384)
    if rng.random() < 0.5:
        cols = -(-cols // GROUP) * GROUP
    case = {"op": op, "rows": rows, "cols": cols, "dtype": rng.choice(("bf16", "bf16", "f16", "f32")),
            "pad": rng.choice((0, 0, 64, 129))}  # columns of the buffer behind each row: x is a slice of something wider
    case["gate" if op == "quantize" else "residual"] = rng.random() < 0.5
    return case


# ------------------------------------------------------------------------------------- inputs


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _hidden(g, rows, cols, dtype, pad):
    """Activations: normal, with a few channels an order of magnitude larger, as hidden states have them."""
    x = torch.randn(rows, cols + pad, generator=g, device="cuda")
    loud = torch.rand(cols + pad, generator=g, device="cuda") < 0.01
    return (x * torch.where(loud, 12.0, 1.0)).to(dtype)[:, :cols]


def _operand(g, rows, k, spread):
    """An 8-bit operand in hand: codes with the row pitch the hardware wants (a multiple of 16), and scales."""
    v = torch.randn(rows, k, generator=g, device="cuda") * spread
    codes, scales = _quantized(v)
    held = torch.zeros(rows, -(-k // 16) * 16, device="cuda", dtype=torch.float8_e4m3fn)[:, :k]
    held.copy_(codes)
    return held, scales


def prepare(case, seed):
    g = _generator(seed)
    state = {"case": case}
    if case["op"] == "matmul":
        state["lhs"], state["lhs_scales"] = _operand(g, case["m"], case["k"], 1.0)
        state["rhs"], state["rhs_scales"] = _operand(g, case["n"], case["k"], case["k"] ** -0.5)
    else:
        dtype, cols = _DTYPE[case["dtype"]], case["cols"]
        state["x"] = _hidden(g, case["rows"], cols * (2 if case.get("gate") else 1), dtype, case["pad"])
        if case["op"] == "norm":
            state["weight"] = (1 + 0.1 * torch.randn(cols, generator=g, device="cuda")).to(dtype)
            state["residual"] = _hidden(g, case["rows"], cols, dtype, case["pad"]) if case["residual"] else None
    if own:
        _build(state)
    return state


def _build(state):
    """The plan and its executable, which a program builds once."""
    import __graft_entry__

    __graft_entry__.load_package()
    from tpu_cake_b200 import scaled_cuda_lowering as scaled

    case = state["case"]
    if case["op"] == "matmul":
        plan = scaled.CudaScaledMatmulPlan(name="perf", n=case["n"], k=case["k"], output_dtype=case["out"])
    elif case["op"] == "norm":
        plan = scaled.CudaRmsNormQuantizePlan(name="perf", columns=case["cols"], input_dtype=case["dtype"], weight_dtype=case["dtype"],
                                              epsilon=EPSILON, with_residual=case["residual"])
    else:
        plan = scaled.CudaQuantizeRowsPlan(name="perf", columns=case["cols"], input_dtype=case["dtype"], gate="silu" if case["gate"] else "none")
    state["plan"], state["executable"] = plan, plan.build(torch.device("cuda", torch.cuda.current_device()))


# ------------------------------------------------------------------------------------- plain form


def _quantized(v):
    """e4m3 codes and e8m0 scales of f32 rows. The exponent comes from the largest magnitude's own bits:
    a = f 2^e with f in [0.5, 1), and a <= 448 2^s = 0.875 2^(s + 9)."""
    rows, cols = v.shape
    groups = -(-cols // GROUP)
    padded = torch.nn.functional.pad(v, (0, groups * GROUP - cols)).reshape(rows, groups, GROUP)
    largest = padded.abs().amax(dim=2)
    fraction, exponent = torch.frexp(largest)
    exponent = exponent - 9 + (fraction > 0.875).to(exponent.dtype)
    exponent = torch.where(largest == 0, torch.zeros_like(exponent), exponent.clamp(min=-127))
    codes = torch.ldexp(padded, -exponent[..., None]).to(torch.float8_e4m3fn)
    return codes.reshape(rows, groups * GROUP)[:, :cols], (exponent + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _dequantized(codes, scales):
    return codes.float() * scales.float().repeat_interleave(GROUP, dim=1)[:, : codes.shape[1]]


def run(state):
    case = state["case"]
    if own:
        plan, executable = state["plan"], state["executable"]
        if case["op"] == "matmul":
            return plan.invoke(executable, state["lhs"], state["lhs_scales"], state["rhs"], state["rhs_scales"])
        if case["op"] == "norm":
            codes, scales, summed = plan.invoke(executable, state["x"], state["weight"], state["residual"])
            return {"codes": codes, "scales": scales, "residual": summed}
        codes, scales = plan.invoke(executable, state["x"])
        return {"codes": codes, "scales": scales}
    if case["op"] == "matmul":
        out = _dequantized(state["lhs"], state["lhs_scales"]) @ _dequantized(state["rhs"], state["rhs_scales"]).t()
        return out.to(_DTYPE[case["out"]])
    if case["op"] == "norm":
        h = state["x"].float()
        if state["residual"] is not None:
            h = h + state["residual"].float()
        scale = 1.0 / torch.sqrt((h * h).mean(dim=1, keepdim=True) + EPSILON)
        codes, scales = _quantized(h * scale * state["weight"].float())
        return {"codes": codes, "scales": scales, "residual": h.to(state["x"].dtype) if state["residual"] is not None else None}
    v = state["x"].float()
    if case["gate"]:
        v = v[:, : case["cols"]] / (1.0 + torch.exp(-v[:, : case["cols"]])) * v[:, case["cols"] :]
    codes, scales = _quantized(v)
    return {"codes": codes, "scales": scales}


# ------------------------------------------------------------------------------------- bounds and definitions


def work(case):
    if case["op"] == "matmul":
        m, k, n = case["m"], case["k"], case["n"]
        groups = -(-k // GROUP)
        return {"bytes": (m + n) * (k + groups) + m * n * _BYTES[case["out"]], "flops": 2 * m * n * k}
    rows, cols, size = case["rows"], case["cols"], _BYTES[case["dtype"]]
    out = rows * (cols + -(-cols // GROUP))
    if case["op"] == "norm":
        return {"bytes": rows * cols * size * (3 if case["residual"] else 1) + cols * size + out, "flops": 6 * rows * cols}
    return {"bytes": rows * cols * size * (2 if case["gate"] else 1) + out, "flops": (7 if case["gate"] else 3) * rows * cols}


def _exact_codes(v):
    """Codes and scales of 64-bit rows from the definition: the least e with max |v| <= 448 * 2^e, then
    steps of 2^(floor(log2 |v|) - 3), and of 2^-9 below 2^-6."""
    rows, cols = v.shape
    codes = torch.empty_like(v)
    scales = torch.empty(rows, -(-cols // GROUP), dtype=torch.float64, device=v.device)
    for g in range(scales.shape[1]):
        part = v[:, g * GROUP : (g + 1) * GROUP]
        a = part.abs().max(dim=1).values
        e = torch.ceil(torch.log2(torch.where(a > 0, a, torch.ones_like(a)) / 448.0))
        e = torch.where(448.0 * torch.exp2(e - 1) >= a, e - 1, e)  # log2 may round across a power of two
        e = torch.where(448.0 * torch.exp2(e) < a, e + 1, e)
        s = torch.where(a > 0, torch.exp2(e.clamp(min=-127)), torch.ones_like(a))
        t = part / s[:, None]
        step = torch.exp2(torch.floor(torch.log2(t.abs().clamp(min=2.0**-6))) - 3)
        codes[:, g * GROUP : (g + 1) * GROUP] = torch.round(t / step) * step
        scales[:, g] = s
    return codes, scales


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "matmul":
        side = []
        for name in ("lhs", "rhs"):
            scales = torch.exp2(state[name + "_scales"].view(torch.uint8).double() - 127)
            value = state[name].double()
            for g in range(scales.shape[1]):
                value[:, g * GROUP : (g + 1) * GROUP] *= scales[:, g : g + 1]
            side.append(value)
        return torch.einsum("mk,nk->mn", side[0], side[1])
    x = state["x"].double()
    if case["op"] == "norm":
        h = x if state["residual"] is None else x + state["residual"].double()
        rms = torch.sqrt(h.pow(2).sum(dim=1, keepdim=True) / case["cols"] + EPSILON)
        codes, scales = _exact_codes(h / rms * state["weight"].double())
        return {"codes": codes, "scales": scales, "residual": None if state["residual"] is None else h}
    if case["gate"]:
        gate, up = x[:, : case["cols"]], x[:, case["cols"] :]
        x = gate * torch.sigmoid(gate) * up
    codes, scales = _exact_codes(x)
    return {"codes": codes, "scales": scales}
