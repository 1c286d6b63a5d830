"""The 8-bit floating-point operators on real work: a block-scaled fp8 x fp8 matrix product and the operators that make
its activations (root-mean-square norm with the residual's addition, gated activation, plain quantisation).

``run`` computes a case in elementary torch operations in 32 bits, or, where ``own`` is set, through the engine's entry
points; ``exact`` is the definition in 64 bits (the 8-bit outputs are given there as the unrounded quotients).
"""
from __future__ import annotations

import math

import torch

own = False

F8_MAX = 448.0        # largest finite e4m3fn value
AMAX_FLOOR = 1e-12    # a group whose largest magnitude is smaller is scaled as if it were this
BLOCK = 128
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one token through a square projection: launch latency and the stream of the weights
        {"name": "linear 1x4096x4096", "op": "linear", "m": 1, "n": 4096, "k": 4096, "dtype": "bf16", "act": "none"},
        # sixteen sequences decoding through a 70B-class up projection: nothing but the stream of the weights
        {"name": "linear 16x28672x8192", "op": "linear", "m": 16, "n": 28672, "k": 8192, "dtype": "f16", "act": "none"},
        # a prefill chunk through a down projection: few tiles, a long K
        {"name": "linear 96x4096x11008", "op": "linear", "m": 96, "n": 4096, "k": 11008, "dtype": "bf16", "act": "none"},
        # ragged in every direction (last blocks of 104 columns and 16 k), bias and activation in the epilogue
        {"name": "linear 777x5000x4112 bias+gelu", "op": "linear", "m": 777, "n": 5000, "k": 4112, "dtype": "f16", "act": "add_fastgelu"},
        # prefill of a 4096-token prompt through an up projection: the matrix cores
        {"name": "linear 4096x11008x4096", "op": "linear", "m": 4096, "n": 11008, "k": 4096, "dtype": "bf16", "act": "none"},
        # norm in front of a decode step: one row, latency
        {"name": "norm 1x4096", "op": "norm", "m": 1, "k": 4096, "dtype": "bf16", "residual": True, "group": 128},
        # odd width, one scale per token (what a per-token epilogue scale takes), no residual
        {"name": "norm 777x5000 per token", "op": "norm", "m": 777, "k": 5000, "dtype": "f16", "residual": False, "group": 0},
        # norm in front of a prefill's projections: bandwidth
        {"name": "norm 4096x8192", "op": "norm", "m": 4096, "k": 8192, "dtype": "bf16", "residual": True, "group": 128},
        # between the two products of a decoding batch's gated MLP
        {"name": "gated 64x11008", "op": "gated", "m": 64, "k": 11008, "dtype": "bf16", "act": "silu", "group": 128},
        # the same of a prefill
        {"name": "gated 4096x11008", "op": "gated", "m": 4096, "k": 11008, "dtype": "f16", "act": "fastgelu", "group": 128},
        # attention's output in front of the output projection, decoding batch
        {"name": "quantize 16x4096", "op": "quantize", "m": 16, "k": 4096, "dtype": "bf16", "group": 128},
        # the same of a long prefill, one scale per token
        {"name": "quantize 8192x8192 per token", "op": "quantize", "m": 8192, "k": 8192, "dtype": "bf16", "group": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear", "norm", "gated", "quantize"])
    dtype = rng.choice(["f16", "bf16"])
    if op == "linear":
        while True:
            m, n = _log(rng, 1, 8192), _log(rng, 64, 28672)
            # K of a checkpoint: a whole number of 16-byte pieces, seldom of 128; now and then any number at all
            k = _log(rng, 64, 16384)
            k = k if rng.random() < 0.1 else max(16, k // 16 * 16) if rng.random() < 0.5 else max(128, k // 128 * 128)
            if rng.random() < 0.6:
                n = max(64, n // 64 * 64)
            if m * n * k <= 4096 * 11008 * 4096 and n * k <= 28672 * 8192:
                return {"op": op, "m": m, "n": n, "k": k, "dtype": dtype, "act": rng.choice(["none", "none", "fastgelu", "add", "add_fastgelu"])}
    while True:
        m, k = _log(rng, 1, 16384), _log(rng, 64, 16384)
        if rng.random() < 0.6:
            k = max(64, k // 64 * 64)
        if m * k <= 4096 * 11008:
            break
    case = {"op": op, "m": m, "k": k, "dtype": dtype, "group": rng.choice([128, 128, 0])}
    if op == "norm":
        case["residual"] = rng.random() < 0.7
    if op == "gated":
        case["act"] = rng.choice(["silu", "fastgelu"])
    return case


def _quantized(v, rows, cols):
    """v (R, C) fp32 -> e4m3 values and one scale for each block of rows x cols."""
    r, c = v.shape
    nr, nc = -(-r // rows), -(-c // cols)
    p = torch.nn.functional.pad(v, (0, nc * cols - c, 0, nr * rows - r)).view(nr, rows, nc, cols)
    s = p.abs().amax(dim=(1, 3)).clamp(min=AMAX_FLOOR) / F8_MAX
    q = (p / s[:, None, :, None]).clamp(-F8_MAX, F8_MAX).view(nr * rows, nc * cols)[:r, :c]
    return q.to(torch.float8_e4m3fn), s


def _activations(g, m, k, scale=1.0):
    """Rows as a transformer's: normal, some channels much larger than the rest, one row in 64 all zero (padding)."""
    v = torch.randn(m, k, device="cuda", generator=g) * scale
    v *= 1 + 15 * (torch.rand(k, device="cuda", generator=g) < 0.01)
    if m >= 64:
        v[torch.arange(m, device="cuda") % 64 == 63] = 0
    return v


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    m, k, dt = case["m"], case["k"], TYPES[case["dtype"]]
    state = {"case": case}
    if case["op"] == "linear":
        n = case["n"]
        state["x"], state["x_scale"] = _quantized(_activations(g, m, k), 1, BLOCK)
        state["w"], state["w_scale"] = _quantized(torch.randn(n, k, device="cuda", generator=g) / math.sqrt(k), BLOCK, BLOCK)
        state["x"], state["w"] = state["x"].contiguous(), state["w"].contiguous()
        state["bias"] = (torch.randn(n, device="cuda", generator=g) * 0.1).to(dt) if case["act"].startswith("add") else None
        return state
    state["x"] = _activations(g, m, k).to(dt)
    if case["op"] == "norm":
        state["weight"] = (1 + 0.2 * torch.randn(k, device="cuda", generator=g)).to(dt)
        state["residual"] = _activations(g, m, k, 4.0).to(dt) if case["residual"] else None
    if case["op"] == "gated":
        # gate and up as the two halves of one fused projection's output
        both = torch.cat([state["x"], torch.randn(m, k, device="cuda", generator=g).to(dt)], dim=1)
        state["gate"], state["up"] = both[:, :k], both[:, k:]
        del state["x"]
    return state


def _fastgelu(v):
    return v / (1 + torch.exp(v * (-2 * 0.035677 * (v * v) - 2 * 0.797885)))  # the engine's FastGelu: these two constants define it


def _rows(y, group):
    """Plain form of the quantisation at the end of norm, gated and quantize."""
    m, k = y.shape
    group = group or k
    n = -(-k // group)
    p = torch.nn.functional.pad(y, (0, n * group - k)).view(m, n, group)
    s = p.abs().amax(dim=2).clamp(min=AMAX_FLOOR) / F8_MAX
    q = (p / s[:, :, None]).clamp(-F8_MAX, F8_MAX).view(m, n * group)[:, :k]
    return {"q": q.to(torch.float8_e4m3fn), "scale": s}


def run(state):
    case = state["case"]
    if own:
        return _own(case, state)
    dt = TYPES[case["dtype"]]
    if case["op"] == "linear":
        n, k = state["w"].shape
        a = state["x"].float() * state["x_scale"].repeat_interleave(BLOCK, 1)[:, :k]
        b = state["w"].float() * state["w_scale"].repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
        y = a @ b.t()
        if state["bias"] is not None:
            y = y + state["bias"].float()
        if case["act"].endswith("fastgelu"):
            y = _fastgelu(y)
        return y.to(dt)
    if case["op"] == "norm":
        h = state["x"].float()
        if state["residual"] is not None:
            h = h + state["residual"].float()
        y = h / torch.sqrt((h * h).mean(dim=1, keepdim=True) + 1e-6) * state["weight"].float()
        out = _rows(y, case["group"])
        if state["residual"] is not None:
            out["residual"] = h.to(dt)
        return out
    if case["op"] == "gated":
        gate = state["gate"].float()
        act = gate / (1 + torch.exp(-gate)) if case["act"] == "silu" else _fastgelu(gate)
        return _rows(act * state["up"].float(), case["group"])
    return _rows(state["x"].float(), case["group"])


def _own(case, state):
    from composable_kernel_amd import torch_ops

    if case["op"] == "linear":
        return torch_ops.fp8_linear(state["x"], state["x_scale"], state["w"], state["w_scale"], bias=state["bias"],
                                    epilogue=case["act"], out_dtype=TYPES[case["dtype"]])
    if case["op"] == "norm":
        q, scale, residual = torch_ops.rmsnorm_fp8(state["x"], state["weight"], residual=state["residual"], eps=1e-6, group_k=case["group"])
        out = {"q": q, "scale": scale}
        if residual is not None:
            out["residual"] = residual
        return out
    if case["op"] == "gated":
        q, scale = torch_ops.gated_fp8(state["gate"], state["up"], activation=case["act"], group_k=case["group"])
    else:
        q, scale = torch_ops.quantize_fp8(state["x"], group_k=case["group"])
    return {"q": q, "scale": scale}


def work(case):
    m, k = case["m"], case["k"]
    if case["op"] == "linear":
        n = case["n"]
        kb = -(-k // BLOCK)
        return {"bytes": m * k + n * k + 4 * kb * (m + -(-n // BLOCK)) + 2 * m * n + (2 * n if case["act"].startswith("add") else 0),
                "flops": 2 * m * n * k}
    scales = 4 * m * (-(-k // case["group"]) if case["group"] else 1)
    if case["op"] == "norm":
        return {"bytes": (3 + (4 if case["residual"] else 0)) * m * k + 2 * k + scales, "flops": 6 * m * k}
    if case["op"] == "gated":
        return {"bytes": 5 * m * k + scales, "flops": 10 * m * k}
    return {"bytes": 3 * m * k + scales, "flops": 3 * m * k}


def exact(case, seed):
    s = prepare(case, seed)
    d = lambda t: t.to(torch.float64)  # noqa: E731
    gelu = lambda v: v * torch.special.expit(2 * (0.797885 * v + 0.035677 * v ** 3))  # noqa: E731
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        y = torch.zeros(m, n, dtype=torch.float64, device="cuda")
        columns = torch.arange(n, device="cuda") // BLOCK
        for j in range(-(-k // BLOCK)):
            at = slice(j * BLOCK, min(k, (j + 1) * BLOCK))
            y += (d(s["x"][:, at]) @ d(s["w"][:, at]).t()) * d(s["x_scale"][:, j:j + 1]) * d(s["w_scale"][:, j])[columns][None, :]
        if s["bias"] is not None:
            y += d(s["bias"])
        return gelu(y) if case["act"].endswith("fastgelu") else y
    if case["op"] == "norm":
        h = d(s["x"]) if s["residual"] is None else d(s["x"]) + d(s["residual"])
        y = h * torch.rsqrt(h.square().sum(1, keepdim=True) / case["k"] + 1e-6) * d(s["weight"])
    elif case["op"] == "gated":
        gate = d(s["gate"])
        y = (gate * torch.special.expit(gate) if case["act"] == "silu" else gelu(gate)) * d(s["up"])
    else:
        y = d(s["x"])
    width = case["group"] or case["k"]
    q, scales = torch.empty_like(y), []
    for at in range(0, case["k"], width):
        part = y[:, at:at + width]
        scale = torch.clamp(torch.amax(torch.abs(part), 1, keepdim=True), min=AMAX_FLOOR) / F8_MAX
        q[:, at:at + width] = part / scale
        scales.append(scale)
    out = {"q": q, "scale": torch.cat(scales, 1)}
    if case["op"] == "norm" and s["residual"] is not None:
        out["residual"] = h
    return out
