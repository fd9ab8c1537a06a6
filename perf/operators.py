"""The FP8 block-scaled linear path of a decoder layer: what its operators compute, and their cases.

Four operators, which a W8A8 (e4m3 x e4m3) decoder layer runs in this order around its
attention:

* ``norm``   residual addition + RMSNorm + e4m3 quantization of the activations,
* ``linear`` matrix product of e4m3 activations (a scale per token and 128 columns) with e4m3
             weights (a scale per 128 x 128 block), fp16 or bf16 output,
* ``silu``   SiLU-gated product of the gate_up output + e4m3 quantization,
* ``quant``  the quantization alone (the attention output, which no norm precedes).

``own`` chooses between the plain form (elementary torch operations in 32 bits) and this
repository's kernels.
"""

from __future__ import annotations

import math

import torch

own = False

E4M3 = torch.float8_e4m3fn
FP8_MAX = 448.0
MIN_SCALE = 1.0 / (448.0 * 512.0)
BLOCK = 128
EPS = 1e-6
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------ cases


def listed() -> list[dict]:
    """Layer sizes of Qwen2.5-7B (hidden 3584, MLP 18944, gate_up 37888), the model this
    repository is configured for, and ragged sizes around them."""
    return [
        # One sequence decoding: the attention output projection, 13 MB of weights.
        {"name": "linear o, one token", "op": "linear", "m": 1, "n": 3584, "k": 3584,
         "dtype": "fp16", "bias": False},
        # A batch of 16 sequences decoding: the widest layer, 136 MB of weights.
        {"name": "linear gate_up, 16 tokens", "op": "linear", "m": 16, "n": 37888, "k": 3584,
         "dtype": "bf16", "bias": False},
        # A large decode batch or a short prompt: long K, few output columns.
        {"name": "linear down, 256 tokens", "op": "linear", "m": 256, "n": 3584, "k": 18944,
         "dtype": "fp16", "bias": False},
        # A ragged prefill chunk with bias on a layer whose sizes no block or tile divides.
        {"name": "linear ragged", "op": "linear", "m": 333, "n": 4613, "k": 2960,
         "dtype": "bf16", "bias": True},
        # Prefill of 4096 tokens through the widest layer.
        {"name": "linear gate_up, 4096 tokens", "op": "linear", "m": 4096, "n": 37888, "k": 3584,
         "dtype": "bf16", "bias": False},
        # The norm before qkv or gate_up, one sequence decoding.
        {"name": "norm, one token", "op": "norm", "m": 1, "h": 3584, "dtype": "fp16",
         "group": 128},
        # A prefill chunk of odd length; one scale per token (the W4A16 linears' FP8 input), and
        # a hidden size that no group divides.
        {"name": "norm ragged, per token", "op": "norm", "m": 333, "h": 5000, "dtype": "bf16",
         "group": 0},
        # A full prefill batch.
        {"name": "norm, 8192 tokens", "op": "norm", "m": 8192, "h": 3584, "dtype": "bf16",
         "group": 128},
        # The MLP's activation for a decode batch, one scale per token.
        {"name": "silu, 16 tokens, per token", "op": "silu", "m": 16, "h": 18944,
         "dtype": "fp16", "group": 0},
        # The same in prefill, a scale per 128 columns for the block-scaled down projection.
        {"name": "silu, 4096 tokens", "op": "silu", "m": 4096, "h": 18944, "dtype": "bf16",
         "group": 128},
        # The attention output of a few sequences.
        {"name": "quant, 7 tokens", "op": "quant", "m": 7, "h": 3584, "dtype": "bf16",
         "group": 128},
        # The attention output of a prefill.
        {"name": "quant, 4096 tokens", "op": "quant", "m": 4096, "h": 3584, "dtype": "fp16",
         "group": 128},
    ]


def _log_between(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    op = rng.choice(["linear", "linear", "linear", "norm", "silu", "quant"])
    dtype = rng.choice(["fp16", "bf16"])
    if op == "linear":
        k = 16 * _log_between(rng, 1, 1184)
        n = _log_between(rng, 1, min(37888, 37888 * 3584 // k))
        m = _log_between(rng, 1, 4096)
        return {"op": op, "m": m, "n": n, "k": k, "dtype": dtype, "bias": rng.random() < 0.3}
    h = _log_between(rng, 8, 18944 if op == "silu" else 8192)
    if rng.random() < 0.6:  # hidden sizes are mostly multiples of 16
        h = max(16, h // 16 * 16)
    most = min(8192, 4096 * 18944 // h)
    group = 128 if op == "quant" else rng.choice([128, 128, 0])
    return {"op": op, "m": _log_between(rng, 1, most), "h": h, "dtype": dtype, "group": group}


def work(case: dict) -> dict:
    m = case["m"]
    if case["op"] == "linear":
        n, k = case["n"], case["k"]
        kb, nb = -(-k // BLOCK), -(-n // BLOCK)
        b = m * k + 4 * m * kb + n * k + 4 * nb * kb + 2 * m * n + (2 * n if case["bias"] else 0)
        return {"bytes": b, "flops": 2 * m * n * k}
    h = case["h"]
    scales = 4 * m * (-(-h // BLOCK) if case["group"] else 1)
    if case["op"] == "norm":  # x, residual and weight in; codes, scales and the sum out
        return {"bytes": 7 * m * h + 2 * h + scales, "flops": 7 * m * h}
    if case["op"] == "silu":  # both halves in; codes and scales out
        return {"bytes": 5 * m * h + scales, "flops": 7 * m * h}
    return {"bytes": 3 * m * h + scales, "flops": 3 * m * h}


# ------------------------------------------------------------------------------------ inputs


def _activations(m: int, h: int, gen: torch.Generator, spread: float) -> torch.Tensor:
    """fp32 [m, h]: normal values with a token's own level, and a few outlier channels, as the
    residual stream of a decoder has them."""
    x = torch.randn((m, h), generator=gen, device="cuda")
    level = torch.exp(0.5 * torch.randn((m, 1), generator=gen, device="cuda"))
    channel = torch.ones(h, device="cuda")
    at = torch.randint(0, h, (max(1, h // 512),), generator=gen, device="cuda")
    channel[at] = 20.0
    return x * level * channel * spread


def _quantized(v: torch.Tensor, rows: int) -> tuple[torch.Tensor, torch.Tensor]:
    """e4m3 codes of ``v`` [r, c] with a scale for each block of ``rows`` x 128."""
    r, c = v.shape
    rb, cb = -(-r // rows), -(-c // BLOCK)
    p = torch.zeros((rb * rows, cb * BLOCK), device=v.device)
    p[:r, :c] = v
    p = p.view(rb, rows, cb, BLOCK)
    s = p.abs().amax(dim=(1, 3)).div(FP8_MAX).clamp(min=MIN_SCALE)
    q = (p / s[:, None, :, None]).clamp(-FP8_MAX, FP8_MAX).to(E4M3)
    return q.view(rb * rows, cb * BLOCK)[:r, :c].contiguous(), s.contiguous()


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    state = {"case": dict(case)}
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        # As a program holds them: the quantized weights of a checkpoint, and activations that
        # an earlier operator has quantized.
        w = torch.randn((n, k), generator=gen, device="cuda") / math.sqrt(k)
        state["wq"], state["w_scale"] = _quantized(w, BLOCK)
        del w
        state["xq"], state["x_scale"] = _quantized(_activations(m, k, gen, 1.0), 1)
        state["bias"] = (torch.randn(n, generator=gen, device="cuda") * 0.5).to(dtype) \
            if case["bias"] else None
        state["out_dtype"] = dtype
    elif case["op"] == "norm":
        m, h = case["m"], case["h"]
        state["x"] = torch.randn((m, h), generator=gen, device="cuda").to(dtype)
        state["residual"] = _activations(m, h, gen, 2.0).to(dtype)
        state["weight"] = (1 + 0.1 * torch.randn(h, generator=gen, device="cuda")).to(dtype)
    elif case["op"] == "silu":
        state["gate_up"] = _activations(case["m"], 2 * case["h"], gen, 1.0).to(dtype)
    else:
        state["x"] = _activations(case["m"], case["h"], gen, 1.0).to(dtype)
    return state


# ------------------------------------------------------------------------------- plain form


def _plain_quant(y: torch.Tensor, group: int) -> tuple[torch.Tensor, torch.Tensor]:
    """e4m3 codes and scales of fp32 ``y`` [m, h], a scale for each ``group`` columns (0: all)."""
    m, h = y.shape
    width = group or h
    g = -(-h // width)
    p = torch.nn.functional.pad(y, (0, g * width - h)).view(m, g, width)
    s = (p.abs().amax(dim=2) / FP8_MAX).clamp(min=MIN_SCALE)
    q = (p / s[:, :, None]).clamp(-FP8_MAX, FP8_MAX).to(E4M3)
    return q.view(m, g * width)[:, :h].contiguous(), s


def _plain_linear(xq, x_scale, wq, w_scale, bias, out_dtype) -> torch.Tensor:
    n, k = wq.shape
    sx = x_scale.repeat_interleave(BLOCK, dim=1)[:, :k]
    sw = w_scale.repeat_interleave(BLOCK, dim=0)[:n].repeat_interleave(BLOCK, dim=1)[:, :k]
    y = (xq.float() * sx) @ (wq.float() * sw).t()
    if bias is not None:
        y = y + bias.float()
    return y.to(out_dtype)


def _plain(state: dict):
    case = state["case"]
    if case["op"] == "linear":
        return _plain_linear(state["xq"], state["x_scale"], state["wq"], state["w_scale"],
                             state["bias"], state["out_dtype"])
    if case["op"] == "norm":
        # The sum is rounded to the stream's type, as the next layer will read it, and the norm
        # is that of the rounded sum.
        total = (state["x"].float() + state["residual"].float()).to(state["x"].dtype)
        f = total.float()
        rstd = torch.rsqrt(f.square().mean(dim=1, keepdim=True) + EPS)
        q, s = _plain_quant(f * rstd * state["weight"].float(), case["group"])
        return {"q": q, "scale": s, "residual": total}
    if case["op"] == "silu":
        g, u = state["gate_up"].float().chunk(2, dim=1)
        q, s = _plain_quant(g / (1 + torch.exp(-g)) * u, case["group"])
        return {"q": q, "scale": s}
    q, s = _plain_quant(state["x"].float(), case["group"])
    return {"q": q, "scale": s}


def run(state: dict):
    if not own:
        return _plain(state)
    from tokenforge_b200 import ops

    case = state["case"]
    if case["op"] == "linear":
        return ops.w8a8_block_linear(state["xq"], state["x_scale"], state["wq"],
                                     state["w_scale"], state["bias"], state["out_dtype"])
    if case["op"] == "norm":
        q, s, total = ops.add_rmsnorm_fp8_quant(state["x"], state["residual"], state["weight"],
                                                EPS, case["group"])
        return {"q": q, "scale": s, "residual": total}
    if case["op"] == "silu":
        q, s = ops.silu_mul_fp8_quant(state["gate_up"], case["group"])
        return {"q": q, "scale": s}
    q, s = ops.e4m3_quant_groups(state["x"])
    return {"q": q, "scale": s}


# ------------------------------------------------------------------------- definition, 64 bits


def _exact_quant(y: torch.Tensor, group: int) -> dict:
    """The values before their rounding to e4m3, and the scales, of ``y`` [m, h] in 64 bits."""
    m, h = y.shape
    width = group or h
    q, scales = torch.empty_like(y), []
    for c in range(0, h, width):
        part = y[:, c:c + width]
        s = torch.maximum(part.abs().max(dim=1, keepdim=True).values / 448.0,
                          torch.full((m, 1), MIN_SCALE, dtype=torch.float64, device=y.device))
        q[:, c:c + width] = part / s
        scales.append(s)
    return {"q": q, "scale": torch.cat(scales, dim=1)}


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        y = torch.zeros((m, n), dtype=torch.float64, device="cuda")
        row_block = torch.arange(n, device="cuda") // BLOCK
        for b, k0 in enumerate(range(0, k, BLOCK)):
            part = state["xq"][:, k0:k0 + BLOCK].double() @ \
                state["wq"][:, k0:k0 + BLOCK].double().t()
            part *= state["x_scale"][:, b].double()[:, None]
            part *= state["w_scale"][:, b].double()[row_block][None, :]
            y += part
        return y if state["bias"] is None else y + state["bias"].double()
    if case["op"] == "norm":
        total = state["x"].double() + state["residual"].double()
        r = total.to(DTYPES[case["dtype"]]).double()  # the norm's input, by definition
        var = (r * r).sum(dim=1, keepdim=True) / case["h"]
        out = _exact_quant(r / torch.sqrt(var + EPS) * state["weight"].double(), case["group"])
        out["residual"] = total
        return out
    if case["op"] == "silu":
        h = case["h"]
        g, u = state["gate_up"][:, :h].double(), state["gate_up"][:, h:].double()
        return _exact_quant(g * torch.sigmoid(g) * u, case["group"])
    return _exact_quant(state["x"].double(), case["group"])
