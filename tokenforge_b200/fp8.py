"""The FP8 block-scaled (W8A8) linear path: e4m3 activations with a scale per token and 128
columns, e4m3 weights with a scale per 128 x 128 block (``pack.W8A8BlockWeights``).

Four operators, in the order a decoder layer runs them around its attention:

* :func:`add_rmsnorm_fp8_quant` residual addition + RMSNorm + e4m3 quantization,
* :func:`w8a8_block_linear`     the matrix product,
* :func:`silu_mul_fp8_quant`    SiLU-gated product of a gate_up output + e4m3 quantization,
* :func:`e4m3_quant_groups`     the quantization alone (an attention output).

Each function first offers its arguments to the host fast path (``csrc/host/fp8_host.cpp``: one
C++ call that checks, allocates and launches); what that does not take as the plain case (strided
or misaligned tensors, another current device, anything wrong) is handled, or refused, below. So
is every call where the extension cannot be loaded, after one warning.

The functions here are the direct launchers; :mod:`tokenforge_b200.ops` exports them and registers
the same names as ``torch.ops.tokenforge.*`` with fakes for tracing. Calls enqueue on the current
CUDA stream of the inputs' device; outputs come from PyTorch's caching allocator.
CPU tensors raise. The reference has no counterpart: it quantizes activations to e4m3
(tokenforge/kernels/ops.py:130-156) but has no linear that consumes them.
"""

from __future__ import annotations

import warnings

import torch

from tokenforge_b200 import _lib

GROUP = 128

_fast = None  # the host fast path's module, loaded by the first call


class _NoFastPath:
    """Stands for the host fast path where it cannot be loaded: takes no call."""

    def _none(self, *args):  # type: ignore[no-untyped-def]
        return None

    add_rmsnorm = silu_mul = quant_groups = block_linear = _none


def _load_fast():  # type: ignore[no-untyped-def]
    global _fast
    _lib.lib()  # without the kernel library nothing runs: that error is not caught
    try:
        _fast = _lib.fp8_host()
    except ImportError as e:
        _fast = _NoFastPath()
        warnings.warn(f"the FP8 operators' host fast path cannot be loaded ({e}); their calls go "
                      "through Python, 10 to 14 us each instead of 4 to 6", RuntimeWarning,
                      stacklevel=3)
    return _fast


_DTYPES = {torch.float16: _lib.TF_DTYPE_FP16, torch.bfloat16: _lib.TF_DTYPE_BF16}
_CODES = (torch.float8_e4m3fn, torch.uint8)


def _stream_dtype(t: torch.Tensor, name: str) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{name} must be fp16 or bf16, got {t.dtype}")
    return code


def _gpu_index(t: torch.Tensor, name: str) -> int:
    index = t.get_device()
    if index < 0:
        raise RuntimeError(f"{name} must be a CUDA tensor (tokenforge_b200 has no CPU path)")
    return index


def _same_gpu(index: int, t: torch.Tensor, name: str) -> None:
    if t.get_device() != index:
        if _gpu_index(t, name) != index:
            raise ValueError(f"{name} is on {t.device}, expected cuda:{index}")


def _rows(t: torch.Tensor) -> tuple[torch.Tensor, int, int]:
    """``t`` as 2-D rows with unit stride along the last dimension (a view where it can be), how
    many rows, and their pitch. Rows that overlap (an expanded tensor) become a copy."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    n, c = t.shape
    pitch, step = t.stride()
    if n <= 1:
        pitch = c
    if (step != 1 and c > 1) or pitch < c:
        t, pitch = t.contiguous(), c
    return t, n, pitch


def _codes_like(x: torch.Tensor) -> torch.Tensor:
    if x.is_contiguous():
        return torch.empty_like(x, dtype=torch.float8_e4m3fn)
    return x.new_empty(x.shape, dtype=torch.float8_e4m3fn)


def _groups_of(columns: int, group_size: int) -> int:
    if group_size not in (0, GROUP):
        raise ValueError(f"group_size must be {GROUP} or 0 (one scale per row), got {group_size}")
    return -(-columns // GROUP) if group_size else 1


def add_rmsnorm_fp8_quant(
    x: torch.Tensor,
    residual: torch.Tensor | None,
    weight: torch.Tensor,
    eps: float,
    group_size: int = GROUP,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``h = x + residual`` (rounded to the inputs' type), RMSNorm of ``h`` in fp32, e4m3 codes.

    x, residual ``[..., H]`` and weight ``[H]`` in fp16 or bf16 (one type). Returns
    ``(q [..., H] e4m3, scale [..., ceil(H / 128)] fp32, h [..., H])``; ``scale [..., 1]`` with
    ``group_size=0``. ``residual=None``: h is x itself. Between h and the codes nothing is
    rounded to 16 bits, unlike :func:`ops.rmsnorm_fp8_quant`, which rounds as the reference does.
    """
    out = (_fast or _load_fast()).add_rmsnorm(x, residual, weight, eps, group_size)
    if out is not None:
        return out
    h = x.shape[-1] if x.dim() else 0
    dtype = _stream_dtype(x, "x")
    if h == 0:
        raise ValueError(f"x must be [..., H] with H >= 1, got {tuple(x.shape)}")
    if weight.dim() != 1 or weight.shape[0] != h:
        raise ValueError(f"weight shape {tuple(weight.shape)} != {(h,)}")
    if weight.dtype != x.dtype:
        raise TypeError(f"weight must be {x.dtype} like x, got {weight.dtype}")
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError(f"residual shape {tuple(residual.shape)} != {tuple(x.shape)}")
        if residual.dtype != x.dtype:
            raise TypeError(f"residual must be {x.dtype} like x, got {residual.dtype}")
    groups = _groups_of(h, group_size)
    index = _gpu_index(x, "x")
    _same_gpu(index, weight, "weight")
    q = _codes_like(x)
    scale = x.new_empty((*x.shape[:-1], groups), dtype=torch.float32)
    x2, t, ldx = _rows(x)
    if weight.stride(0) != 1:
        weight = weight.contiguous()
    if residual is None:
        total, rp, ldr, out = x, None, 0, None
    else:
        _same_gpu(index, residual, "residual")
        total = torch.empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)
        r2, _, ldr = _rows(residual)
        rp, out = r2.data_ptr(), total.data_ptr()
    if t == 0:
        return q, scale, total
    status = _lib.call_on(
        index, _lib.lib().tf_add_rmsnorm_fp8_quant,
        x2.data_ptr(), t, h, ldx, rp, ldr, weight.data_ptr(), eps, dtype, group_size,
        q.data_ptr(), scale.data_ptr(), out, h,
    )  # fmt: skip
    if status:
        _lib.check("tf_add_rmsnorm_fp8_quant", status)
    return q, scale, total


def silu_mul_fp8_quant(
    gate_up: torch.Tensor, group_size: int = GROUP
) -> tuple[torch.Tensor, torch.Tensor]:
    """``y = silu(gate) * up`` of ``gate_up [..., 2I]`` (fp16 or bf16) in fp32, and its e4m3 codes:
    ``(q [..., I], scale [..., ceil(I / 128)] fp32)``; ``scale [..., 1]`` with ``group_size=0``.
    """
    out = (_fast or _load_fast()).silu_mul(gate_up, group_size)
    if out is not None:
        return out
    dtype = _stream_dtype(gate_up, "gate_up")
    width = gate_up.shape[-1] if gate_up.dim() else 0
    if width == 0 or width % 2:
        raise ValueError("gate_up's last dimension must be even (gate and up halves) and not 0, "
                         f"got {tuple(gate_up.shape)}")
    i = width // 2
    groups = _groups_of(i, group_size)
    index = _gpu_index(gate_up, "gate_up")
    lead = gate_up.shape[:-1]
    q = gate_up.new_empty((*lead, i), dtype=torch.float8_e4m3fn)
    scale = gate_up.new_empty((*lead, groups), dtype=torch.float32)
    g2, m, ld = _rows(gate_up)
    if m == 0:
        return q, scale
    status = _lib.call_on(
        index, _lib.lib().tf_silu_mul_fp8_quant,
        g2.data_ptr(), m, i, ld, dtype, group_size, q.data_ptr(), scale.data_ptr(),
    )  # fmt: skip
    if status:
        _lib.check("tf_silu_mul_fp8_quant", status)
    return q, scale


def e4m3_quant_groups(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """e4m3 codes of ``x [..., C]`` (fp16 or bf16) with a scale per 128 columns, exactly
    ``e4m3(x / scale)`` with the fp32 division's rounding: ``(q, scale [..., ceil(C / 128)])``.
    One scale per row: :func:`ops.e4m3_quant_rows`."""
    out = (_fast or _load_fast()).quant_groups(x)
    if out is not None:
        return out
    dtype = _stream_dtype(x, "x")
    c = x.shape[-1] if x.dim() else 0
    if c == 0:
        raise ValueError(f"x must be [..., C] with C >= 1, got {tuple(x.shape)}")
    index = _gpu_index(x, "x")
    q = _codes_like(x)
    scale = x.new_empty((*x.shape[:-1], -(-c // GROUP)), dtype=torch.float32)
    x2, r, ldx = _rows(x)
    if r == 0:
        return q, scale
    status = _lib.call_on(
        index, _lib.lib().tf_e4m3_quant_groups,
        x2.data_ptr(), r, c, ldx, dtype, q.data_ptr(), scale.data_ptr(),
    )  # fmt: skip
    if status:
        _lib.check("tf_e4m3_quant_groups", status)
    return q, scale


def w8a8_block_linear(
    xq: torch.Tensor,
    x_scale: torch.Tensor,
    wq: torch.Tensor,
    w_scale: torch.Tensor,
    bias: torch.Tensor | None = None,
    out_dtype: torch.dtype = torch.float16,
) -> torch.Tensor:
    """``y = (xq * x_scale) @ (wq * w_scale)^T + bias`` with fp32 sums, rounded once.

    xq ``[..., K]`` e4m3 (or its uint8 codes), x_scale fp32 ``[..., ceil(K / 128)]``, wq
    ``[N, K]`` e4m3, w_scale fp32 ``[ceil(N / 128), ceil(K / 128)]``, bias ``[N]`` in the output
    type (fp16 or bf16). K must be a multiple of 16.
    """
    y = (_fast or _load_fast()).block_linear(xq, x_scale, wq, w_scale, bias, out_dtype)
    if y is not None:
        return y
    if xq.dtype not in _CODES:
        raise TypeError(f"xq must be float8_e4m3fn (or its uint8 codes), got {xq.dtype}")
    if wq.dtype not in _CODES:
        raise TypeError(f"wq must be float8_e4m3fn (or its uint8 codes), got {wq.dtype}")
    if x_scale.dtype != torch.float32 or w_scale.dtype != torch.float32:
        raise TypeError(f"x_scale and w_scale must be fp32, got {x_scale.dtype}, {w_scale.dtype}")
    dtype = _DTYPES.get(out_dtype)
    if dtype is None:
        raise TypeError(f"out_dtype must be fp16 or bf16, got {out_dtype}")
    if wq.dim() != 2 or wq.shape[0] == 0 or xq.dim() == 0:
        raise ValueError(f"wq must be [N, K] with N >= 1 and xq [..., K], got {tuple(wq.shape)} "
                         f"and {tuple(xq.shape)}")
    n, k = wq.shape
    if xq.shape[-1] != k:
        raise ValueError(f"xq has K={xq.shape[-1]} but wq has K={k}")
    if k == 0 or k % 16:
        raise ValueError(f"K={k} must be a positive multiple of 16")
    kb = -(-k // GROUP)
    lead = xq.shape[:-1]
    if x_scale.shape != (*lead, kb):
        raise ValueError(f"x_scale shape {tuple(x_scale.shape)} != {(*lead, kb)}")
    if w_scale.shape != (-(-n // GROUP), kb):
        raise ValueError(f"w_scale shape {tuple(w_scale.shape)} != {(-(-n // GROUP), kb)}")
    if not (wq.is_contiguous() and w_scale.is_contiguous()):
        raise ValueError("wq and w_scale must be contiguous")
    if bias is not None:
        if bias.dtype != out_dtype:
            raise TypeError(f"bias must be {out_dtype} like the output, got {bias.dtype}")
        if bias.shape != (n,):
            raise ValueError(f"bias shape {tuple(bias.shape)} != {(n,)}")
    index = _gpu_index(xq, "xq")
    _same_gpu(index, x_scale, "x_scale")
    _same_gpu(index, wq, "wq")
    _same_gpu(index, w_scale, "w_scale")
    bp = None
    if bias is not None:
        _same_gpu(index, bias, "bias")
        if bias.stride(0) != 1:
            bias = bias.contiguous()
        bp = bias.data_ptr()
    y = x_scale.new_empty((*lead, n), dtype=out_dtype)
    x2, m, ldx = _rows(xq)
    xp, wp = x2.data_ptr(), wq.data_ptr()
    if xp % 16 or ldx % 16:
        x2 = x2.clone(memory_format=torch.contiguous_format)
        xp, ldx = x2.data_ptr(), k
    if wp % 16:
        raise ValueError("wq must be 16-byte aligned")
    if m == 0:
        return y
    s2, _, lds = _rows(x_scale)
    lib = _lib.lib()
    status = _lib.call_on(
        index, lib.tf_w8a8_block_linear,
        xp, m, k, ldx, s2.data_ptr(), lds, wp, w_scale.data_ptr(), bp, n, dtype, y.data_ptr(), n,
    )  # fmt: skip
    if status:
        _lib.check("tf_w8a8_block_linear", status)
    return y
