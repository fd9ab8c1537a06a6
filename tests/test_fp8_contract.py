"""Host-side contract of the FP8 block-scaled (W8A8) path, checked without a GPU: argument errors,
fakes, the weight bundle, and the C ABI's refusals (each returns before anything is enqueued)."""

from __future__ import annotations

import warnings

import pytest
import torch

from tokenforge_b200 import _lib, ops
from tokenforge_b200.pack import (
    FP8_MIN_SCALE,
    W8A8BlockWeights,
    dequantize_w8a8_block,
    pack_w8a8_block,
)

E4M3 = torch.float8_e4m3fn


def _linear_args(m=3, n=200, k=272):  # type: ignore[no-untyped-def]
    kb = -(-k // 128)
    return {
        "xq": torch.zeros((m, k), dtype=E4M3),
        "x_scale": torch.ones((m, kb)),
        "wq": torch.zeros((n, k), dtype=E4M3),
        "w_scale": torch.ones((-(-n // 128), kb)),
        "bias": torch.zeros(n, dtype=torch.float16),
        "out_dtype": torch.float16,
    }


@pytest.mark.parametrize(
    "change, error, match",
    [
        ({"xq": torch.zeros((3, 272), dtype=torch.float16)}, TypeError, "xq must be float8"),
        ({"wq": torch.zeros((200, 272), dtype=torch.int8)}, TypeError, "wq must be float8"),
        ({"x_scale": torch.ones((3, 3), dtype=torch.float16)}, TypeError, "must be fp32"),
        ({"out_dtype": torch.float32}, TypeError, "out_dtype"),
        ({"wq": torch.zeros((200, 256), dtype=E4M3)}, ValueError, "wq has K=256"),
        ({"x_scale": torch.ones((3, 2))}, ValueError, "x_scale shape"),
        ({"x_scale": torch.ones((2, 3))}, ValueError, "x_scale shape"),
        ({"w_scale": torch.ones((1, 3))}, ValueError, "w_scale shape"),
        ({"wq": torch.zeros((272, 200), dtype=E4M3).t()}, ValueError, "contiguous"),
        ({"bias": torch.zeros(199, dtype=torch.float16)}, ValueError, "bias shape"),
        ({"bias": torch.zeros(200, dtype=torch.bfloat16)}, TypeError, "bias must be"),
        ({}, RuntimeError, "CUDA"),
    ],
)
def test_linear_refusals(change, error, match) -> None:  # type: ignore[no-untyped-def]
    args = _linear_args() | change
    with pytest.raises(error, match=match):
        ops.w8a8_block_linear(**args)


@pytest.mark.parametrize("k", [8, 24, 1000])
def test_linear_refuses_k_off_sixteen(k: int) -> None:
    with pytest.raises(ValueError, match="multiple of 16"):
        ops.w8a8_block_linear(**_linear_args(k=k))


def test_linear_refuses_no_rows_of_weights() -> None:
    with pytest.raises(ValueError, match="N >= 1"):
        ops.w8a8_block_linear(**_linear_args(n=0))


def test_norm_refusals() -> None:
    x = torch.zeros((2, 64), dtype=torch.float16)
    w = torch.ones(64, dtype=torch.float16)
    f = ops.add_rmsnorm_fp8_quant
    with pytest.raises(TypeError, match="fp16 or bf16"):
        f(x.float(), x.float(), w.float(), 1e-6)
    with pytest.raises(ValueError, match="weight shape"):
        f(x, x, w[:32], 1e-6)
    with pytest.raises(TypeError, match="weight must be"):
        f(x, x, w.bfloat16(), 1e-6)
    with pytest.raises(ValueError, match="residual shape"):
        f(x, x[:1], w, 1e-6)
    with pytest.raises(TypeError, match="residual must be"):
        f(x, x.bfloat16(), w, 1e-6)
    with pytest.raises(ValueError, match="group_size"):
        f(x, x, w, 1e-6, 64)
    with pytest.raises(ValueError, match="H >= 1"):
        f(x[:, :0], x[:, :0], w[:0], 1e-6)
    with pytest.raises(RuntimeError, match="CUDA"):
        f(x, x, w, 1e-6)


def test_silu_and_quant_refusals() -> None:
    x = torch.zeros((2, 64), dtype=torch.bfloat16)
    with pytest.raises(TypeError, match="fp16 or bf16"):
        ops.silu_mul_fp8_quant(x.float())
    with pytest.raises(ValueError, match="even"):
        ops.silu_mul_fp8_quant(x[:, :63])
    with pytest.raises(ValueError, match="group_size"):
        ops.silu_mul_fp8_quant(x, 32)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.silu_mul_fp8_quant(x)
    with pytest.raises(TypeError, match="fp16 or bf16"):
        ops.e4m3_quant_groups(x.double())
    with pytest.raises(ValueError, match="C >= 1"):
        ops.e4m3_quant_groups(x[:, :0])
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.e4m3_quant_groups(x)


def test_fakes_give_the_shapes() -> None:
    from torch._subclasses.fake_tensor import FakeTensorMode

    t = torch.ops.tokenforge
    with FakeTensorMode():
        x = torch.empty((2, 3, 300), dtype=torch.bfloat16)
        q, s, h = t.add_rmsnorm_fp8_quant(x, x, x[0, 0], 1e-6, 128)
        assert (q.shape, q.dtype) == (x.shape, E4M3)
        assert (s.shape, s.dtype) == ((2, 3, 3), torch.float32)
        assert (h.shape, h.dtype) == (x.shape, x.dtype)
        q, s = t.silu_mul_fp8_quant(x, 0)
        assert q.shape == (2, 3, 150) and s.shape == (2, 3, 1)
        q, s = t.e4m3_quant_groups(x)
        assert q.shape == (2, 3, 300) and s.shape == (2, 3, 3)
        a = {k: torch.empty(v.shape, dtype=v.dtype) if isinstance(v, torch.Tensor) else v
             for k, v in _linear_args().items()}
        y = t.w8a8_block_linear(a["xq"], a["x_scale"], a["wq"], a["w_scale"], a["bias"],
                                torch.bfloat16)
        assert y.shape == (3, 200) and y.dtype == torch.bfloat16


@pytest.mark.parametrize("n, k", [(128, 128), (1, 16), (200, 272), (129, 4096)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_pack_w8a8_block(n: int, k: int, dtype: torch.dtype) -> None:
    gen = torch.Generator().manual_seed(n * k)
    w = torch.randn((n, k), generator=gen).to(dtype)
    p = pack_w8a8_block(w)
    assert isinstance(p, W8A8BlockWeights) and (p.n, p.k) == (n, k)
    assert p.wq.dtype == E4M3 and p.w_scale.shape == (-(-n // 128), -(-k // 128))
    d = dequantize_w8a8_block(p).double()
    # e4m3 rounds to within half a step: 2^-4 of the value, or half the subnormal step 2^-9 of
    # its block's scale; 2^-20 covers the fp32 division by the scale and the product with it.
    s = p.w_scale.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    err = (d - w.double()).abs()
    assert bool((err <= w.double().abs() * (2**-4 + 2**-20) + s * 2**-10).all())
    assert float(p.w_scale.min()) >= FP8_MIN_SCALE


def test_pack_refusals_and_zero_blocks() -> None:
    with pytest.raises(ValueError, match="N, K"):
        pack_w8a8_block(torch.zeros((0, 128)))
    with pytest.raises(TypeError, match="fp16, bf16 or fp32"):
        pack_w8a8_block(torch.zeros((8, 128), dtype=torch.float64))
    p = pack_w8a8_block(torch.zeros((8, 128)))
    assert float(p.w_scale) == pytest.approx(FP8_MIN_SCALE) and not p.wq.float().any()


# ------------------------------------------------------------------------------- C ABI refusals
# 16 and 24 stand for addresses (16-byte aligned, and not): every call below is refused before
# any of them is read or anything is enqueued.


def _abi_linear(m=1, k=128, ldx=128, ldxs=1, n=128, dtype=0, ldy=128, xq=16, wq=16, y=16):  # type: ignore[no-untyped-def]
    return _lib.lib().tf_w8a8_block_linear(xq, m, k, ldx, 16, ldxs, wq, 16, None, n, dtype, y, ldy,
                                           None)


@pytest.mark.parametrize(
    "change, status",
    [
        ({"m": -1}, _lib.TF_ERR_INVALID_ARG),
        ({"n": 0}, _lib.TF_ERR_INVALID_ARG),
        ({"k": 0}, _lib.TF_ERR_INVALID_ARG),
        ({"dtype": 2}, _lib.TF_ERR_INVALID_ARG),
        ({"k": 120}, _lib.TF_ERR_UNSUPPORTED),
        ({"ldx": 112}, _lib.TF_ERR_INVALID_ARG),
        ({"ldy": 127}, _lib.TF_ERR_INVALID_ARG),
        ({"ldxs": 0}, _lib.TF_ERR_INVALID_ARG),
        ({"xq": None}, _lib.TF_ERR_INVALID_ARG),
        ({"y": None}, _lib.TF_ERR_INVALID_ARG),
        ({"xq": 24}, _lib.TF_ERR_ALIGNMENT),
        ({"wq": 24}, _lib.TF_ERR_ALIGNMENT),
        ({"ldx": 136}, _lib.TF_ERR_ALIGNMENT),
        ({"m": 0}, _lib.TF_OK),
        ({"m": (1 << 30) + 1}, _lib.TF_ERR_TOO_LARGE),
        ({"n": (1 << 30) + 1, "ldy": (1 << 30) + 1}, _lib.TF_ERR_TOO_LARGE),
    ],
)
def test_abi_linear_status(change, status) -> None:  # type: ignore[no-untyped-def]
    assert _abi_linear(**change) == status


def test_abi_activation_status() -> None:
    lib = _lib.lib()
    bad = _lib.TF_ERR_INVALID_ARG

    def norm(x=16, t=1, h=8, ldx=8, res=16, ldr=8, w=16, dtype=0, group=128, q=16, s=16, out=16,  # type: ignore[no-untyped-def]
             ldo=8):
        return lib.tf_add_rmsnorm_fp8_quant(x, t, h, ldx, res, ldr, w, 1e-6, dtype, group, q, s,
                                            out, ldo, None)

    assert norm(t=-1) == norm(h=0) == norm(dtype=7) == norm(group=64) == bad
    assert norm(x=None) == norm(w=None) == norm(q=None) == norm(s=None) == bad
    assert norm(ldx=7) == norm(ldr=7) == norm(ldo=7) == bad
    assert norm(out=None) == norm(res=None) == bad  # both or neither
    assert norm(t=0) == _lib.TF_OK

    def silu(x=16, m=1, i=8, ld=16, dtype=0, group=0, q=16, s=16):  # type: ignore[no-untyped-def]
        return lib.tf_silu_mul_fp8_quant(x, m, i, ld, dtype, group, q, s, None)

    assert silu(m=-1) == silu(i=0) == silu(ld=15) == silu(dtype=-1) == silu(group=1) == bad
    assert silu(x=None) == silu(q=None) == silu(s=None) == bad
    assert silu(m=0) == _lib.TF_OK

    def quant(x=16, r=1, c=8, ld=8, dtype=0, q=16, s=16):  # type: ignore[no-untyped-def]
        return lib.tf_e4m3_quant_groups(x, r, c, ld, dtype, q, s, None)

    assert quant(r=-1) == quant(c=0) == quant(ld=7) == quant(dtype=2) == bad
    assert quant(x=None) == quant(q=None) == quant(s=None) == bad
    assert quant(r=0) == _lib.TF_OK


# ------------------------------------------------------------------------------- host fast path


@pytest.mark.parametrize("group_size", [2**31, -(2**40), 2**70, -(10**30)])
def test_group_sizes_past_a_machine_word_are_refused(group_size: int) -> None:
    x = torch.zeros((2, 64), dtype=torch.float16)
    with pytest.raises(ValueError, match="group_size"):
        ops.silu_mul_fp8_quant(x, group_size)
    with pytest.raises(ValueError, match="group_size"):
        ops.add_rmsnorm_fp8_quant(x, x, x[0], 1e-6, group_size)


@pytest.fixture
def reload_host_path():  # type: ignore[no-untyped-def]
    """The host fast path is looked for anew inside the test, and again after it."""
    from tokenforge_b200 import fp8

    def reset() -> None:
        fp8._fast = None
        _lib.fp8_host.cache_clear()

    reset()
    yield
    reset()


def _careful_path_refuses() -> None:
    x = torch.zeros((2, 64), dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.e4m3_quant_groups(x)
    with pytest.raises(ValueError, match="group_size"):
        ops.silu_mul_fp8_quant(x, 32)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.add_rmsnorm_fp8_quant(x, x, x[0], 1e-6)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.w8a8_block_linear(**_linear_args())


def test_an_extension_of_another_pytorch_is_not_loaded(reload_host_path, monkeypatch) -> None:  # type: ignore[no-untyped-def]
    """The extension holds PyTorch's and CPython's inline code: one built against others is not
    taken, the operators warn once and go through Python."""
    monkeypatch.setattr(torch, "__version__", "0.0.1+other")
    with pytest.warns(RuntimeWarning, match="host fast path"):
        with pytest.raises(RuntimeError, match="CUDA"):
            ops.e4m3_quant_groups(torch.zeros((2, 64), dtype=torch.float16))
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        _careful_path_refuses()


def test_a_broken_extension_leaves_the_python_path(reload_host_path, monkeypatch, tmp_path) -> None:  # type: ignore[no-untyped-def]
    broken = tmp_path / "fp8_host.so"
    broken.write_bytes(b"not a shared object")
    monkeypatch.setattr(_lib, "host_path", lambda: broken)
    with pytest.warns(RuntimeWarning, match="host fast path"):
        _careful_path_refuses()


def test_the_build_makes_the_extension_that_is_loaded(reload_host_path) -> None:  # type: ignore[no-untyped-def]
    import sysconfig

    path = _lib.host_path()
    assert torch.__version__ in path.name and sysconfig.get_config_var("SOABI") in path.name
    assert path.exists(), "build() did not make the host extension for this PyTorch"
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        _careful_path_refuses()
    assert _lib.fp8_host().__file__ == str(path)


def test_registered_norm_without_a_residual_returns_packed_rows(monkeypatch) -> None:  # type: ignore[no-untyped-def]
    """The copy of x that the registered operator returns has the fake's layout, not x's own. The
    kernel's part is stood in for, so that the wrapper runs without a GPU."""
    def launcher(x, residual, weight, eps, group_size):  # type: ignore[no-untyped-def]
        return torch.empty(x.shape, dtype=E4M3), torch.empty((*x.shape[:-1], 1)), x

    monkeypatch.setattr(ops, "add_rmsnorm_fp8_quant", launcher)
    x = torch.randn((4, 3, 64)).half().transpose(0, 1)
    h = torch.ops.tokenforge.add_rmsnorm_fp8_quant(x, None, x[0, 0], 1e-6, 0)[2]
    assert torch.equal(h, x) and h.data_ptr() != x.data_ptr()
    assert h.stride() == (256, 64, 1)
