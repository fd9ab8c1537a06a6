"""GPU parity of the FP8 block-scaled (W8A8) operators against their definitions in 64 bits.

Tolerances, derived from the arithmetic:

* linear: e4m3 products are exact in fp32. Let S = sum of |xq wq| times the scales. A block's 128
  terms are added in fp32 (each addition off by at most 2^-23 of a partial sum <= S, truncation
  included), then scaled (two roundings) and added over the KB blocks, the K splits and the bias:
  (128 + KB + 32) * 2^-23 * S in all. The output's rounding adds eps(T) / 2 of the value, or half
  the smallest subnormal (2^-25 for fp16).
* codes: with v = y64 / scale, e4m3 rounds to within 2^-4 |v| or 2^-10; y is off by at most
  DELTA |y|, which moves v by as much.
* DELTA: norm: a term of the sum of squares passes at most 150 fp32 roundings (a thread's
  chain of <= 137 for the longest row tested, then 10 of the tree), so rstd is off by 75 + 4 of
  2^-24, y by two more: below 2^-17. silu: exp's error 2 + 1.16 |g| units of 2^-23 for |g| <= 88
  (below 2^-16.2), the division's 2 units and the product: below 2^-15. quant: none, y is the
  input and the codes and scales are exactly those of the fp32 division.
"""

from __future__ import annotations

import pytest
import torch

from tokenforge_b200 import _lib, ops
from tokenforge_b200.pack import FP8_MIN_SCALE, pack_w8a8_block

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn
DTYPES = [torch.float16, torch.bfloat16]
EPS = 1e-6
DELTA = {"norm": 2.0**-17, "silu": 2.0**-15}


def _gen(*key: int) -> torch.Generator:
    seed = 0
    for k in key:
        seed = (seed * 1000003 + k) % (1 << 31)
    return torch.Generator(device="cuda").manual_seed(seed)


# ------------------------------------------------------------------------------- linear


def _linear_inputs(m, n, k, dtype, bias, device):  # type: ignore[no-untyped-def]
    gen = _gen(m, n, k, 5)
    kb, nb = -(-k // 128), -(-n // 128)
    xq = (torch.randn((m, k), generator=gen, device=device) * 60).to(E4M3)
    wq = (torch.randn((n, k), generator=gen, device=device) * 60).to(E4M3)
    # Scales that differ by up to 16 from block to block: a scale taken from a neighbouring block
    # or row is far outside the tolerance.
    xs = torch.exp2(4 * torch.rand((m, kb), generator=gen, device=device) - 8)
    ws = torch.exp2(4 * torch.rand((nb, kb), generator=gen, device=device) - 10)
    b = torch.randn(n, generator=gen, device=device).to(dtype) if bias else None
    return xq, xs, wq, ws, b


def _linear_exact(xq, xs, wq, ws, b):  # type: ignore[no-untyped-def]
    """(y, S) in fp64."""
    (m, k), n = xq.shape, wq.shape[0]
    sx = xs.double().repeat_interleave(128, 1)[:, :k]
    sw = ws.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    x, w = xq.double() * sx, wq.double() * sw
    y, s = x @ w.t(), x.abs() @ w.abs().t()
    if b is not None:
        y, s = y + b.double(), s + b.double().abs()
    return y, s


def _check_linear(y, xq, xs, wq, ws, b):  # type: ignore[no-untyped-def]
    y64, s = _linear_exact(xq, xs, wq, ws, b)
    half = torch.finfo(y.dtype).eps / 2
    tol = half * y64.abs() + (128 + xs.shape[1] + 32) * 2.0**-23 * s * (1 + half) + 2.0**-25
    bad = (y.double() - y64).abs() > tol
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} outputs off"


LINEAR = [
    (1, 3584, 3584), (1, 1, 16), (1, 129, 144), (2, 4608, 3584), (3, 100, 18944), (5, 16, 128),
    (7, 1000, 2064), (8, 3584, 3584), (9, 3584, 1024), (15, 640, 1552), (16, 4608, 3584),
    (17, 256, 256), (31, 513, 656), (32, 3584, 3584), (33, 64, 4096), (63, 1000, 1008),
    (64, 3584, 18944), (65, 257, 400), (100, 3584, 3584), (128, 128, 128), (129, 385, 1168),
    (200, 4608, 3584), (256, 3584, 2368), (257, 1025, 272), (500, 100, 16), (1000, 1000, 1040),
    (1024, 3584, 3584), (1300, 2368, 3584), (2049, 513, 528),
    # Ragged sizes that are too large for the warp-MMA kernel: each tensor-core form, one and
    # several token tiles, K split and not.
    (5, 1003, 9232), (12, 5003, 2064), (16, 129, 16400), (17, 3601, 2576), (32, 20011, 144),
    (48, 2005, 4112), (64, 40001, 272), (70, 1999, 2064), (127, 3000, 1040), (130, 9001, 528),
    (333, 4613, 2960), (400, 515, 8208), (700, 2051, 1040), (1030, 777, 4112), (3000, 2050, 272),
]


@pytest.mark.parametrize("m, n, k", LINEAR)
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear(m: int, n: int, k: int, dtype: torch.dtype, device: torch.device) -> None:
    bias = (m + n) % 2 == 1
    args = _linear_inputs(m, n, k, dtype, bias, device)
    y = ops.w8a8_block_linear(*args, dtype)
    assert y.shape == (m, n) and y.dtype == dtype
    _check_linear(y, *args)
    assert torch.equal(y, ops.w8a8_block_linear(*args, dtype)), "a second call differs"


@pytest.mark.parametrize("n, k", [(264, 416), (2056, 2576)])
@pytest.mark.parametrize("m", [1, 4, 40, 300])
def test_linear_layouts(m: int, n: int, k: int, device: torch.device) -> None:
    """Leading dimensions, rows and scales cut out of wider tensors, misaligned and uint8 codes,
    a bias with a stride, an x expanded over its rows."""
    xq, xs, wq, ws, b = _linear_inputs(m, n, k, torch.float16, True, device)
    y = ops.w8a8_block_linear(xq, xs, wq, ws, b)
    same = [
        (xq.view(torch.uint8), xs, wq.view(torch.uint8), ws, b),
        (torch.cat([xq.view(torch.uint8)] * 2, 1).view(E4M3)[:, :k], xs, wq, ws, b),
        (torch.cat([xq.view(torch.uint8)[:, :3], xq.view(torch.uint8)], 1).view(E4M3)[:, 3:], xs,
         wq, ws, b),
        (xq, torch.cat([xs, xs], 1)[:, : xs.shape[1]], wq, ws, b),
        (xq, xs.t().contiguous().t(), wq, ws, b),
        (xq, xs, wq, ws, torch.stack([b, b], 1)[:, 0]),
    ]
    for i, a in enumerate(same):
        assert torch.equal(y, ops.w8a8_block_linear(*a)), f"layout {i}"
    y3 = ops.w8a8_block_linear(xq[None], xs[None], wq, ws, b)
    assert y3.shape == (1, m, n) and torch.equal(y3[0], y)
    assert ops.w8a8_block_linear(xq[:0], xs[:0], wq, ws, b).shape == (0, n)
    one = ops.w8a8_block_linear(xq[:1].expand(m, k), xs[:1].expand(m, xs.shape[1]), wq, ws, b)
    assert torch.equal(one, ops.w8a8_block_linear(xq[:1].repeat(m, 1), xs[:1].repeat(m, 1), wq,
                                                  ws, b))
    with pytest.raises(ValueError, match="aligned"):
        buf = torch.zeros(n * k + 8, dtype=torch.uint8, device=device)[8:].view(n, k)
        ops.w8a8_block_linear(xq, xs, buf, ws, b)


@pytest.mark.parametrize("n, k, ldy", [(200, 272, 216), (200, 272, 213), (2050, 2576, 2056),
                                       (2050, 2576, 2061), (1999, 4112, 2000)])
@pytest.mark.parametrize("m", [1, 8, 24, 64, 130, 300])
def test_linear_writes_its_rows_only(m: int, n: int, k: int, ldy: int,
                                     device: torch.device) -> None:
    """C ABI with an output wider than N and rows behind the last token."""
    xq, xs, wq, ws, _ = _linear_inputs(m, n, k, torch.float16, False, device)
    y = torch.full((m + 4, ldy), 7.0, dtype=torch.float16, device=device)
    lib = _lib.lib()
    status = lib.tf_w8a8_block_linear(
        xq.data_ptr(), m, k, k, xs.data_ptr(), xs.shape[1], wq.data_ptr(), ws.data_ptr(), None, n,
        _lib.TF_DTYPE_FP16, y.data_ptr(), ldy, _lib.stream_ptr(torch.device("cuda", 0)))
    _lib.check("tf_w8a8_block_linear", status)
    _check_linear(y[:m, :n], xq, xs, wq, ws, None)
    assert bool((y[m:] == 7).all()) and bool((y[:, n:] == 7).all())


@pytest.mark.parametrize("n, k", [(256, 384), (2048, 2560)])
@pytest.mark.parametrize("m", [1, 8, 48, 200])
def test_linear_special_values(m: int, n: int, k: int, device: torch.device) -> None:
    """A NaN code or scale reaches its own row (or column) alone; a zero scale and zero codes
    give 0; an overflowing sum gives the output type's infinity."""
    xq, xs, wq, ws, _ = _linear_inputs(m, n, k, torch.float16, False, device)
    xq = xq.clone().view(torch.uint8)
    xq[m // 2, 130] = 0x7F
    y = ops.w8a8_block_linear(xq, xs, wq, ws)
    nan = torch.isnan(y)
    assert bool(nan[m // 2].all()) and int(nan.sum()) == n
    wq2 = wq.clone().view(torch.uint8)
    wq2[77, 300] = 0xFF
    xq[m // 2, 130] = 0
    nan = torch.isnan(ops.w8a8_block_linear(xq, xs, wq2, ws))
    assert bool(nan[:, 77].all()) and int(nan.sum()) == m
    assert not bool(ops.w8a8_block_linear(xq, torch.zeros_like(xs), wq, ws).any())
    big = torch.full((m, k), 448.0, device=device).to(E4M3)
    y = ops.w8a8_block_linear(big, torch.ones_like(xs), big[:1].repeat(n, 1), torch.ones_like(ws))
    assert bool(torch.isposinf(y).all())


@pytest.mark.parametrize("m", [1, 20, 256])
def test_linear_stream_graph_and_overlap(m: int, device: torch.device) -> None:
    """Two streams at once, and two captured graphs replayed in turn with new inputs."""
    n, k = 3584, 3584
    a = _linear_inputs(m, n, k, torch.bfloat16, True, device)
    b = _linear_inputs(m, n, k + 16, torch.bfloat16, False, device)
    ya = ops.w8a8_block_linear(*a, torch.bfloat16)
    yb = ops.w8a8_block_linear(*b, torch.bfloat16)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        with torch.cuda.stream(s1):
            got.append((ops.w8a8_block_linear(*a, torch.bfloat16), ya))
        with torch.cuda.stream(s2):
            got.append((ops.w8a8_block_linear(*b, torch.bfloat16), yb))
    torch.cuda.synchronize()
    assert all(torch.equal(u, v) for u, v in got)
    graphs = []
    for args, want in ((a, ya), (b, yb)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = ops.w8a8_block_linear(*args, torch.bfloat16)
        graphs.append((g, y, want))
    for _ in range(3):
        for g, y, want in graphs:
            y.zero_()
            g.replay()
            assert torch.equal(y, want)
    a[0].copy_(a[0].flip(0))
    a[1].copy_(a[1].flip(0))
    graphs[0][0].replay()
    assert torch.equal(graphs[0][1], ops.w8a8_block_linear(*a, torch.bfloat16))


# ------------------------------------------------------------------------------- quantizers


def _groups(v: torch.Tensor, group: int) -> torch.Tensor:
    """amax |v| of each group of fp64 ``v`` [r, c]."""
    width = group or v.shape[1]
    g = -(-v.shape[1] // width)
    p = torch.nn.functional.pad(v.abs(), (0, g * width - v.shape[1]))
    return p.view(v.shape[0], g, width).amax(2)


def _check_codes(q, s, y64, group, delta):  # type: ignore[no-untyped-def]
    r, c = y64.shape
    want = (_groups(y64, group) / 448).clamp(min=FP8_MIN_SCALE)
    assert s.shape == want.shape and s.dtype == torch.float32
    assert bool(((s.double() - want).abs() <= want * (delta + 2.0**-23)).all()), "scales"
    v = y64 / s.double().repeat_interleave(group or c, 1)[:, :c]
    tol = v.abs() * (2.0**-4 + 2 * delta + 2.0**-20) + 2.0**-10 * (1 + 2.0**-12)
    bad = (q.double() - v).abs() > tol
    assert not bool(bad.any()), f"{int(bad.sum())} codes off"


def _stream(r, c, dtype, key, device, spread=2.0):  # type: ignore[no-untyped-def]
    gen = _gen(r, c, key)
    x = torch.randn((r, c), generator=gen, device=device) * spread
    x[:, c // 3] *= 30
    return x.to(dtype)


SHAPES = [(1, 3584), (1, 1), (3, 8), (2, 100), (5, 127), (4, 128), (7, 136), (33, 896), (16, 1000),
          (9, 4096), (3, 5000), (300, 3584), (2, 8200), (2, 18944), (1, 32768), (2, 32776),
          (1, 70001)]


@pytest.mark.parametrize("t, h", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", [128, 0])
def test_norm(t: int, h: int, dtype: torch.dtype, group: int, device: torch.device) -> None:
    x, r = _stream(t, h, dtype, 1, device, 1.0), _stream(t, h, dtype, 2, device, 4.0)
    w = (1 + 0.1 * torch.randn(h, generator=_gen(h), device=device)).to(dtype)
    q, s, total = ops.add_rmsnorm_fp8_quant(x, r, w, EPS, group)
    assert q.dtype == E4M3 and q.shape == total.shape == (t, h) and total.dtype == dtype
    want = (x.float() + r.float()).to(dtype)
    assert torch.equal(total, want)
    f = want.double()
    y64 = f / torch.sqrt(f.square().mean(1, keepdim=True) + EPS) * w.double()
    _check_codes(q, s, y64, group, DELTA["norm"])
    # Without a residual: the norm of x itself.
    q, s, total = ops.add_rmsnorm_fp8_quant(want, None, w, EPS, group)
    assert total is want
    _check_codes(q, s, y64, group, DELTA["norm"])


@pytest.mark.parametrize("m, i", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", [128, 0])
def test_silu(m: int, i: int, dtype: torch.dtype, group: int, device: torch.device) -> None:
    gu = _stream(m, 2 * i, dtype, 3, device)
    q, s = ops.silu_mul_fp8_quant(gu, group)
    assert q.dtype == E4M3 and q.shape == (m, i)
    g, u = gu.double().chunk(2, 1)
    _check_codes(q, s, g / (1 + torch.exp(-g)) * u, group, DELTA["silu"])


@pytest.mark.parametrize("r, c", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_quant_is_exact(r: int, c: int, dtype: torch.dtype, device: torch.device) -> None:
    x = _stream(r, c, dtype, 4, device)
    q, s = ops.e4m3_quant_groups(x)
    f = x.cpu().float()
    g = -(-c // 128)
    p = torch.nn.functional.pad(f, (0, g * 128 - c)).view(r, g, 128)
    want = torch.maximum(p.abs().amax(2) / torch.tensor(448.0), torch.tensor(FP8_MIN_SCALE))
    assert torch.equal(s.cpu(), want)
    codes = (p / want[:, :, None]).clamp(-448, 448).to(E4M3).view(r, g * 128)[:, :c]
    assert torch.equal(q.cpu().view(torch.uint8), codes.contiguous().view(torch.uint8))


@pytest.mark.parametrize("dtype", DTYPES)
def test_quant_every_value(dtype: torch.dtype, device: torch.device) -> None:
    """Every finite 16-bit value in groups of its own exponent's neighbours and under every other
    one's maximum: the codes are those of the IEEE division (fp64 division rounded to fp32 would
    round twice, so the CPU's fp32 division is the oracle)."""
    v = torch.arange(65536, dtype=torch.int32).to(torch.uint16).view(dtype)
    v = v[torch.isfinite(v)]
    n = v.numel() // 127 * 127
    body = v[torch.randperm(v.numel(), generator=torch.Generator().manual_seed(1))][:n].view(-1, 127)
    tops = v[v > 0][:: max(1, int((v > 0).sum()) // 60)]
    x = torch.cat([torch.cat([body, torch.full((body.shape[0], 1), float(t)).to(dtype)], 1)
                   for t in tops])
    q, s = ops.e4m3_quant_groups(x.to(device))
    want = torch.maximum(x.float().abs().amax(1, keepdim=True) / torch.tensor(448.0),
                         torch.tensor(FP8_MIN_SCALE))
    assert torch.equal(s.cpu(), want)
    codes = (x.float() / want).clamp(-448, 448).to(E4M3)
    assert torch.equal(q.cpu().view(torch.uint8), codes.view(torch.uint8))


@pytest.mark.parametrize("dtype", DTYPES)
def test_quant_every_value_under_every_maximum(dtype: torch.dtype, device: torch.device) -> None:
    """Each positive finite 16-bit value as a group's maximum over every value up to it, against
    the GPU's IEEE division (torch's tensor by tensor division): what the kernel's single
    residual correction rests on."""
    v = torch.arange(65536, dtype=torch.int32).to(torch.uint16).view(dtype).to(device)
    v = v[torch.isfinite(v)]
    body = torch.cat([v, v.new_zeros(-len(v) % 127)]).view(1, -1, 127)
    tops = v[v > 0]
    for i in range(0, len(tops), 128):
        t = tops[i : i + 128].view(-1, 1, 1)
        x = torch.cat([torch.where(body.abs() <= t, body, torch.zeros_like(body)),
                       t.expand(-1, body.shape[1], 1)], 2).reshape(-1, 128)
        q, s = ops.e4m3_quant_groups(x)
        amax = x.float().abs().amax(1, keepdim=True)
        want = torch.div(amax, torch.full_like(amax, 448.0)).clamp(min=FP8_MIN_SCALE)
        assert torch.equal(s, want)
        codes = torch.div(x.float(), want.expand(-1, 128)).clamp(-448, 448).to(E4M3)
        assert torch.equal(q.view(torch.uint8), codes.view(torch.uint8)), f"maxima from {i}"


@pytest.mark.parametrize("c", [256, 250])
@pytest.mark.parametrize("dtype", DTYPES)
def test_special_values(c: int, dtype: torch.dtype, device: torch.device) -> None:
    """NaN: its group's scale and codes are NaN. Inf: scale Inf, its code NaN, the others 0. Zeros
    and the type's smallest values: the scale's floor and zero codes. Its largest: finite."""
    inf, nan = float("inf"), float("nan")
    big, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    x = torch.ones((5, c), dtype=dtype, device=device)
    x[0, 3], x[1, 200], x[2] = nan, -inf, 0.0
    x[3], x[4] = tiny if dtype == torch.bfloat16 else 0.0, big

    def check(q, s, row_nan):  # type: ignore[no-untyped-def]
        q = q.float()
        a, b = (0, 1) if s.shape[1] > 1 else (0, 0)
        assert bool(torch.isnan(s[0, a])) and bool(torch.isnan(q[0, :128]).all())
        if s.shape[1] > 1 and not row_nan:
            assert not bool(torch.isnan(q[0, 128:]).any())
        if row_nan:  # an infinite row: rstd is 0, so Inf * 0 is NaN
            assert bool(torch.isnan(s[1, b]))
        else:
            assert bool(torch.isinf(s[1, b])) and bool(torch.isnan(q[1, 200]))
            assert int(torch.isnan(q[1]).sum()) == 1 and not bool(q[1, 201:].any())
        assert bool((s[2] == FP8_MIN_SCALE).all()) and not bool(q[2].any())
        assert bool(torch.isfinite(s[3:]).all()) and bool(torch.isfinite(q[3:]).all())

    check(*ops.e4m3_quant_groups(x), False)
    for group in (128, 0):
        # silu(g) * 1: NaN and -Inf in the up half instead
        gu = torch.cat([torch.ones_like(x), x], 1)
        gu[4, c:] = big / 4
        check(*ops.silu_mul_fp8_quant(gu, group), False)
        w = torch.ones(c, dtype=dtype, device=device)
        y = x.clone()
        y[4] = 2.0**15  # its square sum stays finite
        q, s, h = ops.add_rmsnorm_fp8_quant(y, torch.zeros_like(y), w, EPS, group)
        check(q, s, True)
        assert torch.equal(torch.nan_to_num(h, 5.0), torch.nan_to_num(y, 5.0))


@pytest.mark.parametrize("group", [128, 0])
def test_rows_cut_from_wider_tensors(group: int, device: torch.device) -> None:
    """Row strides, misaligned rows, leading dimensions, empty batches, expanded rows and strided
    columns give the codes of the packed rows."""
    t, h = 6, 392
    wide = _stream(t, 2 * h + 16, torch.bfloat16, 7, device)
    w = (1 + 0.1 * torch.randn(h, generator=_gen(1), device=device)).to(torch.bfloat16)
    for off in (0, 8, 1, 3):
        x = wide[:, off : off + h]
        r = wide[:, h + off : 2 * h + off]
        got = ops.add_rmsnorm_fp8_quant(x, r, w, EPS, group)
        want = ops.add_rmsnorm_fp8_quant(x.contiguous(), r.contiguous(), w, EPS, group)
        assert torch.equal(got[2], want[2])
        y64 = want[2].double()
        y64 = y64 / torch.sqrt(y64.square().mean(1, keepdim=True) + EPS) * w.double()
        _check_codes(got[0], got[1], y64, group, DELTA["norm"])
        g = wide[:, off : off + 2 * h]
        got, want = ops.silu_mul_fp8_quant(g, group), ops.silu_mul_fp8_quant(g.contiguous(), group)
        assert torch.equal(got[0].view(torch.uint8), want[0].view(torch.uint8))
        assert torch.equal(got[1], want[1])
        if group:
            got, want = ops.e4m3_quant_groups(x), ops.e4m3_quant_groups(x.contiguous())
            assert torch.equal(got[0].view(torch.uint8), want[0].view(torch.uint8))
            assert torch.equal(got[1], want[1])
    x = wide[:, :h]
    q, s, total = ops.add_rmsnorm_fp8_quant(x.reshape(2, 3, h), x.reshape(2, 3, h), w, EPS, group)
    assert q.shape == (2, 3, h) and s.shape[:2] == (2, 3) and total.shape == (2, 3, h)
    q, s, total = ops.add_rmsnorm_fp8_quant(x[:0], x[:0], w, EPS, group)
    assert q.shape == (0, h) and s.shape[0] == 0 and total.shape == (0, h)
    q, s = ops.silu_mul_fp8_quant(x[:1].expand(4, h), group)
    assert torch.equal(q.view(torch.uint8), q[:1].view(torch.uint8).expand_as(q))
    q2, s2 = ops.silu_mul_fp8_quant(wide[:, : 2 * h : 2], group)
    q3, s3 = ops.silu_mul_fp8_quant(wide[:, : 2 * h : 2].contiguous(), group)
    assert torch.equal(q2.view(torch.uint8), q3.view(torch.uint8)) and torch.equal(s2, s3)


def test_norm_in_place_through_the_abi(device: torch.device) -> None:
    """residual_out may be the residual or x: the same codes, the same sum; the rows behind the
    last stay as they were."""
    lib = _lib.lib()
    for h in (3584, 333):
        x, r = _stream(5, h, torch.float16, 8, device), _stream(5, h, torch.float16, 9, device)
        w = torch.ones(h, dtype=torch.float16, device=device)
        q0, s0, t0 = ops.add_rmsnorm_fp8_quant(x[:4], r[:4], w, EPS)
        for into in ("residual", "x"):
            x1, r1 = x.clone(), r.clone()
            out = r1 if into == "residual" else x1
            q = torch.zeros((5, h), dtype=torch.uint8, device=device)
            s = torch.zeros((5, s0.shape[1]), device=device)
            status = lib.tf_add_rmsnorm_fp8_quant(
                x1.data_ptr(), 4, h, h, r1.data_ptr(), h, w.data_ptr(), EPS, _lib.TF_DTYPE_FP16,
                128, q.data_ptr(), s.data_ptr(), out.data_ptr(), h,
                _lib.stream_ptr(torch.device("cuda", 0)))
            _lib.check("tf_add_rmsnorm_fp8_quant", status)
            assert torch.equal(q[:4], q0.view(torch.uint8)) and torch.equal(s[:4], s0)
            assert torch.equal(out[:4], t0)
            assert torch.equal(out[4], (r if into == "residual" else x)[4])
            assert not bool(q[4].any()) and not bool(s[4].any())


# ------------------------------------------------------------------------------- together


@pytest.mark.parametrize("m", [1, 6, 32, 150])
@pytest.mark.parametrize("dtype", DTYPES)
def test_mlp_block(m: int, dtype: torch.dtype, device: torch.device) -> None:
    """The MLP half of a decoder layer as it is used: norm, gate_up, silu, down, then the next
    norm; each step against its definition on the step's actual inputs, then the whole run
    captured and replayed on new inputs, and with programmatic dependent launch."""
    h, i = 640, 1184
    gen = _gen(m, 11)
    w1 = pack_w8a8_block(torch.randn((2 * i, h), generator=gen, device=device) / h**0.5)
    w2 = pack_w8a8_block(torch.randn((h, i), generator=gen, device=device) / i**0.5)
    gamma = (1 + 0.1 * torch.randn(h, generator=gen, device=device)).to(dtype)
    x, r = _stream(m, h, dtype, 12, device, 1.0), _stream(m, h, dtype, 13, device, 3.0)

    def run(check: bool):  # type: ignore[no-untyped-def]
        q, s, total = ops.add_rmsnorm_fp8_quant(x, r, gamma, EPS)
        gu = ops.w8a8_block_linear(q, s, w1.wq, w1.w_scale, None, dtype)
        q2, s2 = ops.silu_mul_fp8_quant(gu)
        d = ops.w8a8_block_linear(q2, s2, w2.wq, w2.w_scale, None, dtype)
        q3, s3, total3 = ops.add_rmsnorm_fp8_quant(d, total, gamma, EPS, 0)
        if check:
            _check_linear(gu, q, s, w1.wq, w1.w_scale, None)
            _check_linear(d, q2, s2, w2.wq, w2.w_scale, None)
            a, b = gu.double().chunk(2, 1)
            _check_codes(q2, s2, a / (1 + torch.exp(-a)) * b, 128, DELTA["silu"])
            f = total3.double()
            y64 = f / torch.sqrt(f.square().mean(1, keepdim=True) + EPS) * gamma.double()
            _check_codes(q3, s3, y64, 0, DELTA["norm"])
        return q3, s3, total3

    def same(a, b):  # type: ignore[no-untyped-def]
        return all(torch.equal(u.view(torch.uint8), v.view(torch.uint8)) for u, v in zip(a, b))

    want = run(True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(False)
    graph.replay()
    assert same(got, want)
    x.copy_(x.flip(1))
    want = run(True)
    graph.replay()
    assert same(got, want)
    old = _lib.get_launch_flags()
    try:
        _lib.set_launch_flags(_lib.TF_LAUNCH_PDL)
        for _ in range(20):
            last = run(False)
        assert same(last, want)
    finally:
        _lib.set_launch_flags(old)


def test_registered_ops_match_the_launchers(device: torch.device) -> None:
    t = torch.ops.tokenforge
    x = _stream(4, 512, torch.float16, 20, device)
    w = torch.ones(512, dtype=torch.float16, device=device)
    p = pack_w8a8_block(torch.randn((256, 512), generator=_gen(3), device=device))
    q, s, h = t.add_rmsnorm_fp8_quant(x, x, w, EPS, 128)
    assert torch.equal(h, x + x)
    _, _, h0 = t.add_rmsnorm_fp8_quant(x, None, w, EPS, 128)
    assert torch.equal(h0, x) and h0.data_ptr() != x.data_ptr()
    y = t.w8a8_block_linear(q, s, p.wq, p.w_scale, None, torch.float16)
    assert torch.equal(y, ops.w8a8_block_linear(q, s, p.wq, p.w_scale))
    q1, s1 = t.silu_mul_fp8_quant(x, 128)
    q2, s2 = ops.silu_mul_fp8_quant(x)
    assert torch.equal(q1.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s1, s2)
    q1, s1 = t.e4m3_quant_groups(x)
    q2, s2 = ops.e4m3_quant_groups(x)
    assert torch.equal(q1.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s1, s2)


def test_e4m3_per_row_codes_feed_the_w4a16_linear(device: torch.device) -> None:
    """group_size=0 gives what w4a16_linear_fp8 takes: one scale per token."""
    from tests.numerics import cases

    w = cases.layer_weights(256, 512, 1).to(device)
    x = _stream(3, 512, torch.float16, 21, device)
    gamma = torch.ones(512, dtype=torch.float16, device=device)
    q, s, _ = ops.add_rmsnorm_fp8_quant(x, x, gamma, EPS, 0)
    y = torch.ops.tokenforge.w4a16_linear_fp8(q, s, w.qweight_t, w.scales, w.qzeros, None, 128)
    deq = torch.ops.tokenforge.w4a16_dequant(w.qweight_t, w.scales, w.qzeros, 128).double()
    a = q.double() * s.double()
    y64, mag = a @ deq.t(), a.abs() @ deq.abs().t()
    tol = 2.0**-11 * y64.abs() + 700 * 2.0**-23 * mag + 2.0**-25
    assert bool(((y.double() - y64).abs() <= tol).all())


def test_host_threads_on_streams_of_their_own(device: torch.device) -> None:
    """Four host threads, a stream each, through every kernel form at once."""
    import threading

    p = pack_w8a8_block(torch.randn((1000, 528), generator=_gen(9), device=device))
    xs = [_stream(m, 528, torch.bfloat16, m, device) for m in (1, 20, 40, 300)]

    def chain(x):  # type: ignore[no-untyped-def]
        q, s = ops.e4m3_quant_groups(x)
        return ops.w8a8_block_linear(q, s, p.wq, p.w_scale, None, torch.bfloat16)

    want = [chain(x) for x in xs]
    torch.cuda.synchronize()
    same = []

    def work() -> None:
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                got = [chain(x) for x in xs]
            stream.synchronize()
            same.append(all(torch.equal(a, b) for a, b in zip(got, want)))

    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert same == [True] * 4
    assert _lib.device_error() == 0


def test_plain_and_careful_host_paths_agree(device: torch.device) -> None:
    """One-dimensional inputs, a Parameter as weight, an integer eps, a tensor subclass and a
    misaligned view give what the packed tensors give, whichever host path takes them."""
    class Sub(torch.Tensor):
        pass

    x = _stream(3, 640, torch.float16, 30, device)
    w = torch.nn.Parameter(torch.ones(640, dtype=torch.float16, device=device))
    q, s, h = ops.add_rmsnorm_fp8_quant(x, x, w, 1.0)
    q1, s1, h1 = ops.add_rmsnorm_fp8_quant(x, x, w, 1)
    assert torch.equal(q.view(torch.uint8), q1.view(torch.uint8)) and torch.equal(s, s1)
    q1, s1, h1 = ops.add_rmsnorm_fp8_quant(x[1], x[1], w, 1.0)
    assert q1.shape == (640,) and s1.shape == (5,) and torch.equal(h1, h[1])
    assert torch.equal(q1.view(torch.uint8), q[1].view(torch.uint8)) and torch.equal(s1, s[1])
    q2, s2 = ops.e4m3_quant_groups(x.as_subclass(Sub))
    q3, s3 = ops.e4m3_quant_groups(x)
    assert torch.equal(q2.view(torch.uint8), q3.view(torch.uint8)) and torch.equal(s2, s3)
    p = pack_w8a8_block(torch.randn((200, 640), generator=_gen(31), device=device))
    y = ops.w8a8_block_linear(q, s, p.wq, p.w_scale)
    assert torch.equal(ops.w8a8_block_linear(q[2], s[2], p.wq, p.w_scale), y[2])
    buf = torch.zeros(3 * 640 + 4, dtype=torch.uint8, device=device)
    off = buf[4:].view(3, 640)
    off.copy_(q.view(torch.uint8))
    assert torch.equal(ops.w8a8_block_linear(off, s, p.wq, p.w_scale), y)
