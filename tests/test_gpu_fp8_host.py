"""GPU tests of how the FP8 block-scaled operators behave towards their callers: exception types,
the interpreter lock, traced programs and errors of earlier launches."""

from __future__ import annotations

import threading
import time

import pytest
import torch

from tokenforge_b200 import _lib, ops
from tokenforge_b200.pack import pack_w8a8_block

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


def test_outputs_that_do_not_fit_raise_out_of_memory(device: torch.device) -> None:
    """Under a limit on this process's memory, an output above it raises torch.OutOfMemoryError (a
    RuntimeError's subclass that serving code catches), from every operator."""
    x = torch.zeros((1 << 16, 4096), dtype=torch.float16, device=device)
    w = torch.ones(4096, dtype=torch.float16, device=device)
    xq = torch.zeros((1 << 16, 16), dtype=E4M3, device=device)
    xs, ws = torch.ones((1 << 16, 1), device=device), torch.ones((64, 1), device=device)
    wq = torch.zeros((8192, 16), dtype=E4M3, device=device)
    calls = [
        lambda: ops.add_rmsnorm_fp8_quant(x, x, w, 1e-6),
        lambda: ops.silu_mul_fp8_quant(x),
        lambda: ops.e4m3_quant_groups(x),
        lambda: ops.w8a8_block_linear(xq, xs, wq, ws),
    ]
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(device).total_memory
    used = torch.cuda.memory_reserved(device)
    try:
        torch.cuda.set_per_process_memory_fraction((used + (8 << 20)) / total)
        for call in calls:
            with pytest.raises(torch.OutOfMemoryError):
                call()
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    ops.e4m3_quant_groups(x)


def test_other_threads_run_while_a_launch_waits(device: torch.device) -> None:
    """With the launch queue full behind a kernel of 0.4 s or more (torch's bounded spin), the call
    that waits for a free place must let other Python threads run, as every torch call does."""
    x = torch.zeros((1, 256), dtype=torch.float16, device=device)
    ops.e4m3_quant_groups(x)

    def longest_gap() -> float:
        gaps: list[float] = []
        stop = threading.Event()

        def tick() -> None:
            last = time.perf_counter()
            while not stop.is_set():
                time.sleep(0.001)
                now = time.perf_counter()
                gaps.append(now - last)
                last = now

        torch.cuda.synchronize()
        thread = threading.Thread(target=tick)
        thread.start()
        try:
            begin = time.perf_counter()
            torch.cuda._sleep(800_000_000)  # cycles: 0.4 s at the highest clock, 1.965 GHz
            for _ in range(6000):
                ops.e4m3_quant_groups(x)
            enqueued = time.perf_counter() - begin
            torch.cuda.synchronize()
        finally:
            stop.set()
            thread.join()
        assert enqueued > 0.3, "the queue was not full: nothing waited"
        return max(gaps)

    # A busy host may hold a thread up once; a launch that keeps the lock does it every time.
    gaps = [longest_gap()]
    while gaps[-1] > 0.15 and len(gaps) < 4:
        gaps.append(longest_gap())
    assert gaps[-1] <= 0.15, f"another thread stood still for {gaps} s"


def test_without_the_extension_the_results_are_the_same(device: torch.device, monkeypatch) -> None:  # type: ignore[no-untyped-def]
    from tokenforge_b200 import fp8

    gen = torch.Generator(device=device).manual_seed(5)
    x = torch.randn((20, 640), generator=gen, device=device).bfloat16()
    p = pack_w8a8_block(torch.randn((200, 640), generator=gen, device=device))
    w = torch.ones(640, dtype=torch.bfloat16, device=device)

    def run():  # type: ignore[no-untyped-def]
        q, s, h = ops.add_rmsnorm_fp8_quant(x, x, w, 1e-6)
        y = ops.w8a8_block_linear(q, s, p.wq, p.w_scale, None, torch.bfloat16)
        return [q, s, h, y, *ops.silu_mul_fp8_quant(x, 0), *ops.e4m3_quant_groups(x)]

    want = run()
    monkeypatch.setattr(fp8, "_fast", fp8._NoFastPath())
    for a, b in zip(want, run(), strict=True):
        assert a.dtype == b.dtype and torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def _operands(device):  # type: ignore[no-untyped-def]
    """Arguments of the four registered operators on inputs of several layouts."""
    gen = torch.Generator(device=device).manual_seed(3)
    w = torch.ones(64, dtype=torch.float16, device=device)
    p = pack_w8a8_block(torch.randn((48, 64), generator=gen, device=device))

    def layouts(c):  # type: ignore[no-untyped-def]
        base = torch.randn((4, 3, 2 * c), generator=gen, device=device).half()
        return [base[:, :, :c].contiguous(), base[:, :, :c], base[:, :, :c].contiguous().transpose(0, 1),
                base[:, :, ::2], base[:, :, :c].contiguous().permute(2, 0, 1).contiguous().permute(1, 2, 0)]

    t = torch.ops.tokenforge
    for x in layouts(64):
        yield t.add_rmsnorm_fp8_quant, (x, None, w, 1e-6, 128)
        yield t.add_rmsnorm_fp8_quant, (x, x.flip(0), w, 1e-6, 0)
        yield t.silu_mul_fp8_quant, (x, 128)
        yield t.e4m3_quant_groups, (x,)
        q, s = ops.e4m3_quant_groups(x)
        yield t.w8a8_block_linear, (q, s, p.wq, p.w_scale, None, torch.bfloat16)
        q, s = q.transpose(0, 1), s.transpose(0, 1)
        yield t.w8a8_block_linear, (q, s, p.wq, p.w_scale, None, torch.float16)


def test_registered_ops_pass_opcheck(device: torch.device) -> None:
    """test_schema multiplies its inputs and outputs, which torch does not do in e4m3."""
    for op, args in _operands(device):
        torch.library.opcheck(op.default, args, test_utils="test_faketensor")


def test_fakes_give_the_strides(device: torch.device) -> None:
    """What a traced program plans with is what the operator returns, layout included."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    for op, args in _operands(device):
        real = op(*args)
        with FakeTensorMode() as mode:
            fake = op(*[mode.from_tensor(a) if isinstance(a, torch.Tensor) else a for a in args])
        real, fake = (r if isinstance(r, tuple) else (r,) for r in (real, fake))
        for r, f in zip(real, fake, strict=True):
            assert (r.shape, r.dtype, r.stride()) == (f.shape, f.dtype, f.stride()), (op, args)


def _launches(lib, device):  # type: ignore[no-untyped-def]
    """C ABI calls of every FP8 kernel's launcher, each taking a stream."""
    x = torch.zeros((600, 512), dtype=torch.float16, device=device)
    w = torch.ones(512, dtype=torch.float16, device=device)
    q = torch.zeros((600, 512), dtype=torch.uint8, device=device)
    s = torch.zeros((600, 4), device=device)
    wq = torch.zeros((512, 512), dtype=torch.uint8, device=device)
    ws = torch.zeros((4, 4), device=device)
    h, y = torch.empty_like(x), torch.empty_like(x)

    def linear(m, n):  # type: ignore[no-untyped-def]
        return lambda stream: lib.tf_w8a8_block_linear(
            q.data_ptr(), m, 512, 512, s.data_ptr(), 4, wq.data_ptr(), ws.data_ptr(), None, n, 0,
            y.data_ptr(), 512, stream)

    return {
        "quant": lambda stream: lib.tf_e4m3_quant_groups(
            x.data_ptr(), 4, 512, 512, 0, q.data_ptr(), s.data_ptr(), stream),
        "silu": lambda stream: lib.tf_silu_mul_fp8_quant(
            x.data_ptr(), 4, 256, 512, 0, 0, q.data_ptr(), s.data_ptr(), stream),
        "norm": lambda stream: lib.tf_add_rmsnorm_fp8_quant(
            x.data_ptr(), 4, 512, 512, x.data_ptr(), 512, w.data_ptr(), 1e-6, 0, 128,
            q.data_ptr(), s.data_ptr(), h.data_ptr(), 512, stream),
        "linear, warp MMA": linear(4, 512),
        "linear, tensor cores": linear(600, 512),
    }


@pytest.mark.parametrize("name", ["quant", "silu", "norm", "linear, warp MMA",
                                  "linear, tensor cores"])
def test_a_refused_launch_does_not_fail_the_next_call(name: str, device: torch.device) -> None:
    """A launch that CUDA refuses (here: into the legacy stream while another stream captures) is
    reported by its own call alone; the next calls of the library succeed."""
    from cuda.bindings import runtime as rt

    lib = _lib.lib()
    launch = _launches(lib, device)[name]
    words = torch.zeros((128, 2), dtype=torch.int32, device=device)
    packed = torch.zeros((16, 16), dtype=torch.int32, device=device)
    torch.cuda.synchronize()
    err, side = rt.cudaStreamCreate()  # a blocking one: it excludes work in the legacy stream
    assert err == 0
    mode = rt.cudaStreamCaptureMode.cudaStreamCaptureModeGlobal
    assert rt.cudaStreamBeginCapture(side, mode)[0] == 0
    status = launch(None)
    rt.cudaStreamEndCapture(side)
    rt.cudaStreamDestroy(side)
    assert status == _lib.TF_ERR_CUDA
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.tf_awq_repack(words.data_ptr(), 128, 16, packed.data_ptr(), stream) == _lib.TF_OK
    assert launch(stream) == _lib.TF_OK
    torch.cuda.synchronize()
