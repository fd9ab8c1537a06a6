"""GPU tests of the block-scaled FP8 linear's tensor-core kernels at sizes that are sure to reach
each of them, and of the activation operators where a CTA walks several rows.

Which kernel a call takes (w8a8_capi.cu, w8a8_gemm_sm100.cu): the warp-MMA kernel while the weight
bytes read by all passes of 8 tokens stay within 20 MB (one pass) or 10 MB (several); else up to
16, 32 and 64 tokens the kernel with that many tokens as columns; above 512 tokens always the CTA
pair kernel.
"""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_fp8_block import _linear_inputs
from tokenforge_b200 import _lib, ops

pytestmark = pytest.mark.gpu


def test_tensor_core_kernels_back_to_back(device: torch.device) -> None:
    """Programmatic dependents of different forms in one stream, without a pause: each CTA's shared
    memory and TMEM pass straight to the next kernel's, so whatever a kernel still had under way
    at its end (an arrival on a barrier of its own) would land in its successor. Pairs with K split
    over a cluster, pairs with several tiles each, and each token width of the other form."""
    sizes = [(640, 512, 2576), (1030, 2056, 400), (12, 5000, 2064), (700, 4613, 272),
             (24, 3600, 2576), (600, 264, 4112), (48, 2000, 4112), (2049, 2050, 144)]
    args = [_linear_inputs(m, n, k, torch.bfloat16, False, device) for m, n, k in sizes]
    want = []
    for a in args:
        want.append(ops.w8a8_block_linear(*a, torch.bfloat16))
        torch.cuda.synchronize()
    for _ in range(25):
        got = [ops.w8a8_block_linear(*a, torch.bfloat16) for a in args]
    torch.cuda.synchronize()
    for size, g, w in zip(sizes, got, want):
        assert torch.equal(g, w), size
    assert _lib.device_error() == 0
