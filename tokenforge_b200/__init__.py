"""B200-native (sm_100a) backend for TokenForge's quantized-linear hot path.

Importing :mod:`tokenforge_b200.ops` registers the ``torch.ops.tokenforge`` namespace
(``w4a16_linear``, ``w4a16_dequant``, ``rmsnorm_fp8_quant``, ``awq_repack``) on top of the
kernel library ``lib/libtokenforge_b200.so``, whose C ABI is declared in
``include/tokenforge_b200.h``. The same namespace holds the FP8 block-scaled path
(``w8a8_block_linear``, ``add_rmsnorm_fp8_quant``, ``silu_mul_fp8_quant``,
``e4m3_quant_groups``; :mod:`tokenforge_b200.fp8`).
"""

from tokenforge_b200.pack import (
    AWQ_ORDER,
    AWQ_REVERSE_ORDER,
    PACK_FACTOR,
    SUPPORTED_GROUP_SIZES,
    W4A16Weights,
    W8A8BlockWeights,
)

__all__ = [
    "AWQ_ORDER",
    "AWQ_REVERSE_ORDER",
    "PACK_FACTOR",
    "SUPPORTED_GROUP_SIZES",
    "W4A16Weights",
    "W8A8BlockWeights",
]
