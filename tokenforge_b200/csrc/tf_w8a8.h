// Operands and launchers of the block-scaled FP8 (W8A8) linear.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace tfb {

struct W8A8Args {
  const uint8_t* xq;     // e4m3 [M, K], row stride ldx bytes
  const float* x_scale;  // [M, ceil(K / 128)], row stride ld_xs
  const uint8_t* wq;     // e4m3 [N, K]
  const float* w_scale;  // [ceil(N / 128), ceil(K / 128)]
  const uint16_t* bias;  // dtype [N] or null
  uint16_t* y;           // dtype [M, N], row stride ldy
  int64_t M, N, K, ldx, ld_xs, ldy;
  int32_t dtype;         // TF_DTYPE_FP16 / TF_DTYPE_BF16
};

int launch_w8a8_gemv(const W8A8Args& a, cudaStream_t stream);
int launch_w8a8_tc(const W8A8Args& a, cudaStream_t stream);

}  // namespace tfb
