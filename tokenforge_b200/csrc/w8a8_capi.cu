// C ABI of the block-scaled FP8 linear: argument checks and the choice of kernel.
#include "tf_common.cuh"
#include "tf_plan.h"
#include "tf_w8a8.h"

using namespace tfb;

extern "C" int tf_w8a8_block_linear(const uint8_t* xq, int64_t M, int64_t K, int64_t ldx,
                                    const float* x_scale, int64_t ld_xs, const uint8_t* wq,
                                    const float* w_scale, const uint16_t* bias, int64_t N,
                                    int32_t dtype, uint16_t* y, int64_t ldy, void* stream) {
  if (M < 0 || N < 1 || K < 1 || (dtype != TF_DTYPE_FP16 && dtype != TF_DTYPE_BF16))
    return TF_ERR_INVALID_ARG;
  if (K % 16 != 0) return TF_ERR_UNSUPPORTED;
  if (M == 0) return TF_OK;
  if (!xq || !x_scale || !wq || !w_scale || !y || ldx < K || ld_xs < cdiv(K, 128) || ldy < N)
    return TF_ERR_INVALID_ARG;
  if (!aligned16(xq) || !aligned16(wq) || ldx % 16 != 0) return TF_ERR_ALIGNMENT;
  // Tile coordinates are 32-bit numbers.
  constexpr int64_t kMost = int64_t(1) << 30;
  if (M > kMost || N > kMost || K > kMost) return TF_ERR_TOO_LARGE;
  const W8A8Args a{xq, x_scale, wq, w_scale, bias, y, M, N, K, ldx, ld_xs, ldy, dtype};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  // The warp-MMA kernel starts soonest and needs no tensor maps; the tensor-core kernels stream
  // more weights at once, read them once for more tokens and split a long K over more SMs. Up to
  // 8 tokens it takes weights of 20 MB (3584 x 3584: 6.0 against 7.2 us; 7168 x 3584: 10.4 against
  // 9.5; 512 x 18944: 18.8 against 10.5). More tokens read the weights again, 8 at a time, from
  // L2: up to 10 MB of such reads (64 x 1000 x 1008: 4.7 against 5.8 us, 16 x 2048 x 2048: 4.0
  // against 6.0, 16 x 3584 x 3584: 10.0 against 7.4).
  const int64_t passes = cdiv(M, 8);
  const bool gemv = K <= 8192 && M <= 2048 &&
                    passes * N * K <= (int64_t(passes == 1 ? 20 : 10) << 20);
  return gemv ? launch_w8a8_gemv(a, s) : launch_w8a8_tc(a, s);
}
