// Decode form of the block-scaled FP8 linear: y[m, n] = sum_b sx[m, b] sw[n / 128, b] *
// sum_{k in b} xq[m, k] wq[n, k] for few tokens, bound by reading the weights once.
//
// A warp owns 16 weight rows and walks 128-wide K blocks; its m16n8k32 e4m3 MMAs put the rows in
// the MMA's m and 8 tokens in its n dimension. The order of k inside a block is free as long as
// both operands share it, so every lane loads 16 contiguous bytes of its row (and of its token)
// and feeds their four words to two MMAs: no shared memory, no conversion, no shuffle. The four
// MMAs of a block start from zero, and their fp32 sum is scaled into the running fp32 sum, so
// nothing is accumulated across blocks under different scales. K is split over the warps of a
// CTA (block b goes to warp b mod WK), whose sums are added in warp order in shared memory. More
// than 8 tokens are more rows of CTAs, which find the weights in L2.
//
// Measured: 1 x 3584 x 3584 in 6.0 us with cold weights (4.6 to 5.6 us a call in a stream of them),
// 64 x 1000 x 1008 in 4.7 us. Bound by launch and one HBM round trip there; on 136 MB it
// stops at 3.9 TB/s (bytes in flight: 16 warps an SM, three 2 KB blocks each), where the
// tensor-core kernel takes over.
#include <algorithm>

#include "tf_common.cuh"
#include "tf_fp8_act.cuh"
#include "tf_plan.h"
#include "tf_w8a8.h"

namespace tfb {
namespace {

constexpr int kWarps = 8;
constexpr int kRows = 16;    // weight rows of a warp tile
constexpr int kTokens = 8;   // tokens of a CTA
constexpr int kStages = 3;   // K blocks in flight per warp

__device__ __forceinline__ void mma_e4m3(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

struct Stage {
  uint4 w[2][2];  // [row g, g + 8][64-wide half of the block]
  uint4 x[2];     // token g
  float sx[2];    // tokens 2t, 2t + 1
  float sw;
};

template <typename T>
__global__ void __launch_bounds__(32 * kWarps, 2) w8a8_gemv_kernel(const W8A8Args a, int wk,
                                                                  int w_early) {
  __shared__ float part[kWarps][kTokens][kRows + 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int wn = kWarps / wk;                  // row tiles of this CTA
  const int tile = warp / wk, kw = warp % wk;  // this warp's tile and share of K
  const int64_t row0 = (static_cast<int64_t>(blockIdx.x) * wn + tile) * kRows;
  const int64_t m0 = static_cast<int64_t>(blockIdx.y) * kTokens;
  const int kblocks = static_cast<int>(cdiv(a.K, 128));
  // Rows past N read row N - 1 (their sums are dropped); tokens past M are zeros.
  const uint8_t* wr0 = a.wq + min(row0 + g, a.N - 1) * a.K + 16 * t;
  const uint8_t* wr1 = a.wq + min(row0 + g + 8, a.N - 1) * a.K + 16 * t;
  const uint8_t* xr = a.xq + (m0 + g) * a.ldx + 16 * t;
  const float* swr = a.w_scale + (min(row0, a.N - 1) / 128) * kblocks;
  const float* sx0 = a.x_scale + (m0 + 2 * t) * a.ld_xs;
  const float* sx1 = sx0 + a.ld_xs;
  const bool x_ok = m0 + g < a.M, s0_ok = m0 + 2 * t < a.M, s1_ok = m0 + 2 * t + 1 < a.M;
  const uint4 zero = make_uint4(0, 0, 0, 0);

  Stage st[kStages];
  if (!w_early) pdl_begin();
  auto load_w = [&](Stage& s, int b) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t k = static_cast<int64_t>(b) * 128 + 64 * h;
      const bool ok = k + 16 * t < a.K;
      s.w[0][h] = ok ? ld_stream_v4(wr0 + k) : zero;
      s.w[1][h] = ok ? ld_stream_v4(wr1 + k) : zero;
    }
    s.sw = swr[b];
  };
  auto load_x = [&](Stage& s, int b) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t k = static_cast<int64_t>(b) * 128 + 64 * h;
      s.x[h] = x_ok && k + 16 * t < a.K ? *reinterpret_cast<const uint4*>(xr + k) : zero;
    }
    s.sx[0] = s0_ok ? sx0[b] : 0.f;
    s.sx[1] = s1_ok ? sx1[b] : 0.f;
  };
#pragma unroll
  for (int s = 0; s < kStages; ++s)
    if (kw + s * wk < kblocks) load_w(st[s], kw + s * wk);
  // The activations may belong to the preceding kernel.
  if (w_early) pdl_begin();
#pragma unroll
  for (int s = 0; s < kStages; ++s)
    if (kw + s * wk < kblocks) load_x(st[s], kw + s * wk);

  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int b0 = kw; b0 < kblocks; b0 += kStages * wk) {
#pragma unroll
    for (int s = 0; s < kStages; ++s) {
      const int b = b0 + s * wk;
      if (b < kblocks) {
        float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint4 &u = st[s].w[0][h], &v = st[s].w[1][h], &x = st[s].x[h];
          mma_e4m3(d, u.x, v.x, u.y, v.y, x.x, x.y);
          mma_e4m3(d, u.z, v.z, u.w, v.w, x.z, x.w);
        }
        const float f0 = st[s].sx[0] * st[s].sw, f1 = st[s].sx[1] * st[s].sw;
        acc[0] = fmaf(d[0], f0, acc[0]);
        acc[1] = fmaf(d[1], f1, acc[1]);
        acc[2] = fmaf(d[2], f0, acc[2]);
        acc[3] = fmaf(d[3], f1, acc[3]);
        const int nb = b + kStages * wk;
        if (nb < kblocks) {
          load_w(st[s], nb);
          load_x(st[s], nb);
        }
      }
    }
  }
  part[warp][2 * t][g] = acc[0];
  part[warp][2 * t + 1][g] = acc[1];
  part[warp][2 * t][g + 8] = acc[2];
  part[warp][2 * t + 1][g + 8] = acc[3];
  __syncthreads();
  // Outputs of the CTA: wn tiles x 8 tokens x 16 rows.
  for (int i = threadIdx.x; i < wn * kTokens * kRows; i += 32 * kWarps) {
    const int r = i % kRows, tl = (i / kRows) % wn, m = i / (kRows * wn);
    const int64_t n = (static_cast<int64_t>(blockIdx.x) * wn + tl) * kRows + r;
    if (n < a.N && m0 + m < a.M) {
      float v = 0.f;
      for (int w = 0; w < wk; ++w) v += part[tl * wk + w][m][r];
      if (a.bias != nullptr) v += widen(reinterpret_cast<const T*>(a.bias)[n]);
      narrow(v, reinterpret_cast<T*>(a.y) + (m0 + m) * a.ldy + n);
    }
  }
}

}  // namespace

// K is split over more warps until the warps fill 148 SMs of 16, and never so far that a warp
// has no block.
int launch_w8a8_gemv(const W8A8Args& a, cudaStream_t stream) {
  const int64_t tiles = cdiv(a.N, kRows), kblocks = cdiv(a.K, 128);
  int wk = 1;
  while (wk < kWarps && tiles * wk < 148 * 16 && 2 * wk <= kblocks) wk *= 2;
  const int64_t gx = cdiv(tiles, kWarps / wk), gy = cdiv(a.M, kTokens);
  if (gx > 0x7fffffffLL || gy > 65535) return TF_ERR_TOO_LARGE;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(gx), static_cast<unsigned>(gy));
  cfg.blockDim = dim3(32 * kWarps);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const int w_early = (launch_flags() & TF_LAUNCH_PDL) ? 1 : 0;
  const cudaError_t e = a.dtype == TF_DTYPE_FP16
                            ? cudaLaunchKernelEx(&cfg, w8a8_gemv_kernel<__half>, a, wk, w_early)
                            : cudaLaunchKernelEx(&cfg, w8a8_gemv_kernel<__nv_bfloat16>, a, wk,
                                                 w_early);
  if (e != cudaSuccess) return cuda_failed(e);
  return TF_OK;
}

}  // namespace tfb
