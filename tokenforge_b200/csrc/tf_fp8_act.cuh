// Element helpers of the FP8 activation operators (fp8_act.cu): fp16 / bf16 vectors widened to
// fp32, the |y| maximum on bit patterns, and the e4m3 codes of a group under one scale.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "tf_common.cuh"
#include "tf_rmsnorm.cuh"

namespace tfb {

// Two packed values as fp32.
__device__ __forceinline__ float2 widen2(uint32_t v, __half) {
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
__device__ __forceinline__ float2 widen2(uint32_t v, __nv_bfloat16) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
}
// Two fp32 values rounded to nearest and packed.
__device__ __forceinline__ uint32_t narrow2(float lo, float hi, __half) {
  return h2_as_u32(__floats2half2_rn(lo, hi));
}
__device__ __forceinline__ uint32_t narrow2(float lo, float hi, __nv_bfloat16) {
  const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&b);
}
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void narrow(float f, __half* out) { *out = __float2half_rn(f); }
__device__ __forceinline__ void narrow(float f, __nv_bfloat16* out) { *out = __float2bfloat16_rn(f); }

template <typename T>
__device__ __forceinline__ void widen8(const uint4& v, float (&f)[8]) {
  const uint32_t* u = reinterpret_cast<const uint32_t*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 p = widen2(u[i], T());
    f[2 * i] = p.x;
    f[2 * i + 1] = p.y;
  }
}

// |y| maxima are taken on the bit patterns of |y| as unsigned integers. For finite values that
// is the order of the values; Inf is above them and NaN above Inf, so a NaN in a group becomes
// its maximum, its scale and (below) every code of it, as in the elementary operations.
__device__ __forceinline__ uint32_t abs_bits(float f) { return __float_as_uint(f) & 0x7FFFFFFFu; }

// scale = max(amax / 448, 1 / (448 * 512)); a NaN maximum gives a NaN scale.
__device__ __forceinline__ float scale_of_bits(uint32_t amax_bits) {
  const float a = __uint_as_float(amax_bits);
  const float s = __fdiv_rn(a, kFp8Max);
  return s < kMinScale ? kMinScale : s;
}

// Maximum over the 16 lanes of a half warp that hold one 128-column group (8 columns a lane).
__device__ __forceinline__ uint32_t half_warp_max(uint32_t v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Divisor of one group. kExact: the quotient y / scale is the IEEE division's (two residual
// corrections of y * RN(1 / scale), tf_rmsnorm.cuh names the method): used where y is an input
// value, so that the codes are the exact ones. Otherwise y * RN(1 / scale): y carries a few
// fp32 roundings of its own already, and 1.5 more of 2^-24 are far below e4m3's half step 2^-4.
// Every quotient whose code is not zero has |y| >= 2^-28 (scale >= 2^-17.8), so no step below
// leaves the normal range where it counts; scales reach 7.6e35 (bf16), whose reciprocal is
// normal.
struct GroupDiv {
  float b, r;
};
__device__ __forceinline__ GroupDiv group_div(float scale) {
  return GroupDiv{scale, __frcp_rn(scale)};
}
template <bool kExact>
__device__ __forceinline__ float divide(float y, const GroupDiv& d) {
  float q = __fmul_rn(y, d.r);
  if constexpr (kExact) {
    // An infinite scale (an infinite value in the group) makes the residual NaN: keep y * 0.
    if (d.r != 0.f) {
      // Residual b q - y times -r: in this sign a zero keeps its own.
      q = __fmaf_rn(__fmaf_rn(d.b, q, -y), -d.r, q);
      q = __fmaf_rn(__fmaf_rn(d.b, q, -y), -d.r, q);
    }
  }
  return q;
}
template <bool kExact>
__device__ __forceinline__ uint2 codes8(const float (&y)[8], const GroupDiv& d) {
  uint32_t c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    c[i] = cvt_e4m3x2(divide<kExact>(y[2 * i], d), divide<kExact>(y[2 * i + 1], d));
  return make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
}

}  // namespace tfb
