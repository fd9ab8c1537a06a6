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
__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint32_t abs_bits(float f) { return __float_as_uint(f) & 0x7FFFFFFFu; }

// scale = max(amax / 448, 1 / (448 * 512)) with the IEEE quotient: q0 = amax * RN(1 / 448) is
// within one ulp of it, and one residual correction rounds it correctly (tf_rmsnorm.cuh names the
// method), where the result is above the floor (far above the subnormal range). Inf and NaN have
// no residual: they keep q0.
__device__ __forceinline__ float scale_of_bits(uint32_t amax_bits) {
  constexpr float kInv = 1.0f / kFp8Max;
  const float a = __uint_as_float(amax_bits);
  float s = __fmul_rn(a, kInv);
  if (amax_bits < 0x7F800000u) s = __fmaf_rn(__fmaf_rn(-s, kFp8Max, a), kInv, s);
  return s < kMinScale ? kMinScale : s;
}

// y = g / (1 + exp(-g)) * u for a pair, exp(-g) = 2^(-g log2 e). The approximate exponential and
// reciprocal are within a few units of 2^-23 each (and the rounding of -g log2 e adds |g| of
// them, where y is small by e^-|g|). For g < -87 the quotient is 0, below 1e-36 of |u|.
__device__ __forceinline__ uint64_t silu_mul2(float2 g, float2 u) {
  const uint64_t x = mul_f32x2(f32x2(g.x, g.y), f32x2(-1.44269504f, -1.44269504f));
  const float2 t = split_f32x2(x);
  float e0, e1, r0, r1;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(t.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(t.y));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r0) : "f"(1.0f + e0));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r1) : "f"(1.0f + e1));
  return mul_f32x2(mul_f32x2(f32x2(g.x, g.y), f32x2(r0, r1)), f32x2(u.x, u.y));
}

// Maximum over the 16 lanes of a half warp that hold one 128-column group (8 columns a lane).
__device__ __forceinline__ uint32_t half_warp_max(uint32_t v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// e4m3 codes of eight values under one scale. kExact: each quotient is the IEEE division's (one
// residual correction of y * RN(1 / scale)); used where y is an input value of 16 bits, so that
// the codes are the exact ones. One correction is within 2^-22 ulp of the quotient's rounding; it
// could only change a code where a quotient lies that close to the middle between two fp32 values
// next to an e4m3 rounding boundary, and no 16-bit value under a scale of this rule does: all of
// them, under every maximum of either type, were compared with the division. Otherwise
// y * RN(1 / scale): y carries a few fp32 roundings of its own already, and 1.5 more of 2^-24 are
// far below e4m3's half step 2^-4. Every quotient whose code is not zero has |y| >= 2^-28 (scale
// >= 2^-17.8), so no step leaves the normal range where it counts; scales reach 7.6e35 (bf16),
// whose reciprocal is normal. An infinite scale has no residual (it would be NaN): it keeps y * 0.
template <bool kExact>
__device__ __forceinline__ uint2 codes8(const float (&y)[8], float scale) {
  const float r = __frcp_rn(scale);
  const uint64_t r2 = f32x2(r, r), nr2 = f32x2(-r, -r), b2 = f32x2(scale, scale);
  const bool correct = kExact && r != 0.f;
  uint32_t c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint64_t v = f32x2(y[2 * i], y[2 * i + 1]);
    uint64_t q = mul_f32x2(v, r2);
    // Residual b q - y times -r: in this sign a zero keeps its own.
    if (correct) q = fma_f32x2(fma_f32x2(b2, q, f32x2(-y[2 * i], -y[2 * i + 1])), nr2, q);
    const float2 f = split_f32x2(q);
    c[i] = cvt_e4m3x2(f.x, f.y);
  }
  return make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
}
// One code, for rows that are not 16-byte vectors.
template <bool kExact>
__device__ __forceinline__ uint8_t code1(float y, float scale) {
  const float r = __frcp_rn(scale);
  float q = __fmul_rn(y, r);
  if (kExact && r != 0.f) q = __fmaf_rn(__fmaf_rn(scale, q, -y), -r, q);
  return static_cast<uint8_t>(cvt_e4m3x2(q, 0.f) & 0xFFu);
}

// Division of n < 2^31 by a divisor fixed at launch: n / d = (mulhi(n, mul) + n) >> shift
// (T. Granlund, P. L. Montgomery, "Division by invariant integers using multiplication", 1994).
struct FastDiv {
  uint32_t d, mul, shift;
};
inline FastDiv fast_div(uint32_t d) {
  uint32_t shift = 0;
  while ((uint64_t(1) << shift) < d) ++shift;
  const uint64_t mul = ((uint64_t(1) << 32) * ((uint64_t(1) << shift) - d)) / d + 1;
  return FastDiv{d, static_cast<uint32_t>(mul), shift};
}
__device__ __forceinline__ uint32_t div_by(uint32_t n, const FastDiv& f) {
  return (__umulhi(n, f.mul) + n) >> f.shift;
}

}  // namespace tfb
