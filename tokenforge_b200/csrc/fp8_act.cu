// FP8 activation operators of the block-scaled (W8A8) linear path: each reads its fp16 or bf16
// input once and writes e4m3 codes with a scale per 128 columns of a row (or per row).
//
//   tf_add_rmsnorm_fp8_quant  h = T(x + residual); y = h * rsqrt(mean(h^2) + eps) * weight
//   tf_silu_mul_fp8_quant     y = g / (1 + exp(-g)) * u
//   tf_e4m3_quant_groups      y = x
//   scale = max(amax|y| / 448, 1 / (448 * 512)),  q = e4m3_rne_satfinite(y / scale)
//
// Everything between the input and the codes is fp32: y is not rounded to the stream's type
// (the reference's rmsnorm_fp8_quant, kept as its own operator, rounds it twice). h is, because
// it is an output: the next layer adds to the rounded sum, so the norm is of that sum too.
// A 128-column group is 16 lanes of 8 columns (one 16-byte vector each), so its maximum is four
// shuffles inside a half warp and no row-wide step is needed after the norm's sum of squares.
//
// Measured, inputs larger than L2: norm 8192 x 3584 bf16 33.7 us (6.1 TB/s, 95 % of a copy's rate),
// silu 4096 x 18944 bf16 66.3 us (5.9 TB/s), per row 64.3 us, quant 8192 x 18944 80.5 us (5.8 TB/s):
// bound by HBM, with instruction issue at about three quarters. One row: 2.0 to 2.7 us.
#include <algorithm>

#include "tf_common.cuh"
#include "tf_fp8_act.cuh"
#include "tf_plan.h"

namespace tfb {
namespace {

constexpr int kGroup = 128;
constexpr int kGroupVecs = kGroup / 8;

__device__ __forceinline__ uint32_t warp_max_bits(uint32_t v) {
  return __reduce_max_sync(0xffffffffu, v);
}

__device__ __forceinline__ float warp_sum_f(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Block-wide maximum / sum: one value a warp in shared memory, then every warp reduces them.
__device__ __forceinline__ uint32_t block_max_bits(uint32_t v, uint32_t* sh) {
  v = warp_max_bits(v);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  return warp_max_bits(lane < static_cast<int>(blockDim.x >> 5) ? sh[lane] : 0u);
}
__device__ __forceinline__ float block_sum_f(float v, float* sh) {
  v = warp_sum_f(v);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  return warp_sum_f(lane < static_cast<int>(blockDim.x >> 5) ? sh[lane] : 0.f);
}

__device__ __forceinline__ uint32_t max_bits8(const float (&y)[8]) {
  float m = fabsf(y[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) m = max_nan(m, fabsf(y[i]));
  return abs_bits(m);
}

__device__ __forceinline__ float rstd_f(float sumsq, int64_t H, float eps) {
  return __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(sumsq, static_cast<float>(H)), eps)));
}

// y = h * rstd * weight of one vector.
template <typename T>
__device__ __forceinline__ void norm8(const uint4& h, const uint4& w, float rstd, float (&y)[8]) {
  const uint32_t* hp = reinterpret_cast<const uint32_t*>(&h);
  const uint32_t* wp = reinterpret_cast<const uint32_t*>(&w);
  const uint64_t r2 = f32x2(rstd, rstd);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 a = widen2(hp[e], T()), b = widen2(wp[e], T());
    const float2 f = split_f32x2(mul_f32x2(mul_f32x2(f32x2(a.x, a.y), r2), f32x2(b.x, b.y)));
    y[2 * e] = f.x;
    y[2 * e + 1] = f.y;
  }
}

// ------------------------------------------------------------------ residual + RMSNorm + FP8

struct NormArgs {
  const uint16_t* x;
  const uint16_t* residual;  // null: no addition
  const uint16_t* weight;
  uint16_t* sum_out;
  uint8_t* q;
  float* scale;
  int64_t T, H, ldx, ldr, ldo;
  float eps;
  int group;      // 128, or 0 for one scale per row
  int w_early;    // the weight may be read before the preceding kernel has finished
};

// CTAs walk the rows (row, row + grid, ...), VPT 16-byte vectors of a row per thread, the row's sum
// held in registers. A row's loads, its two reductions and its stores follow each other, so the
// next row's loads are issued before the current one is reduced: with a CTA per row and no
// lookahead, 8192 rows of 3584 bf16 took 40.4 us.
// Resident CTAs of 512 threads an SM, by registers (smaller CTAs in proportion).
constexpr int norm_ctas(int vpt) { return vpt <= 2 ? 2 : 1; }

template <typename T, int VPT>
__global__ void __launch_bounds__(512, norm_ctas(VPT)) add_rmsnorm_row_kernel(const NormArgs a) {
  constexpr bool kAhead = VPT <= 4;  // eight vectors and the next eight do not fit the registers
  __shared__ float sh_sum[2][32];
  __shared__ uint32_t sh_max[2][32];
  const int tid = threadIdx.x, nt = blockDim.x;
  const int nvec = static_cast<int>(a.H / 8);
  const int groups = (nvec + kGroupVecs - 1) / kGroupVecs;
  const uint4* w = reinterpret_cast<const uint4*>(a.weight);
  uint4 g[VPT], x[VPT], r[VPT];
  if (!a.w_early) pdl_begin();
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int j = tid + nt * i;
    g[i] = j < nvec ? w[j] : make_uint4(0, 0, 0, 0);
  }
  auto load = [&](int64_t row) {
    const uint4* xr = reinterpret_cast<const uint4*>(a.x + row * a.ldx);
    const uint4* rr = reinterpret_cast<const uint4*>(a.residual + row * a.ldr);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int j = tid + nt * i;
      x[i] = j < nvec ? xr[j] : make_uint4(0, 0, 0, 0);
      if (a.residual != nullptr) r[i] = j < nvec ? rr[j] : make_uint4(0, 0, 0, 0);
    }
  };
  // x and the residual (and the outputs) may belong to the preceding kernel on the stream.
  if (a.w_early) pdl_begin();
  if (kAhead) load(blockIdx.x);
  int phase = 0;
  for (int64_t row = blockIdx.x; row < a.T; row += gridDim.x, phase ^= 1) {
    if (!kAhead) load(row);
    uint4 v[VPT];
    if (a.residual != nullptr) {
      uint4* sr = reinterpret_cast<uint4*>(a.sum_out + row * a.ldo);
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        float fx[8], fr[8];
        widen8<T>(x[i], fx);
        widen8<T>(r[i], fr);
        uint32_t* o = reinterpret_cast<uint32_t*>(&v[i]);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          o[e] = narrow2(fx[2 * e] + fr[2 * e], fx[2 * e + 1] + fr[2 * e + 1], T());
        if (tid + nt * i < nvec) sr[tid + nt * i] = v[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < VPT; ++i) v[i] = x[i];
    }
    if (kAhead && row + gridDim.x < a.T) load(row + gridDim.x);
    float sumsq = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      float f[8];
      widen8<T>(v[i], f);
#pragma unroll
      for (int e = 0; e < 8; ++e) sumsq = fmaf(f[e], f[e], sumsq);
    }
    const float rstd = rstd_f(block_sum_f(sumsq, sh_sum[phase]), a.H, a.eps);
    uint2* qr = reinterpret_cast<uint2*>(a.q + row * a.H);
    // 0 * rstd may be NaN past the row: those lanes take no part in the maxima.
    if (a.group != 0) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int j = tid + nt * i;
        float y[8];
        norm8<T>(v[i], g[i], rstd, y);
        const float s = scale_of_bits(half_warp_max(j < nvec ? max_bits8(y) : 0u));
        if (j < nvec) {
          if (j % kGroupVecs == 0) a.scale[row * groups + j / kGroupVecs] = s;
          qr[j] = codes8<false>(y, s);
        }
      }
    } else {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        float y[8];
        norm8<T>(v[i], g[i], rstd, y);
        if (tid + nt * i < nvec) m = max(m, max_bits8(y));
      }
      const float s = scale_of_bits(block_max_bits(m, sh_max[phase]));
      if (tid == 0) a.scale[row] = s;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        float y[8];
        norm8<T>(v[i], g[i], rstd, y);  // the same operations: the same bits
        if (tid + nt * i < nvec) qr[tid + nt * i] = codes8<false>(y, s);
      }
    }
  }
}

// Rows that are not 16-byte vectors, up to 8192 columns: a CTA per row, a warp per 128-column
// group (GP groups a warp), lane l of it columns l, l + 32, l + 64, l + 96, in registers.
template <typename T, int GP>
__global__ void __launch_bounds__(512) add_rmsnorm_group_kernel(const NormArgs a) {
  __shared__ float sh_sum[32];
  __shared__ uint32_t sh_max[32];
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  const int H = static_cast<int>(a.H), groups = (H + kGroup - 1) / kGroup;
  const T* w = reinterpret_cast<const T*>(a.weight);
  const T* xr = reinterpret_cast<const T*>(a.x) + row * a.ldx;
  const T* rr = reinterpret_cast<const T*>(a.residual) + row * a.ldr;
  T* sr = reinterpret_cast<T*>(a.sum_out) + row * a.ldo;
  auto column = [&](int p, int j) { return (warp + nw * p) * kGroup + lane + 32 * j; };
  float g[GP][4], y[GP][4];
  pdl_begin();
#pragma unroll
  for (int p = 0; p < GP; ++p)
#pragma unroll
    for (int j = 0; j < 4; ++j) g[p][j] = column(p, j) < H ? widen(w[column(p, j)]) : 0.f;
#pragma unroll
  for (int p = 0; p < GP; ++p)
#pragma unroll
    for (int j = 0; j < 4; ++j) y[p][j] = column(p, j) < H ? widen(xr[column(p, j)]) : 0.f;
  if (a.residual != nullptr) {
    float r[GP][4];
#pragma unroll
    for (int p = 0; p < GP; ++p)
#pragma unroll
      for (int j = 0; j < 4; ++j) r[p][j] = column(p, j) < H ? widen(rr[column(p, j)]) : 0.f;
#pragma unroll
    for (int p = 0; p < GP; ++p)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        T t;
        narrow(y[p][j] + r[p][j], &t);
        if (column(p, j) < H) sr[column(p, j)] = t;
        y[p][j] = widen(t);
      }
  }
  float sumsq = 0.f;
#pragma unroll
  for (int p = 0; p < GP; ++p)
#pragma unroll
    for (int j = 0; j < 4; ++j) sumsq = fmaf(y[p][j], y[p][j], sumsq);
  const float rstd = rstd_f(block_sum_f(sumsq, sh_sum), a.H, a.eps);
  uint32_t m[GP], all = 0;
#pragma unroll
  for (int p = 0; p < GP; ++p) {
    m[p] = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      y[p][j] = y[p][j] * rstd * g[p][j];
      if (column(p, j) < H) m[p] = max(m[p], abs_bits(y[p][j]));
    }
    all = max(all, m[p]);
  }
  float s = 0.f;
  if (a.group == 0) {
    s = scale_of_bits(block_max_bits(all, sh_max));
    if (threadIdx.x == 0) a.scale[row] = s;
  }
  uint8_t* qr = a.q + row * a.H;
#pragma unroll
  for (int p = 0; p < GP; ++p) {
    if (a.group != 0) {
      s = scale_of_bits(warp_max_bits(m[p]));
      if (lane == 0 && warp + nw * p < groups) a.scale[row * groups + warp + nw * p] = s;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (column(p, j) < H) qr[column(p, j)] = code1<false>(y[p][j], s);
  }
}

// Any H and alignment: one CTA of 512 threads per row, four sweeps over it (all but the first
// hit L2). A warp takes one 128-column group at a time.
template <typename T>
__global__ void __launch_bounds__(512) add_rmsnorm_any_kernel(const NormArgs a) {
  __shared__ float sh_sum[32];
  __shared__ uint32_t sh_max[32];
  const int64_t row = blockIdx.x;
  const T* w = reinterpret_cast<const T*>(a.weight);
  const T* xr = reinterpret_cast<const T*>(a.x) + row * a.ldx;
  const T* rr = reinterpret_cast<const T*>(a.residual) + row * a.ldr;
  T* sr = reinterpret_cast<T*>(a.sum_out) + row * a.ldo;
  pdl_begin();
  float sumsq = 0.f;
  for (int64_t c = threadIdx.x; c < a.H; c += blockDim.x) {
    float f = widen(xr[c]);
    if (a.residual != nullptr) {
      T t;
      narrow(f + widen(rr[c]), &t);
      sr[c] = t;
      f = widen(t);
    }
    sumsq = fmaf(f, f, sumsq);
  }
  const float rstd = rstd_f(block_sum_f(sumsq, sh_sum), a.H, a.eps);
  __syncthreads();  // the sums written above are read back by other threads below
  const T* hr = a.residual != nullptr ? sr : xr;
  auto y_of = [&](int64_t c) { return widen(hr[c]) * rstd * widen(w[c]); };
  uint8_t* qr = a.q + row * a.H;
  auto put = [&](int64_t c, float s) { qr[c] = code1<false>(y_of(c), s); };
  if (a.group != 0) {
    const int lane = threadIdx.x & 31;
    const int64_t groups = (a.H + kGroup - 1) / kGroup;
    for (int64_t g = threadIdx.x >> 5; g < groups; g += blockDim.x >> 5) {
      const int64_t c1 = min(a.H, (g + 1) * kGroup);
      uint32_t m = 0;
      for (int64_t c = g * kGroup + lane; c < c1; c += 32) m = max(m, abs_bits(y_of(c)));
      const float s = scale_of_bits(warp_max_bits(m));
      if (lane == 0) a.scale[row * groups + g] = s;
      for (int64_t c = g * kGroup + lane; c < c1; c += 32) put(c, s);
    }
  } else {
    uint32_t m = 0;
    for (int64_t c = threadIdx.x; c < a.H; c += blockDim.x) m = max(m, abs_bits(y_of(c)));
    const float s = scale_of_bits(block_max_bits(m, sh_max));
    if (threadIdx.x == 0) a.scale[row] = s;
    for (int64_t c = threadIdx.x; c < a.H; c += blockDim.x) put(c, s);
  }
}

// ------------------------------------------------------------- elementwise sources + groups

// What a group's value is made of. Load reads the vectors of 8 columns, value turns them to y.
template <typename T>
struct SiluSource {
  static constexpr bool kExact = false;
  static __device__ __forceinline__ float one(const T* row, int64_t c, int64_t C) {
    const float g = widen(row[c]), u = widen(row[C + c]);
    return split_f32x2(silu_mul2(make_float2(g, g), make_float2(u, u))).x;
  }
  struct Raw {
    uint4 g, u;
  };
  static __device__ __forceinline__ Raw load(const T* row, int64_t j, int64_t C) {
    return Raw{ld_stream_v4(row + 8 * j), ld_stream_v4(row + C + 8 * j)};
  }
  // y, and the bits of its largest magnitude.
  static __device__ __forceinline__ uint32_t value(const Raw& r, float (&y)[8]) {
    const uint32_t* g = reinterpret_cast<const uint32_t*>(&r.g);
    const uint32_t* u = reinterpret_cast<const uint32_t*>(&r.u);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = split_f32x2(silu_mul2(widen2(g[e], T()), widen2(u[e], T())));
      y[2 * e] = f.x;
      y[2 * e + 1] = f.y;
    }
    return max_bits8(y);
  }
};
template <typename T>
struct CopySource {
  static constexpr bool kExact = true;
  static __device__ __forceinline__ float one(const T* row, int64_t c, int64_t) {
    return widen(row[c]);
  }
  struct Raw {
    uint4 x;
  };
  static __device__ __forceinline__ Raw load(const T* row, int64_t j, int64_t) {
    return Raw{ld_stream_v4(row + 8 * j)};
  }
  // The maximum of the 16-bit patterns, two at a time: the same order as the widened values'.
  static __device__ __forceinline__ uint32_t value(const Raw& r, float (&y)[8]) {
    widen8<T>(r.x, y);
    constexpr uint32_t kAbs = 0x7FFF7FFFu;
    const uint32_t m = __vmaxu2(__vmaxu2(r.x.x & kAbs, r.x.y & kAbs),
                                __vmaxu2(r.x.z & kAbs, r.x.w & kAbs));
    const uint32_t top = max(m & 0xFFFFu, m >> 16);
    return __float_as_uint(widen2(top, T()).x);
  }
};

struct GroupArgs {
  const uint16_t* x;
  uint8_t* q;
  float* scale;
  int64_t R, C, ldx;
};

// Scale per group, aligned rows. Row r's C / 8 vectors are padded to whole groups of 16; the
// padded vectors of all rows, in order, are dealt to half warps, U of them a thread, so that U
// (or 2 U) loads are in flight before the first one is used.
template <typename T, template <typename> class Source, int U>
__global__ void __launch_bounds__(256) quant_groups_kernel(const GroupArgs a, const FastDiv per_row) {
  const int nvec = static_cast<int>(a.C / 8);
  const int groups = static_cast<int>(per_row.d) / kGroupVecs;
  const uint32_t total = static_cast<uint32_t>(a.R) * per_row.d;
  const T* x = reinterpret_cast<const T*>(a.x);
  pdl_begin();
  const uint32_t base = blockIdx.x * (256 * U) + threadIdx.x;
  typename Source<T>::Raw raw[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const uint32_t s = base + 256 * i;
    const uint32_t row = div_by(s, per_row);
    const int vec = static_cast<int>(s - row * per_row.d);
    if (s < total && vec < nvec)
      raw[i] = Source<T>::load(x + static_cast<int64_t>(row) * a.ldx, vec, a.C);
  }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const uint32_t s = base + 256 * i;
    const uint32_t row = div_by(s, per_row);
    const int vec = static_cast<int>(s - row * per_row.d);
    const bool ok = s < total && vec < nvec;
    float y[8];
    const uint32_t m = Source<T>::value(raw[i], y);
    const float sc = scale_of_bits(half_warp_max(ok ? m : 0u));
    if (ok) {
      if (vec % kGroupVecs == 0) a.scale[static_cast<int64_t>(row) * groups + vec / kGroupVecs] = sc;
      reinterpret_cast<uint2*>(a.q + row * a.C)[vec] = codes8<Source<T>::kExact>(y, sc);
    }
  }
}

// Scale per group, any C and alignment: a warp per group, columns lane, lane + 32, ...
template <typename T, template <typename> class Source>
__global__ void __launch_bounds__(256) quant_groups_any_kernel(const GroupArgs a,
                                                              const FastDiv per_row) {
  const uint32_t groups = per_row.d;
  const uint32_t id = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  pdl_begin();
  if (id >= static_cast<uint32_t>(a.R) * groups) return;
  const int64_t row = div_by(id, per_row), g = id - static_cast<uint32_t>(row) * groups;
  const T* xr = reinterpret_cast<const T*>(a.x) + row * a.ldx;
  float y[4];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t c = g * kGroup + lane + 32 * i;
    y[i] = c < a.C ? Source<T>::one(xr, c, a.C) : 0.f;
    m = max(m, abs_bits(y[i]));
  }
  const float s = scale_of_bits(warp_max_bits(m));
  if (lane == 0) a.scale[id] = s;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t c = g * kGroup + lane + 32 * i;
    if (c < a.C) a.q[row * a.C + c] = code1<Source<T>::kExact>(y[i], s);
  }
}

// One scale per row, aligned rows of at most 1024 * VPT vectors: a CTA walks the rows, y in
// registers, the next row's loads issued before the current row's maximum is reduced.
template <typename T, template <typename> class Source, int VPT>
__global__ void __launch_bounds__(1024) quant_row_kernel(const GroupArgs a) {
  __shared__ uint32_t sh_max[2][32];
  const int nvec = static_cast<int>(a.C / 8), tid = threadIdx.x, nt = blockDim.x;
  pdl_begin();
  typename Source<T>::Raw raw[VPT];
  auto load = [&](int64_t row) {
    const T* xr = reinterpret_cast<const T*>(a.x) + row * a.ldx;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if (tid + nt * i < nvec) raw[i] = Source<T>::load(xr, tid + nt * i, a.C);
  };
  load(blockIdx.x);
  int phase = 0;
  for (int64_t row = blockIdx.x; row < a.R; row += gridDim.x, phase ^= 1) {
    float y[VPT][8];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if (tid + nt * i < nvec) m = max(m, Source<T>::value(raw[i], y[i]));
    if (row + gridDim.x < a.R) load(row + gridDim.x);
    const float s = scale_of_bits(block_max_bits(m, sh_max[phase]));
    if (tid == 0) a.scale[row] = s;
    uint2* qr = reinterpret_cast<uint2*>(a.q + row * a.C);
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if (tid + nt * i < nvec) qr[tid + nt * i] = codes8<Source<T>::kExact>(y[i], s);
  }
}

// One scale per row, any C and alignment: two sweeps (the second hits L2).
template <typename T, template <typename> class Source>
__global__ void __launch_bounds__(1024) quant_row_any_kernel(const GroupArgs a) {
  __shared__ uint32_t sh_max[32];
  const int64_t row = blockIdx.x;
  const T* xr = reinterpret_cast<const T*>(a.x) + row * a.ldx;
  pdl_begin();
  uint32_t m = 0;
  for (int64_t c = threadIdx.x; c < a.C; c += blockDim.x)
    m = max(m, abs_bits(Source<T>::one(xr, c, a.C)));
  const float s = scale_of_bits(block_max_bits(m, sh_max));
  if (threadIdx.x == 0) a.scale[row] = s;
  for (int64_t c = threadIdx.x; c < a.C; c += blockDim.x)
    a.q[row * a.C + c] = code1<Source<T>::kExact>(Source<T>::one(xr, c, a.C), s);
}

// ----------------------------------------------------------------------------- host side

template <typename... Args>
int launch(void (*kernel)(Args...), int64_t grid, int threads, cudaStream_t stream, Args... a) {
  if (grid > 0x7fffffffLL) return TF_ERR_TOO_LARGE;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a...);
  if (e != cudaSuccess) return cuda_failed(e);
  return TF_OK;
}

bool dtype_ok(int32_t dtype) { return dtype == TF_DTYPE_FP16 || dtype == TF_DTYPE_BF16; }

template <typename T>
int launch_norm(const NormArgs& a, cudaStream_t stream) {
  const bool vec = a.H % 8 == 0 && a.H <= 512 * 8 * 8 && aligned16(a.x) && a.ldx % 8 == 0 &&
                   aligned16(a.weight) && (reinterpret_cast<uintptr_t>(a.q) & 7u) == 0 &&
                   (a.residual == nullptr || (aligned16(a.residual) && a.ldr % 8 == 0 &&
                                              aligned16(a.sum_out) && a.ldo % 8 == 0));
  if (!vec && a.H <= 64 * kGroup) {
    const int groups = static_cast<int>(cdiv(a.H, kGroup));
    const int gp = groups <= 16 ? 1 : groups <= 32 ? 2 : 4;
    const int threads = 32 * static_cast<int>(cdiv(groups, gp));
    switch (gp) {
      case 1: return launch(add_rmsnorm_group_kernel<T, 1>, a.T, threads, stream, a);
      case 2: return launch(add_rmsnorm_group_kernel<T, 2>, a.T, threads, stream, a);
      default: return launch(add_rmsnorm_group_kernel<T, 4>, a.T, threads, stream, a);
    }
  }
  if (!vec) return launch(add_rmsnorm_any_kernel<T>, a.T, 512, stream, a);
  const int64_t nvec = a.H / 8;
  // Two vectors a thread from 64 of them on: half the threads a row, so twice the rows in flight
  // (3584 columns, 8192 rows: 34.0 us, 39.0 with one vector).
  const int vpt = nvec <= 64 ? 1 : nvec <= 1024 ? 2 : nvec <= 2048 ? 4 : 8;
  const int threads = static_cast<int>(cdiv(cdiv(nvec, vpt), 32) * 32);
  const int64_t grid = std::min<int64_t>(a.T, 148 * (512 * norm_ctas(vpt) / threads));
  switch (vpt) {
    case 1: return launch(add_rmsnorm_row_kernel<T, 1>, grid, threads, stream, a);
    case 2: return launch(add_rmsnorm_row_kernel<T, 2>, grid, threads, stream, a);
    case 4: return launch(add_rmsnorm_row_kernel<T, 4>, grid, threads, stream, a);
    default: return launch(add_rmsnorm_row_kernel<T, 8>, grid, threads, stream, a);
  }
}

bool vec_rows(const GroupArgs& a) {
  return a.C % 8 == 0 && aligned16(a.x) && a.ldx % 8 == 0 &&
         (reinterpret_cast<uintptr_t>(a.q) & 7u) == 0;
}

template <typename T, template <typename> class Source>
int launch_groups(const GroupArgs& a, cudaStream_t stream) {
  constexpr int U = 4;
  const bool vec = vec_rows(a);
  const int64_t groups = cdiv(a.C, kGroup);
  const int64_t per_row = vec ? groups * kGroupVecs : groups;  // slots, of vectors or of groups
  if (per_row >= (int64_t(1) << 30)) return TF_ERR_TOO_LARGE;
  const FastDiv div = fast_div(static_cast<uint32_t>(per_row));
  // Slots are 31-bit numbers: more rows than that take several launches.
  const int64_t most = ((int64_t(1) << 31) - 256 * U - 1) / per_row;
  for (int64_t r0 = 0; r0 < a.R; r0 += most) {
    GroupArgs part = a;
    part.R = std::min(most, a.R - r0);
    part.x = a.x + r0 * a.ldx;
    part.q = a.q + r0 * a.C;
    part.scale = a.scale + r0 * groups;
    const int64_t slots = part.R * per_row;
    const int st = vec ? launch(quant_groups_kernel<T, Source, U>, cdiv(slots, 256 * U), 256,
                                stream, part, div)
                       : launch(quant_groups_any_kernel<T, Source>, cdiv(slots, 8), 256, stream,
                                part, div);
    if (st != TF_OK) return st;
  }
  return TF_OK;
}

template <typename T, template <typename> class Source>
int launch_rows(const GroupArgs& a, cudaStream_t stream) {
  const int64_t nvec = a.C / 8;
  if (!vec_rows(a) || nvec > 4096)
    return launch(quant_row_any_kernel<T, Source>, a.R, 1024, stream, a);
  const int vpt = static_cast<int>(cdiv(nvec, 1024));
  const int threads = static_cast<int>(cdiv(cdiv(nvec, vpt), 32) * 32);
  const int64_t grid = std::min<int64_t>(a.R, 148 * (1024 / threads));
  switch (vpt) {
    case 1: return launch(quant_row_kernel<T, Source, 1>, grid, threads, stream, a);
    case 2: return launch(quant_row_kernel<T, Source, 2>, grid, threads, stream, a);
    case 3: return launch(quant_row_kernel<T, Source, 3>, grid, threads, stream, a);
    default: return launch(quant_row_kernel<T, Source, 4>, grid, threads, stream, a);
  }
}

}  // namespace
}  // namespace tfb

using namespace tfb;

extern "C" int tf_add_rmsnorm_fp8_quant(const uint16_t* x, int64_t T, int64_t H, int64_t ldx,
                                        const uint16_t* residual, int64_t ldr,
                                        const uint16_t* weight, float eps, int32_t dtype,
                                        int32_t group_size, uint8_t* q, float* scale_out,
                                        uint16_t* residual_out, int64_t ldo, void* stream) {
  if (T < 0 || H < 1 || !dtype_ok(dtype) || (group_size != 0 && group_size != kGroup))
    return TF_ERR_INVALID_ARG;
  if (T == 0) return TF_OK;
  if (!x || !weight || !q || !scale_out || ldx < H || (residual == nullptr) != (residual_out == nullptr))
    return TF_ERR_INVALID_ARG;
  if (residual && (ldr < H || ldo < H)) return TF_ERR_INVALID_ARG;
  const NormArgs a{x, residual, weight, residual_out, q, scale_out, T, H, ldx,
                   residual ? ldr : 0, residual ? ldo : 0, eps, group_size,
                   (launch_flags() & TF_LAUNCH_PDL) ? 1 : 0};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == TF_DTYPE_FP16 ? launch_norm<__half>(a, s) : launch_norm<__nv_bfloat16>(a, s);
}

extern "C" int tf_silu_mul_fp8_quant(const uint16_t* gate_up, int64_t M, int64_t I, int64_t ld,
                                     int32_t dtype, int32_t group_size, uint8_t* q,
                                     float* scale_out, void* stream) {
  if (M < 0 || I < 1 || !dtype_ok(dtype) || (group_size != 0 && group_size != kGroup))
    return TF_ERR_INVALID_ARG;
  if (M == 0) return TF_OK;
  if (!gate_up || !q || !scale_out || ld < 2 * I) return TF_ERR_INVALID_ARG;
  const GroupArgs a{gate_up, q, scale_out, M, I, ld};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (group_size == 0)
    return dtype == TF_DTYPE_FP16 ? launch_rows<__half, SiluSource>(a, s)
                                  : launch_rows<__nv_bfloat16, SiluSource>(a, s);
  return dtype == TF_DTYPE_FP16 ? launch_groups<__half, SiluSource>(a, s)
                                : launch_groups<__nv_bfloat16, SiluSource>(a, s);
}

extern "C" int tf_e4m3_quant_groups(const uint16_t* x, int64_t R, int64_t C, int64_t ldx,
                                    int32_t dtype, uint8_t* q, float* scale_out, void* stream) {
  if (R < 0 || C < 1 || !dtype_ok(dtype)) return TF_ERR_INVALID_ARG;
  if (R == 0) return TF_OK;
  if (!x || !q || !scale_out || ldx < C) return TF_ERR_INVALID_ARG;
  const GroupArgs a{x, q, scale_out, R, C, ldx};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == TF_DTYPE_FP16 ? launch_groups<__half, CopySource>(a, s)
                                : launch_groups<__nv_bfloat16, CopySource>(a, s);
}
