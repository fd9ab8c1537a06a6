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
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, abs_bits(y[i]));
  return m;
}

__device__ __forceinline__ float rstd_f(float sumsq, int64_t H, float eps) {
  return __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(sumsq, static_cast<float>(H)), eps)));
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
  int group;  // 128, or 0 for one scale per row
};

// One CTA per row, VPT 16-byte vectors per thread, the row's sum held in registers.
template <typename T, int VPT>
__global__ void __launch_bounds__(512) add_rmsnorm_row_kernel(const NormArgs a) {
  __shared__ float sh_sum[32];
  __shared__ uint32_t sh_max[32];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, nt = blockDim.x;
  const int nvec = static_cast<int>(a.H / 8);
  const uint4* w = reinterpret_cast<const uint4*>(a.weight);
  const uint4* xr = reinterpret_cast<const uint4*>(a.x + row * a.ldx);
  const uint4* rr = reinterpret_cast<const uint4*>(a.residual + row * a.ldr);
  uint4* sr = reinterpret_cast<uint4*>(a.sum_out + row * a.ldo);
  uint4 g[VPT], v[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int j = tid + nt * i;
    g[i] = j < nvec ? __ldg(w + j) : make_uint4(0, 0, 0, 0);
  }
  // x and the residual (and the outputs) may belong to the preceding kernel on the stream.
  pdl_wait();
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int j = tid + nt * i;
    v[i] = j < nvec ? xr[j] : make_uint4(0, 0, 0, 0);
  }
  if (a.residual != nullptr) {
    uint4 r[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int j = tid + nt * i;
      r[i] = j < nvec ? rr[j] : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int j = tid + nt * i;
      float fx[8], fr[8];
      widen8<T>(v[i], fx);
      widen8<T>(r[i], fr);
      uint32_t* o = reinterpret_cast<uint32_t*>(&v[i]);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        o[e] = narrow2(fx[2 * e] + fr[2 * e], fx[2 * e + 1] + fr[2 * e + 1], T());
      if (j < nvec) sr[j] = v[i];
    }
  }
  float sumsq = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    float f[8];
    widen8<T>(v[i], f);
#pragma unroll
    for (int e = 0; e < 8; ++e) sumsq = fmaf(f[e], f[e], sumsq);
  }
  const float rstd = rstd_f(block_sum_f(sumsq, sh_sum), a.H, a.eps);
  float y[VPT][8];
  uint32_t m[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    float gw[8];
    widen8<T>(v[i], y[i]);
    widen8<T>(g[i], gw);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[i][e] = y[i][e] * rstd * gw[e];
    m[i] = tid + nt * i < nvec ? max_bits8(y[i]) : 0u;  // 0 * rstd may be NaN past the row
  }
  uint2* qr = reinterpret_cast<uint2*>(a.q + row * a.H);
  if (a.group != 0) {
    const int groups = (nvec + kGroupVecs - 1) / kGroupVecs;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int j = tid + nt * i;
      const float s = scale_of_bits(half_warp_max(m[i]));
      if (j < nvec) {
        if (j % kGroupVecs == 0) a.scale[row * groups + j / kGroupVecs] = s;
        qr[j] = codes8<false>(y[i], group_div(s));
      }
    }
  } else {
    uint32_t mm = 0;
#pragma unroll
    for (int i = 0; i < VPT; ++i) mm = max(mm, m[i]);
    const float s = scale_of_bits(block_max_bits(mm, sh_max));
    if (tid == 0) a.scale[row] = s;
    const GroupDiv d = group_div(s);
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if (tid + nt * i < nvec) qr[tid + nt * i] = codes8<false>(y[i], d);
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
  pdl_wait();
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
  auto put = [&](int64_t c, const GroupDiv& d) {
    qr[c] = static_cast<uint8_t>(cvt_e4m3x2(divide<false>(y_of(c), d), 0.f) & 0xFFu);
  };
  if (a.group != 0) {
    const int lane = threadIdx.x & 31;
    const int64_t groups = (a.H + kGroup - 1) / kGroup;
    for (int64_t g = threadIdx.x >> 5; g < groups; g += blockDim.x >> 5) {
      const int64_t c1 = min(a.H, (g + 1) * kGroup);
      uint32_t m = 0;
      for (int64_t c = g * kGroup + lane; c < c1; c += 32) m = max(m, abs_bits(y_of(c)));
      const float s = scale_of_bits(warp_max_bits(m));
      if (lane == 0) a.scale[row * groups + g] = s;
      const GroupDiv d = group_div(s);
      for (int64_t c = g * kGroup + lane; c < c1; c += 32) put(c, d);
    }
  } else {
    uint32_t m = 0;
    for (int64_t c = threadIdx.x; c < a.H; c += blockDim.x) m = max(m, abs_bits(y_of(c)));
    const float s = scale_of_bits(block_max_bits(m, sh_max));
    if (threadIdx.x == 0) a.scale[row] = s;
    const GroupDiv d = group_div(s);
    for (int64_t c = threadIdx.x; c < a.H; c += blockDim.x) put(c, d);
  }
}

// ------------------------------------------------------------- elementwise sources + groups

// What a group's value is made of. Load reads the vectors of 8 columns, value turns them to y.
template <typename T>
struct SiluSource {
  static constexpr bool kExact = false;
  static __device__ __forceinline__ float one(const T* row, int64_t c, int64_t C) {
    const float g = widen(row[c]);
    return __fdividef(g, 1.0f + __expf(-g)) * widen(row[C + c]);
  }
  struct Raw {
    uint4 g, u;
  };
  static __device__ __forceinline__ Raw load(const T* row, int64_t j, int64_t C) {
    return Raw{ldg_stream_v4(row + 8 * j), ldg_stream_v4(row + C + 8 * j)};
  }
  static __device__ __forceinline__ void value(const Raw& r, float (&y)[8]) {
    float g[8], u[8];
    widen8<T>(r.g, g);
    widen8<T>(r.u, u);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = __fdividef(g[e], 1.0f + __expf(-g[e])) * u[e];
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
    return Raw{ldg_stream_v4(row + 8 * j)};
  }
  static __device__ __forceinline__ void value(const Raw& r, float (&y)[8]) {
    widen8<T>(r.x, y);
  }
};

struct GroupArgs {
  const uint16_t* x;
  uint8_t* q;
  float* scale;
  int64_t R, C, ldx;
};

// Scale per group, aligned rows. Row r's C / 8 vectors are padded to whole groups of 16; the
// padded vectors of all rows, in order, are dealt to half warps, U of them a thread.
template <typename T, template <typename> class Source, int U>
__global__ void __launch_bounds__(256) quant_groups_kernel(const GroupArgs a) {
  const int64_t nvec = a.C / 8;
  const int64_t groups = (nvec + kGroupVecs - 1) / kGroupVecs;
  const int64_t total = a.R * groups * kGroupVecs;
  const T* x = reinterpret_cast<const T*>(a.x);
  pdl_wait();
  const int64_t base = static_cast<int64_t>(blockIdx.x) * (256 * U) + threadIdx.x;
  typename Source<T>::Raw raw[U];
  int64_t row[U], vec[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int64_t s = base + 256 * i;
    row[i] = s / (groups * kGroupVecs);
    vec[i] = s - row[i] * (groups * kGroupVecs);
    if (s >= total) vec[i] = nvec;
    if (vec[i] < nvec) raw[i] = Source<T>::load(x + row[i] * a.ldx, vec[i], a.C);
  }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    float y[8];
    uint32_t m = 0;
    if (vec[i] < nvec) {
      Source<T>::value(raw[i], y);
      m = max_bits8(y);
    }
    const float s = scale_of_bits(half_warp_max(m));
    if (vec[i] < nvec) {
      if (vec[i] % kGroupVecs == 0) a.scale[row[i] * groups + vec[i] / kGroupVecs] = s;
      reinterpret_cast<uint2*>(a.q + row[i] * a.C)[vec[i]] =
          codes8<Source<T>::kExact>(y, group_div(s));
    }
  }
}

// Scale per group, any C and alignment: a warp per group, columns lane, lane + 32, ...
template <typename T, template <typename> class Source>
__global__ void __launch_bounds__(256) quant_groups_any_kernel(const GroupArgs a) {
  const int64_t groups = (a.C + kGroup - 1) / kGroup;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  pdl_wait();
  if (id >= a.R * groups) return;
  const int64_t row = id / groups, g = id - row * groups;
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
  const GroupDiv d = group_div(s);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t c = g * kGroup + lane + 32 * i;
    if (c < a.C)
      a.q[row * a.C + c] =
          static_cast<uint8_t>(cvt_e4m3x2(divide<Source<T>::kExact>(y[i], d), 0.f) & 0xFFu);
  }
}

// One scale per row, aligned rows of at most 1024 * VPT vectors: a CTA per row, y in registers.
template <typename T, template <typename> class Source, int VPT>
__global__ void __launch_bounds__(1024) quant_row_kernel(const GroupArgs a) {
  __shared__ uint32_t sh_max[32];
  const int64_t row = blockIdx.x;
  const int nvec = static_cast<int>(a.C / 8), tid = threadIdx.x, nt = blockDim.x;
  const T* xr = reinterpret_cast<const T*>(a.x) + row * a.ldx;
  pdl_wait();
  typename Source<T>::Raw raw[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i)
    if (tid + nt * i < nvec) raw[i] = Source<T>::load(xr, tid + nt * i, a.C);
  float y[VPT][8];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < VPT; ++i)
    if (tid + nt * i < nvec) {
      Source<T>::value(raw[i], y[i]);
      m = max(m, max_bits8(y[i]));
    }
  const float s = scale_of_bits(block_max_bits(m, sh_max));
  if (tid == 0) a.scale[row] = s;
  const GroupDiv d = group_div(s);
  uint2* qr = reinterpret_cast<uint2*>(a.q + row * a.C);
#pragma unroll
  for (int i = 0; i < VPT; ++i)
    if (tid + nt * i < nvec) qr[tid + nt * i] = codes8<Source<T>::kExact>(y[i], d);
}

// One scale per row, any C and alignment: two sweeps (the second hits L2).
template <typename T, template <typename> class Source>
__global__ void __launch_bounds__(1024) quant_row_any_kernel(const GroupArgs a) {
  __shared__ uint32_t sh_max[32];
  const int64_t row = blockIdx.x;
  const T* xr = reinterpret_cast<const T*>(a.x) + row * a.ldx;
  pdl_wait();
  uint32_t m = 0;
  for (int64_t c = threadIdx.x; c < a.C; c += blockDim.x)
    m = max(m, abs_bits(Source<T>::one(xr, c, a.C)));
  const float s = scale_of_bits(block_max_bits(m, sh_max));
  if (threadIdx.x == 0) a.scale[row] = s;
  const GroupDiv d = group_div(s);
  for (int64_t c = threadIdx.x; c < a.C; c += blockDim.x)
    a.q[row * a.C + c] = static_cast<uint8_t>(
        cvt_e4m3x2(divide<Source<T>::kExact>(Source<T>::one(xr, c, a.C), d), 0.f) & 0xFFu);
}

// ----------------------------------------------------------------------------- host side

template <typename Args>
int launch(void (*kernel)(Args), int64_t grid, int threads, cudaStream_t stream, const Args& a) {
  if (grid > 0x7fffffffLL) return TF_ERR_TOO_LARGE;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = (launch_flags() & TF_LAUNCH_PDL) ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
  if (e != cudaSuccess) {
    last_cuda_error() = static_cast<int>(e);
    return TF_ERR_CUDA;
  }
  return TF_OK;
}

bool dtype_ok(int32_t dtype) { return dtype == TF_DTYPE_FP16 || dtype == TF_DTYPE_BF16; }

template <typename T>
int launch_norm(const NormArgs& a, cudaStream_t stream) {
  const bool vec = a.H % 8 == 0 && a.H <= 512 * 8 * 8 && aligned16(a.x) && a.ldx % 8 == 0 &&
                   aligned16(a.weight) && (reinterpret_cast<uintptr_t>(a.q) & 7u) == 0 &&
                   (a.residual == nullptr || (aligned16(a.residual) && a.ldr % 8 == 0 &&
                                              aligned16(a.sum_out) && a.ldo % 8 == 0));
  if (!vec) return launch(add_rmsnorm_any_kernel<T>, a.T, 512, stream, a);
  const int64_t nvec = a.H / 8;
  const int vpt = nvec <= 512 ? 1 : nvec <= 1024 ? 2 : nvec <= 2048 ? 4 : 8;
  const int threads = static_cast<int>(cdiv(cdiv(nvec, vpt), 32) * 32);
  switch (vpt) {
    case 1: return launch(add_rmsnorm_row_kernel<T, 1>, a.T, threads, stream, a);
    case 2: return launch(add_rmsnorm_row_kernel<T, 2>, a.T, threads, stream, a);
    case 4: return launch(add_rmsnorm_row_kernel<T, 4>, a.T, threads, stream, a);
    default: return launch(add_rmsnorm_row_kernel<T, 8>, a.T, threads, stream, a);
  }
}

bool vec_rows(const GroupArgs& a) {
  return a.C % 8 == 0 && aligned16(a.x) && a.ldx % 8 == 0 &&
         (reinterpret_cast<uintptr_t>(a.q) & 7u) == 0;
}

template <typename T, template <typename> class Source>
int launch_groups(const GroupArgs& a, cudaStream_t stream) {
  const int64_t groups = cdiv(a.C, kGroup);
  if (!vec_rows(a))
    return launch(quant_groups_any_kernel<T, Source>, cdiv(a.R * groups, 8), 256, stream, a);
  constexpr int U = 4;
  return launch(quant_groups_kernel<T, Source, U>, cdiv(a.R * groups * kGroupVecs, 256 * U), 256,
                stream, a);
}

template <typename T, template <typename> class Source>
int launch_rows(const GroupArgs& a, cudaStream_t stream) {
  const int64_t nvec = a.C / 8;
  if (!vec_rows(a) || nvec > 4096)
    return launch(quant_row_any_kernel<T, Source>, a.R, 1024, stream, a);
  const int vpt = nvec <= 1024 ? 1 : nvec <= 2048 ? 2 : nvec <= 3072 ? 3 : 4;
  const int threads = static_cast<int>(cdiv(cdiv(nvec, vpt), 32) * 32);
  switch (vpt) {
    case 1: return launch(quant_row_kernel<T, Source, 1>, a.R, threads, stream, a);
    case 2: return launch(quant_row_kernel<T, Source, 2>, a.R, threads, stream, a);
    case 3: return launch(quant_row_kernel<T, Source, 3>, a.R, threads, stream, a);
    default: return launch(quant_row_kernel<T, Source, 4>, a.R, threads, stream, a);
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
                   residual ? ldr : 0, residual ? ldo : 0, eps, group_size};
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
