// Block-scaled FP8 linear on the sm_100a tensor cores: e4m3 x e4m3 tcgen05.mma with the scales of
// each 128-wide K block applied between blocks.
//
//   y[m, n] = sum_b sx[m, b] * sw[n / 128, b] * (sum_{k in b} xq[m, k] * wq[n, k])  (+ bias[n])
//
// The tensor core cannot hold a sum across blocks, because every (token, block) has a scale of
// its own. So each 128-wide block is one accumulation of four K = 32 MMAs into a TMEM buffer
// (the first overwrites it), and promotion warps read the buffer with tcgen05.ld and add it,
// times the scales, to the tile's running sum in their fp32 registers. A ring of TMEM buffers
// lets the tensor core fill the next block while one is promoted.
//
// Two forms, by which operand gives the accumulator's 128 lanes:
//   tokens as lanes (kSwap = false): tile of 128 tokens x 256 weight rows; a lane is a token, so
//     a block's scale is one number per thread and 128 columns, and promotion costs one packed
//     FMA per two values. Two warps per TMEM quadrant, 128 columns each. For M > 64.
//   weight rows as lanes (kSwap = true): tile of 128 weight rows x 16, 32 or 64 tokens, for few
//     tokens: no tensor-core rows are wasted on missing tokens, the weight stream sets the pace,
//     and the scale of a column (token) comes from shared memory. One warp per quadrant, two
//     CTAs per SM.
//
// Warps: 0 TMA producer, 1 TMEM allocation and MMA issue, then the promotion warps, then one
// that fetches the block's scales into a small ring. Persistent CTAs walk the tiles with the
// token tile fastest (the weight tile stays in L2); when there are fewer tiles than SMs, the
// CTAs of a cluster split K instead, and sum their tiles through distributed shared memory in
// rank order, so the result does not depend on timing and no workspace is needed. Every wait is
// bounded (2 s): on a time-out the kernel records an error code for tf_device_error, stops, lets
// its copies and MMAs finish, frees its TMEM and returns.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <mutex>

#include "tf_common.cuh"
#include "tf_fp8_act.cuh"
#include "tf_plan.h"
#include "tf_tcgen05.cuh"
#include "tf_w8a8.h"

namespace tfb {

__device__ int g_w8a8_error = 0;

namespace {

constexpr int kLanes = 128;  // accumulator lanes = rows of the A operand
constexpr int kBlockK = 128;  // K of a scale block = one 128-byte swizzle row of e4m3
constexpr unsigned long long kWaitLimitNs = 2000000000ull;

enum WaitSite : int {
  kErrProducer = 0x401,
  kErrMmaFull = 0x402,
  kErrMmaAcc = 0x403,
  kErrPromote = 0x404,
  kErrScale = 0x405,
  kErrDrain = 0x406,
};

template <bool kSwap, int kCols>
struct Cfg {
  static constexpr int kColGroups = kSwap ? 1 : 2;     // promotion warps per TMEM quadrant
  static constexpr int kColsPerThread = kCols / kColGroups;
  static constexpr int kPromoteWarps = 4 * kColGroups;
  static constexpr int kScaleWarp = 2 + kPromoteWarps;
  static constexpr int kThreads = 32 * (3 + kPromoteWarps);
  static constexpr int kCtasPerSm = kSwap ? 2 : 1;
  static constexpr int kABytes = kLanes * kBlockK;
  static constexpr int kBBytes = kCols * kBlockK;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kAccs = kSwap ? 4 : 2;          // TMEM buffers (and scale-ring entries)
  static constexpr int kTmemCols = kAccs * kCols;
  // Scales of a block: one per token of the tile, then the weight blocks' (2 x 128 rows).
  static constexpr int kTokens = kSwap ? kCols : kLanes;
  static constexpr int kScaleFloats = kTokens + 4;
  static constexpr int kBudget = (kSwap ? 112 : 226) * 1024;
  static constexpr int kTail = 1024 + kAccs * kScaleFloats * 4 + 512;  // alignment, ring, barriers
  static constexpr int kStages = std::min(8, (kBudget - kTail) / kStageBytes);
  static constexpr int kRingOff = kStages * kStageBytes;
  static constexpr int kBarOff = kRingOff + (kAccs * kScaleFloats * 4 + 15) / 16 * 16;
  // The cluster's exchange of partial tiles reuses the stages once the last block is done.
  static constexpr int kExchange = kLanes * kCols * 4;
  static_assert(kExchange <= kRingOff, "exchange buffer fits the stages");
  static constexpr int kSmem = 1024 + kBarOff + 512;
  static_assert(kTmemCols >= 32 && (kTmemCols & (kTmemCols - 1)) == 0 &&
                    kTmemCols * kCtasPerSm <= 512, "TMEM");
  static_assert((2 * kStages + 3 * kAccs) * 8 + 8 <= 512, "barriers");
};

struct TcArgs {
  W8A8Args a;
  int kb_total, tok_tiles, w_tiles, splits;
};

__device__ __noinline__ bool mbar_wait_slow(uint64_t* bar, uint32_t parity, int site) {
  const unsigned long long t0 = global_ns();
  while (true) {
    for (int i = 0; i < 128; ++i)
      if (mbar_try_wait(bar, parity)) return true;
    if (*reinterpret_cast<volatile int*>(&g_w8a8_error) != 0) return false;
    if (global_ns() - t0 > kWaitLimitNs) {
      atomicCAS(&g_w8a8_error, 0, site);
      return false;
    }
  }
}
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, int site) {
  if (mbar_try_wait(bar, parity)) return true;
  return mbar_wait_slow(bar, parity, site);
}

// D[tmem] (+)= A[smem] * B[smem]^T, e4m3 inputs, fp32 accumulate, K = 32, issued by one thread.
__device__ __forceinline__ void umma_e4m3(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                          uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile(
      "barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
          : "memory");
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t local, uint32_t rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote) : "memory");
  return v;
}

// Tile u of the walk: token tiles fastest.
struct Tile {
  int64_t m0, n0;
};
template <bool kSwap, int kCols>
__device__ __forceinline__ Tile tile_of(int u, const TcArgs& p) {
  const int tt = u % p.tok_tiles, wt = u / p.tok_tiles;
  return kSwap ? Tile{static_cast<int64_t>(tt) * kCols, static_cast<int64_t>(wt) * kLanes}
               : Tile{static_cast<int64_t>(tt) * kLanes, static_cast<int64_t>(wt) * kCols};
}

// Eight consecutive outputs of one token (tokens as lanes), bias added.
template <typename T>
__device__ __forceinline__ void store8(const W8A8Args& a, int64_t m, int64_t n, bool vec,
                                       const float (&v)[8]) {
  T* y = reinterpret_cast<T*>(a.y) + m * a.ldy + n;
  const T* bias = reinterpret_cast<const T*>(a.bias);
  if (vec && n + 8 <= a.N) {
    float b[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (bias != nullptr)
#pragma unroll
      for (int e = 0; e < 8; ++e) b[e] = widen(bias[n + e]);
    uint4 o;
    o.x = narrow2(v[0] + b[0], v[1] + b[1], T());
    o.y = narrow2(v[2] + b[2], v[3] + b[3], T());
    o.z = narrow2(v[4] + b[4], v[5] + b[5], T());
    o.w = narrow2(v[6] + b[6], v[7] + b[7], T());
    *reinterpret_cast<uint4*>(y) = o;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (n + e < a.N) narrow(v[e] + (bias != nullptr ? widen(bias[n + e]) : 0.f), y + e);
  }
}

template <bool kSwap, int kCols, typename T>
__global__ void __launch_bounds__(Cfg<kSwap, kCols>::kThreads, Cfg<kSwap, kCols>::kCtasPerSm)
    w8a8_tc_kernel(const __grid_constant__ CUtensorMap tm_a,
                   const __grid_constant__ CUtensorMap tm_b, const TcArgs p) {
  using C = Cfg<kSwap, kCols>;
  constexpr int S = C::kStages, R = C::kAccs;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  float* ring = reinterpret_cast<float*>(smem + C::kRingOff);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kBarOff);
  uint64_t* empty = full + S;       // the MMAs that read the stage completed
  uint64_t* acc_full = empty + S;   // a block's sum is in TMEM
  uint64_t* acc_empty = acc_full + R;  // its buffer and scale entry have been read
  uint64_t* sc_full = acc_empty + R;   // the block's scales are in the ring
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sc_full + R);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int r = 0; r < R; ++r) {
      mbar_init(&acc_full[r], 1);
      mbar_init(&acc_empty[r], C::kPromoteWarps);
      mbar_init(&sc_full[r], 32);
    }
    fence_barrier_init();
    prefetch_tmap(&tm_a);
    prefetch_tmap(&tm_b);
  }
  if (warp == 1) tmem_alloc(tmem_slot, C::kTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // The activations (and y) may belong to the preceding kernel on the stream.
  pdl_wait();

  // This CTA's tiles, and its share of K in each: with splits > 1 a cluster has one tile.
  const int rank = p.splits > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int kb0 = static_cast<int>(static_cast<int64_t>(p.kb_total) * rank / p.splits);
  const int kb1 = static_cast<int>(static_cast<int64_t>(p.kb_total) * (rank + 1) / p.splits);
  const int tiles = p.tok_tiles * p.w_tiles;
  const int first = blockIdx.x / p.splits, step = gridDim.x / p.splits;

  if (warp == 0) {
    if (lane == 0) {
      uint32_t it = 0;
      bool ok = true;
      for (int u = first; ok && u < tiles; u += step) {
        const Tile t = tile_of<kSwap, kCols>(u, p);
        const int ra = static_cast<int>(kSwap ? t.n0 : t.m0);
        const int rb = static_cast<int>(kSwap ? t.m0 : t.n0);
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const uint32_t s = it % S;
          if (!mbar_wait(&empty[s], ((it / S) & 1u) ^ 1u, kErrProducer)) {
            ok = false;
            break;
          }
          uint8_t* st = smem + s * C::kStageBytes;
          mbar_expect_tx(&full[s], C::kStageBytes);
          tma_load_2d(st, &tm_a, &full[s], kb * kBlockK, ra);
          tma_load_2d(st + C::kABytes, &tm_b, &full[s], kb * kBlockK, rb);
        }
      }
      // Every armed stage must have landed before the CTA may exit.
      for (uint32_t j = it > S ? it - S : 0; j < it; ++j)
        if (!mbar_wait(&full[j % S], (j / S) & 1u, kErrDrain)) break;
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = (1u << 4) | (static_cast<uint32_t>(kCols >> 3) << 17) |
                                 (static_cast<uint32_t>(kLanes >> 4) << 24);
      uint32_t it = 0;
      bool ok = true;
      for (int u = first; ok && u < tiles; u += step) {
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const uint32_t s = it % S, r = it % R;
          if (!mbar_wait(&acc_empty[r], ((it / R) & 1u) ^ 1u, kErrMmaAcc) ||
              !mbar_wait(&full[s], (it / S) & 1u, kErrMmaFull)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t a_desc = sw128_desc(smem_u32(smem + s * C::kStageBytes));
          const uint64_t b_desc = sw128_desc(smem_u32(smem + s * C::kStageBytes + C::kABytes));
#pragma unroll
          for (int kk = 0; kk < kBlockK / 32; ++kk)
            umma_e4m3(tmem + r * kCols, a_desc + 2 * kk, b_desc + 2 * kk, idesc, kk > 0);
          umma_commit(&empty[s]);
          umma_commit(&acc_full[r]);
        }
      }
      // After an error the MMAs already issued must finish before the TMEM is released.
      if (!ok && it > 0) mbar_wait(&empty[(it - 1) % S], ((it - 1) / S) & 1u, kErrDrain);
    }
  } else if (warp == C::kScaleWarp) {
    // Scale entry: sx of the tile's tokens (times sw with weight rows as lanes), then sw of the
    // two 128-row weight blocks. Lane l fetches tokens l, l + 32, ...; the loads of a block are
    // issued before the wait for its ring entry.
    constexpr int kPer = (C::kTokens + 31) / 32;
    const int nb_total = static_cast<int>(cdiv(p.a.N, 128));
    uint32_t it = 0;
    bool ok = true;
    for (int u = first; ok && u < tiles; u += step) {
      const Tile t = tile_of<kSwap, kCols>(u, p);
      const int nb0 = static_cast<int>(t.n0 / 128);
      const float* sw0 = p.a.w_scale + static_cast<int64_t>(nb0) * p.kb_total;
      const float* sw1 =
          p.a.w_scale + static_cast<int64_t>(min(nb0 + 1, nb_total - 1)) * p.kb_total;
      const float* sx[kPer];
      bool have[kPer];
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int tok = lane + 32 * i;
        have[i] = tok < C::kTokens && t.m0 + tok < p.a.M;
        sx[i] = p.a.x_scale + (have[i] ? t.m0 + tok : 0) * p.a.ld_xs;
      }
      for (int kb = kb0; kb < kb1; ++kb, ++it) {
        const uint32_t r = it % R;
        float v[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) v[i] = have[i] ? sx[i][kb] : 0.f;
        const float w0 = __ldg(sw0 + kb), w1 = __ldg(sw1 + kb);
        if (!mbar_wait(&acc_empty[r], ((it / R) & 1u) ^ 1u, kErrScale)) {
          ok = false;
          break;
        }
        float* e = ring + r * C::kScaleFloats;
#pragma unroll
        for (int i = 0; i < kPer; ++i)
          if (lane + 32 * i < C::kTokens) e[lane + 32 * i] = kSwap ? v[i] * w0 : v[i];
        if (!kSwap && lane == 0) {
          e[C::kTokens] = w0;
          e[C::kTokens + 1] = w1;
        }
        mbar_arrive(&sc_full[r]);
      }
    }
  }

  // Promotion: lane q * 32 + l of the accumulator, columns c0 .. c0 + kColsPerThread.
  const int q = warp & 3, cg = (warp - 2) >> 2;
  const int c0 = cg * C::kColsPerThread;
  const int row = 32 * q + lane;
  constexpr int N2 = C::kColsPerThread / 2;
  uint64_t acc[N2];
  Tile last = {0, 0};
  if (warp >= 2 && warp < C::kScaleWarp) {
    const uint32_t taddr = tmem + (static_cast<uint32_t>(32 * q) << 16) + c0;
    const bool vec = p.a.ldy % 8 == 0 && (reinterpret_cast<uintptr_t>(p.a.y) & 15u) == 0;
    uint32_t it = 0;
    bool ok = true;
    for (int u = first; ok && u < tiles; u += step) {
      const Tile t = tile_of<kSwap, kCols>(u, p);
      last = t;
#pragma unroll
      for (int i = 0; i < N2; ++i) acc[i] = 0;
      for (int kb = kb0; kb < kb1; ++kb, ++it) {
        const uint32_t r = it % R, ph = (it / R) & 1u;
        // The vote keeps the warp together: tcgen05.ld is a warp-wide instruction.
        if (!__all_sync(0xffffffffu, mbar_wait(&sc_full[r], ph, kErrPromote) &&
                                         mbar_wait(&acc_full[r], ph, kErrPromote))) {
          ok = false;
          break;
        }
        tc_fence_after();
        const float* e = ring + r * C::kScaleFloats;
        uint64_t s2 = 0;
        if constexpr (!kSwap) {
          const float s = e[row] * e[C::kTokens + cg];
          s2 = f32x2(s, s);
        }
        const uint32_t src = taddr + r * kCols;
        constexpr int kChunks = C::kColsPerThread / 16;
        uint32_t d[2][16];
        tmem_ld16(src, d[0]);
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          tmem_ld16_wait(d[c & 1]);
          if (c + 1 < kChunks) {
            tmem_ld16(src + 16 * (c + 1), d[(c + 1) & 1]);
          } else if constexpr (!kSwap) {
            // The buffer and the scales are in registers: release both.
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[r]);
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if constexpr (kSwap) s2 = *reinterpret_cast<const uint64_t*>(e + 16 * c + 2 * j);
            acc[8 * c + j] = fma_f32x2(
                f32x2(__uint_as_float(d[c & 1][2 * j]), __uint_as_float(d[c & 1][2 * j + 1])), s2,
                acc[8 * c + j]);
          }
        }
        if constexpr (kSwap) {  // the scales are read up to the last column
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&acc_empty[r]);
        }
      }
      if (ok && p.splits == 1) {
        if constexpr (kSwap) {
          const int64_t n = t.n0 + row;
          if (n < p.a.N) {
            const float b = p.a.bias != nullptr
                                ? widen(reinterpret_cast<const T*>(p.a.bias)[n]) : 0.f;
            T* y = reinterpret_cast<T*>(p.a.y) + t.m0 * p.a.ldy + n;
#pragma unroll
            for (int i = 0; i < N2; ++i) {
              const float2 v = split_f32x2(acc[i]);
              if (t.m0 + 2 * i < p.a.M) narrow(v.x + b, y + 2 * i * p.a.ldy);
              if (t.m0 + 2 * i + 1 < p.a.M) narrow(v.y + b, y + (2 * i + 1) * p.a.ldy);
            }
          }
        } else if (t.m0 + row < p.a.M) {
#pragma unroll
          for (int c = 0; c < C::kColsPerThread / 8; ++c) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 f = split_f32x2(acc[4 * c + e]);
              v[2 * e] = f.x;
              v[2 * e + 1] = f.y;
            }
            if (t.n0 + c0 + 8 * c < p.a.N) store8<T>(p.a, t.m0 + row, t.n0 + c0 + 8 * c, vec, v);
          }
        }
      }
    }
  }

  if (p.splits > 1) {
    // Partial tiles as [column][lane] in the (drained) stages; column chunks of 8 are summed by
    // rank chunk mod splits, over the ranks in order.
    float* part = reinterpret_cast<float*>(smem);
    if (warp >= 2 && warp < C::kScaleWarp) {
#pragma unroll
      for (int i = 0; i < N2; ++i) {
        const float2 v = split_f32x2(acc[i]);
        part[(c0 + 2 * i) * kLanes + row] = v.x;
        part[(c0 + 2 * i + 1) * kLanes + row] = v.y;
      }
    }
    __syncwarp();
    cluster_sync();
    if (warp >= 2 && warp < C::kScaleWarp) {
      const bool vec = p.a.ldy % 8 == 0 && (reinterpret_cast<uintptr_t>(p.a.y) & 15u) == 0;
      // Warps of one quadrant alternate over the rank's chunks.
      for (int c = rank + cg * p.splits; c < kCols / 8; c += C::kColGroups * p.splits) {
        const int64_t col0 = (kSwap ? last.m0 : last.n0) + 8 * c;
        const int64_t lane_i = (kSwap ? last.n0 : last.m0) + row;
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        const uint32_t at = smem_u32(part + 8 * c * kLanes + row);
        for (int k = 0; k < p.splits; ++k)
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] += ld_cluster_f32(at + 4 * e * kLanes, k);
        if constexpr (kSwap) {
          if (lane_i < p.a.N) {
            const float b = p.a.bias != nullptr
                                ? widen(reinterpret_cast<const T*>(p.a.bias)[lane_i]) : 0.f;
            T* y = reinterpret_cast<T*>(p.a.y) + col0 * p.a.ldy + lane_i;
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (col0 + e < p.a.M) narrow(v[e] + b, y + e * p.a.ldy);
          }
        } else if (lane_i < p.a.M && col0 < p.a.N) {
          store8<T>(p.a, lane_i, col0, vec, v);
        }
      }
    }
    __syncwarp();
    cluster_sync();  // no CTA leaves while a peer reads its shared memory
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmemCols);
  }
}

// ----------------------------------------------------------------------------- host side

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    cudaDriverEntryPointQueryResult q;
    void* f = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
  });
  return fn;
}

bool make_map(CUtensorMap* map, const void* base, int64_t inner, int64_t rows, int64_t row_bytes,
              int box_rows) {
  auto fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(row_bytes)};
  cuuint32_t box[2] = {kBlockK, static_cast<cuuint32_t>(box_rows)};
  cuuint32_t estr[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box,
            estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr int kSms = 148;

template <bool kSwap, int kCols, typename T>
int launch_tc(const W8A8Args& a, cudaStream_t stream) {
  using C = Cfg<kSwap, kCols>;
  TcArgs p;
  p.a = a;
  p.kb_total = static_cast<int>(cdiv(a.K, kBlockK));
  const int64_t tok_tiles = cdiv(a.M, kSwap ? kCols : kLanes);
  const int64_t w_tiles = cdiv(a.N, kSwap ? kLanes : kCols);
  const int64_t tiles = tok_tiles * w_tiles;
  if (tiles > 0x7fffffffLL) return TF_ERR_TOO_LARGE;
  p.tok_tiles = static_cast<int>(tok_tiles);
  p.w_tiles = static_cast<int>(w_tiles);
  // K splits: the count that leaves the busiest SM the fewest blocks, an exchange counted as two
  // blocks; all CTAs of a split launch must fit the GPU at once to be worth it.
  const int slots = kSms * C::kCtasPerSm;
  p.splits = 1;
  int64_t best = cdiv(tiles, slots) * p.kb_total;
  for (int s = 2; s <= 8 && s <= p.kb_total && tiles * s <= slots; ++s) {
    const int64_t cost = cdiv(p.kb_total, s) + 2;
    if (cost < best) {
      best = cost;
      p.splits = s;
    }
  }
  CUtensorMap ma, mb;
  const bool ok = kSwap ? make_map(&ma, a.wq, a.K, a.N, a.K, kLanes) &&
                              make_map(&mb, a.xq, a.K, a.M, a.ldx, kCols)
                        : make_map(&ma, a.xq, a.K, a.M, a.ldx, kLanes) &&
                              make_map(&mb, a.wq, a.K, a.N, a.K, kCols);
  if (!ok) return TF_ERR_ALIGNMENT;

  auto kernel = w8a8_tc_kernel<kSwap, kCols, T>;
  static std::once_flag attr_once[64];
  int dev = 0;
  cudaGetDevice(&dev);
  cudaError_t e = cudaSuccess;
  std::call_once(attr_once[dev & 63], [&] {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  });
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.splits > 1 ? tiles * p.splits
                                                        : std::min<int64_t>(tiles, slots)));
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (p.splits > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = static_cast<unsigned>(p.splits);
    attr[n].val.clusterDim.y = 1;
    attr[n++].val.clusterDim.z = 1;
  }
  if (launch_flags() & TF_LAUNCH_PDL) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, kernel, ma, mb, p);
  if (e != cudaSuccess) {
    last_cuda_error() = static_cast<int>(e);
    return TF_ERR_CUDA;
  }
  return TF_OK;
}

template <bool kSwap, int kCols>
int launch_typed(const W8A8Args& a, cudaStream_t stream) {
  return a.dtype == TF_DTYPE_FP16 ? launch_tc<kSwap, kCols, __half>(a, stream)
                                  : launch_tc<kSwap, kCols, __nv_bfloat16>(a, stream);
}

}  // namespace

int launch_w8a8_tc(const W8A8Args& a, cudaStream_t stream) {
  if (a.M <= 16) return launch_typed<true, 16>(a, stream);
  if (a.M <= 32) return launch_typed<true, 32>(a, stream);
  if (a.M <= 64) return launch_typed<true, 64>(a, stream);
  return launch_typed<false, 256>(a, stream);
}

int w8a8_device_error(int* code) {
  const cudaError_t e = cudaMemcpyFromSymbol(code, g_w8a8_error, sizeof(int));
  if (e != cudaSuccess) {
    last_cuda_error() = static_cast<int>(e);
    return TF_ERR_CUDA;
  }
  return TF_OK;
}

int w8a8_reset_device_error() {
  const int zero = 0;
  const cudaError_t e = cudaMemcpyToSymbol(g_w8a8_error, &zero, sizeof(int));
  if (e != cudaSuccess) {
    last_cuda_error() = static_cast<int>(e);
    return TF_ERR_CUDA;
  }
  return TF_OK;
}

}  // namespace tfb
