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
// Two kernels, by which operand gives the accumulator's 128 lanes:
//   w8a8_pair_kernel, tokens as lanes, many tokens: a CTA pair (two SMs, cta_group::2 MMAs)
//     computes 256 tokens x 256 weight rows, each CTA holding 128 tokens' sums and half of the
//     weight rows in shared memory, so a block costs an SM 32 KB of loads instead of the 48 KB of a
//     single CTA's 128 x 256 tile. (A kernel of such tiles stopped at 2180 TFLOP/s even without
//     promotion. Why is not established: L2 is at a third of its throughput here.) A lane is a
//     token, so a block's scale is one number per thread, and promotion costs one packed FMA per
//     two values. Two warps per TMEM quadrant, 128 columns each.
//     Measured, bf16, a graph of calls: 4096 x 37888 x 3584 in 461 to 516 us (2410 to 2160
//     TFLOP/s, with the GPU's power state), 1024 x 37888 x 3584 in 124, 1024 x 3584 x 18944 in 67,
//     256 x 3584 x 18944 in 27. Bound by the promotion, 847 cycles a block where its MMAs take 512
//     (1024 x 37888 x 3584: an SM is active for 189.8 thousand cycles, 224 blocks, tile ends
//     included), and by the clock, which falls to 1.6 GHz in that kernel and to 1.44 in a second of
//     such calls, under the power cap.
//   w8a8_swap_kernel, weight rows as lanes, few tokens: tile of 128 weight rows x 16, 32 or 64
//     tokens. No tensor-core rows are wasted on missing tokens, the weight stream sets the pace,
//     and the scale of a column (token) comes from shared memory. One warp per quadrant.
//     Measured: 16 x 37888 x 3584 in 25.1 us (5.46 TB/s, 85 % of a copy's rate), 16 x 3584 x
//     18944 in 17.4 us (28 weight tiles, 4 shares of K each: 112 of 148 SMs, since 26 clusters of 5
//     are resident at once, and 2 us of exchange).
//
// Warps: 0 TMA producer, 1 TMEM allocation and MMA issue (the pair's warp 3 issues every other
// block), 2 fetches each block's scales into a small ring; warps from 4 on promote. Persistent CTAs
// (pairs) walk the tiles with the token tile fastest, so the weight tile stays in L2. When there
// are fewer tiles than SMs, the CTAs of a cluster split K instead and sum their tiles through
// distributed shared memory in a fixed order, so the result does not depend on timing and no
// workspace is needed. Every wait is bounded (2 s): on a time-out the kernel records an error
// code for tf_device_error, stops, lets its copies and MMAs finish, frees its TMEM and returns. No
// TMA multicast is used.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
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

struct TcArgs {
  W8A8Args a;
  int kb_total, tok_tiles, w_tiles, splits;
  int tma_out;     // y can be written by TMA
  int vec_scales;  // x_scale rows are 16-byte aligned
};

__device__ __forceinline__ bool mbar_wait_slow(uint64_t* bar, uint32_t parity, int site) {
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

// A wait that nothing ends early: for copies and MMAs in flight, and their arrivals, which must
// finish before shared memory or TMEM is given up. False if it gave up.
__device__ __forceinline__ bool mbar_drain(uint64_t* bar, uint32_t parity) {
  const unsigned long long t0 = global_ns();
  while (!mbar_try_wait(bar, parity))
    if (global_ns() - t0 > kWaitLimitNs) {
      atomicCAS(&g_w8a8_error, 0, kErrDrain);
      return false;
    }
  return true;
}
// The commits of a CTA's last blocks arrive on its `empty` barriers asynchronously, and in the pair
// kernel they come from the other CTA: the producer, whose loads have used stages 0 .. it - 1,
// waits for those of the last `kStages`, or the CTA could exit, and its shared memory pass to
// another kernel, with an arrival on the way. After an error some are never sent: one wait then
// runs into its limit and the others are given up.
template <int kStages>
__device__ __forceinline__ void drain_empty(uint64_t* empty, uint32_t it) {
  for (uint32_t j = it > kStages ? it - kStages : 0; j < it; ++j)
    if (!mbar_drain(&empty[j % kStages], (j / kStages) & 1u)) return;
}

// D[tmem] (+)= A[smem] * B[smem]^T, e4m3 inputs, fp32 accumulate, K = 32, issued by one thread
// (of the leading CTA of a pair).
__device__ __forceinline__ void umma_e4m3(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                          uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_e4m3_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                               uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Instruction descriptor: fp32 D, e4m3 A and B, both K-major, `rows` x `cols`.
__device__ __forceinline__ constexpr uint32_t idesc_e4m3(int rows, int cols) {
  return (1u << 4) | (static_cast<uint32_t>(cols >> 3) << 17) |
         (static_cast<uint32_t>(rows >> 4) << 24);
}

template <int kRegs>
__device__ __forceinline__ void set_max_regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}
template <int kRegs>
__device__ __forceinline__ void set_max_regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
}

// The first 1024-byte boundary, as an offset from the array (an address rounded as an integer
// would lose its address space, and every access become a generic one).
__device__ __forceinline__ uint8_t* align_smem(uint8_t* raw) {
  return raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
}

// K blocks [kb0, kb1) of share `index` of `splits`.
__device__ __forceinline__ int kb_begin(const TcArgs& p, int index) {
  return static_cast<int>(static_cast<int64_t>(p.kb_total) * index / p.splits);
}

// One entry of the scale ring: one value per token of the tile, then up to four of the weight
// blocks.
template <int kTokens>
struct ScaleEntry {
  float sx[kTokens];
  float sw[4];
};

// Where a split tile's partial sums lie in shared memory: 16-byte vector c (columns 4c .. 4c + 3)
// of lane `row`, the lanes of one vector next to each other, so that a warp reads 512 contiguous
// bytes of a peer (rows of a whole tile, a warp's vectors 1 KB apart, made an exchange three
// times slower).
__device__ __forceinline__ uint32_t part_at(int row, int c) {
  return static_cast<uint32_t>((c * kLanes + row) * 16);
}

// The scale warp's view of one tile: lane l fetches tokens l, l + 32, ... of `kTokens`, four K
// blocks at a time (one 16-byte load a token where rows allow it) and
// one such group ahead of its use: fetched block by block, every eighth one (a new 32-byte
// sector) stalled the promotion for the time of an L2 miss.
template <int kTokens>
struct ScaleRows {
  static constexpr int kPer = (kTokens + 31) / 32;
  const float* base;  // this lane's first token
  int count;          // tokens of the tile from it on
  float x[kPer][4], next[kPer][4];
  __device__ __forceinline__ ScaleRows(const TcArgs& p, int64_t m0, int lane) {
    base = p.a.x_scale + (m0 + lane) * p.a.ld_xs;
    count = static_cast<int>(min(p.a.M - m0, static_cast<int64_t>(kTokens))) - lane;
  }
  __device__ __forceinline__ void fetch(const TcArgs& p, int group) {
    const int kb = 4 * group;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const float* at = base + 32 * i * p.a.ld_xs + kb;
      if (p.vec_scales && kb + 4 <= p.kb_total) {
        const float4 v = 32 * i < count ? *reinterpret_cast<const float4*>(at)
                                        : make_float4(0.f, 0.f, 0.f, 0.f);
        next[i][0] = v.x;
        next[i][1] = v.y;
        next[i][2] = v.z;
        next[i][3] = v.w;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          next[i][j] = 32 * i < count && kb + j < p.kb_total ? at[j] : 0.f;
      }
    }
  }
  __device__ __forceinline__ void advance() {
#pragma unroll
    for (int i = 0; i < kPer; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) x[i][j] = next[i][j];
  }
};

// ------------------------------------------------------------------ tokens as lanes, CTA pair

struct Pair {
  static constexpr int kTokens = 2 * kLanes;  // of a tile; each CTA holds 128
  static constexpr int kCols = 256;           // weight rows of a tile; each CTA stages 128
  static constexpr int kColGroups = 2;        // promotion warps per TMEM quadrant
  static constexpr int kColsPerThread = kCols / kColGroups;
  static constexpr int kPromoteWarps = 4 * kColGroups;
  static constexpr int kThreads = 128 + 32 * kPromoteWarps;
  // Registers a thread: at launch, then of the first warpgroup and of the promoting ones; the
  // shares add up to what the CTA was launched with.
  static constexpr int kLaunchRegs = 168, kControlRegs = 88, kPromoteRegs = 208;
  static_assert(128 * kControlRegs + 32 * kPromoteWarps * kPromoteRegs == kThreads * kLaunchRegs,
                "register split");
  static constexpr int kABytes = kLanes * kBlockK;
  static constexpr int kBBytes = kCols / 2 * kBlockK;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kStages = 4;
  static constexpr int kTmemCols = 2 * kCols;  // two buffers
  static constexpr int kScaleSlots = 4;
  using Scales = ScaleEntry<kLanes>;
  // Output staging of a promotion warp: tiles of 32 tokens x 64 columns of 16 bits, 128-byte
  // swizzle.
  static constexpr int kOutCols = 64, kOutTile = 32 * kOutCols * 2;
  static constexpr int kOutBytes = kColsPerThread / kOutCols * kOutTile;
  static constexpr int kOutOff = kStages * kStageBytes;
  static constexpr int kRingOff = kOutOff + kPromoteWarps * kOutBytes;
  static constexpr int kBarOff = kRingOff + kScaleSlots * static_cast<int>(sizeof(Scales));
  static constexpr int kSmem = 1024 + kBarOff + 512;
  static_assert(kSmem <= 227 * 1024 && kTmemCols <= 512, "budgets");
  // The exchange of partial tiles reuses the stages once the last block is done.
  static_assert(kLanes * kCols * 4 <= kOutOff, "exchange buffer");
};

// Staging of a warp's outputs in shared memory: 32 tokens x 64 columns a tile, a token's 128 bytes
// swizzled as TMA expects them (16-byte chunk c of row r at chunk c ^ (r & 7)).
__device__ __forceinline__ uint32_t staged(int row, int col) {
  return static_cast<uint32_t>(col >> 6) * Pair::kOutTile + row * 128 +
         ((((col >> 3) ^ row) & 7) << 4) + (col & 7) * 2;
}
// Writes this lane's token, `kCols` columns from v(0), v(1), ...
template <typename T, int kCols, typename V>
__device__ __forceinline__ void stage_row(uint8_t* out, int lane, V v) {
#pragma unroll
  for (int c = 0; c < kCols / 8; ++c) {
    uint4 o;
    o.x = narrow2(v(8 * c), v(8 * c + 1), T());
    o.y = narrow2(v(8 * c + 2), v(8 * c + 3), T());
    o.z = narrow2(v(8 * c + 4), v(8 * c + 5), T());
    o.w = narrow2(v(8 * c + 6), v(8 * c + 7), T());
    *reinterpret_cast<uint4*>(out + staged(lane, 8 * c)) = o;
  }
}
// Copies the staged tokens m .. m + 31 to y, kCols columns from n on. Rows of 16-byte vectors: a
// lane a vector. Others: a lane reads pairs of columns; where the row starts at an odd address (in
// units of two outputs) its words are made of a pair's second column and the next pair's first,
// so that every row is written in 4-byte words but for its ends (a store of 2 bytes a lane, with
// a load each, cost 2.5 us more on 333 x 4613).
template <typename T, int kCols>
__device__ __forceinline__ void copy_rows(const W8A8Args& a, const uint8_t* out, int64_t m,
                                          int64_t n, bool vec, int lane) {
  const int rows = static_cast<int>(min(static_cast<int64_t>(32), a.M - m));
  T* y = reinterpret_cast<T*>(a.y) + m * a.ldy + n;
  if (vec && n + kCols <= a.N) {
    constexpr int kLanesPerRow = kCols / 8, kRowsPerStep = 32 / kLanesPerRow;
    const int c = lane % kLanesPerRow * 8;
#pragma unroll
    for (int r = lane / kLanesPerRow; r < 32; r += kRowsPerStep)
      if (r < rows)
        *reinterpret_cast<uint4*>(y + r * a.ldy + c) =
            *reinterpret_cast<const uint4*>(out + staged(r, c));
    return;
  }
  constexpr int kPairs = kCols / 2, kSpan = kPairs < 32 ? kPairs : 32, kPer = kPairs / kSpan;
  if (n >= a.N) return;
  const int lim = static_cast<int>(min(static_cast<int64_t>(kCols), a.N - n));
  const int l = lane % kSpan;
#pragma unroll 2
  for (int r0 = 0; r0 < rows; r0 += 32 / kSpan) {
    const int r = r0 + lane / kSpan;
    uint16_t* to = reinterpret_cast<uint16_t*>(y + r * a.ldy);
    const int odd = static_cast<int>(reinterpret_cast<uintptr_t>(to) >> 1) & 1;
    uint32_t w[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      w[i] = *reinterpret_cast<const uint32_t*>(out + staged(r, 2 * (l + kSpan * i)));
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      uint32_t next = __shfl_down_sync(0xffffffffu, w[i], 1, kSpan);
      if (i + 1 < kPer) {
        const uint32_t first = __shfl_sync(0xffffffffu, w[(i + 1) % kPer], 0, kSpan);
        if (l == kSpan - 1) next = first;
      }
      const int c = 2 * (l + kSpan * i) + odd;
      const uint32_t v = odd ? __funnelshift_r(w[i], next, 16) : w[i];
      if (r < rows) {
        if (c + 1 < lim)
          *reinterpret_cast<uint32_t*>(to + c) = v;
        else if (c < lim)
          to[c] = static_cast<uint16_t>(v);
        if (odd && c == 1) to[0] = static_cast<uint16_t>(w[i]);
      }
    }
  }
}
// Lane l's bias of column n + l (0 past N).
template <typename T>
__device__ __forceinline__ float bias_of(const W8A8Args& a, int64_t n) {
  return n < a.N ? widen(reinterpret_cast<const T*>(a.bias)[n]) : 0.f;
}

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* src, int c0,
                                             int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(smem_u32(src)), "r"(c0), "r"(c1)
               : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// The stores issued by this thread have read their shared memory.
__device__ __forceinline__ void tma_store_read_wait() {
  asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
}

template <typename T>
__global__ void __launch_bounds__(Pair::kThreads, 1)
    w8a8_pair_kernel(const __grid_constant__ CUtensorMap tm_x,
                     const __grid_constant__ CUtensorMap tm_w,
                     const __grid_constant__ CUtensorMap tm_y, const TcArgs p) {
  using C = Pair;
  constexpr int S = C::kStages, R = C::kScaleSlots;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align_smem(smem_raw);
  C::Scales* ring = reinterpret_cast<C::Scales*>(smem + C::kRingOff);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kBarOff);  // leader: both CTAs' bytes
  uint64_t* empty = full + S;          // each CTA: the MMAs have read the stage
  uint64_t* acc_full = empty + S;      // each CTA: a block's sums are in TMEM, its scales in the ring
  uint64_t* acc_empty = acc_full + 2;  // leader: both CTAs have read them
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  static_assert((2 * S + 4) * 8 + 8 <= 512, "barriers");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_cta_rank());
  const int side = rank & 1, lead = rank & ~1, share = rank >> 1;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1 + 32);  // the MMAs' commit and the scale warp's lanes
      mbar_init(&acc_empty[b], 2 * C::kPromoteWarps);
    }
    fence_barrier_init();
    prefetch_tmap(&tm_x);
    prefetch_tmap(&tm_w);
  }
  if (warp == 1) tmem_alloc_pair(tmem_slot, C::kTmemCols);
  tc_fence_before();
  __syncthreads();
  cluster_barrier();  // the peer's barriers and TMEM are ready
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // The activations (and y) may belong to the preceding kernel on the stream.
  pdl_begin();

  // This pair's tiles, and its share of K in each: with splits > 1 a cluster has one tile.
  const int kb0 = kb_begin(p, share), kb1 = kb_begin(p, share + 1);
  const int tiles = p.tok_tiles * p.w_tiles;
  const int first = static_cast<int>(blockIdx.x) / (2 * p.splits);
  const int step = static_cast<int>(gridDim.x) / (2 * p.splits);

  // The two groups share no code below, since they differ in the registers they may name. Both
  // end with the same barriers: the exchange's first (splits > 1), the cluster's last one.
  if (warp < 4) {
    set_max_regs_dec<C::kControlRegs>();
    if (warp == 0 && lane == 0) {
      uint32_t it = 0;
      bool ok = true;
      for (int u = first; ok && u < tiles; u += step) {
        const int m0 = u % p.tok_tiles * C::kTokens + kLanes * side;
        const int n0 = u / p.tok_tiles * C::kCols + C::kCols / 2 * side;
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const uint32_t s = it % S;
          if (!mbar_wait(&empty[s], ((it / S) & 1u) ^ 1u, kErrProducer)) {
            ok = false;
            break;
          }
          uint8_t* st = smem + s * C::kStageBytes;
          const uint32_t bar = map_to_rank(smem_u32(&full[s]), lead);
          if (side == 0) mbar_expect_tx(&full[s], 2 * C::kStageBytes);
          tma_load_2d_pair(st, &tm_x, bar, kb * kBlockK, m0);
          tma_load_2d_pair(st + C::kABytes, &tm_w, bar, kb * kBlockK, n0);
        }
      }
      // Every armed stage must have landed (in both CTAs) before either may exit.
      if (side == 0)
        for (uint32_t j = it > S ? it - S : 0; j < it; ++j)
          mbar_drain(&full[j % S], (j / S) & 1u);
      drain_empty<S>(empty, it);
    } else if ((warp == 1 || warp == 3) && lane == 0 && side == 0) {
      // Two issuing threads, for even and odd blocks (and TMEM buffers): an MMA's issue waits for
      // the one before it, so while one thread waits on barriers and commits, the other one's
      // MMAs keep the tensor core busy.
      constexpr uint32_t idesc = idesc_e4m3(C::kTokens, C::kCols);
      const uint16_t both = static_cast<uint16_t>(3u << lead);
      const uint32_t b = warp >> 1;
      uint32_t it = 0;
      bool ok = true, issued = false;
      for (int u = first; ok && u < tiles; u += step) {
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          if ((it & 1u) != b) continue;
          const uint32_t s = it % S;
          if (!mbar_wait(&acc_empty[b], ((it >> 1) & 1u) ^ 1u, kErrMmaAcc) ||
              !mbar_wait(&full[s], (it / S) & 1u, kErrMmaFull)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t a_desc = sw128_desc(smem_u32(smem + s * C::kStageBytes));
          const uint64_t b_desc = sw128_desc(smem_u32(smem + s * C::kStageBytes + C::kABytes));
#pragma unroll
          for (int kk = 0; kk < kBlockK / 32; ++kk)
            umma_e4m3_pair(tmem + b * C::kCols, a_desc + 2 * kk, b_desc + 2 * kk, idesc, kk > 0);
          umma_commit_pair(&acc_full[b], both);
          umma_commit_pair(&empty[s], both);
          issued = true;
        }
      }
      // After an error the MMAs already issued must finish before the TMEM is released.
      if (!ok && issued) {
        const uint32_t last = ((it & 1u) == b ? it : it - 1) - 2;  // this thread's last block
        mbar_drain(&acc_full[b], (last >> 1) & 1u);
      }
    } else if (warp == 2) {
      // The loads of a block are issued before the wait for its ring entry. The wait is for the
      // sums two blocks back, which use the same barrier: they also tell that every warp is done
      // with the block before those (its TMEM buffer was overwritten), four back, whose entry
      // this block takes.
      const int nb_last = static_cast<int>(cdiv(p.a.N, 128)) - 1;
      uint32_t it = 0;
      bool ok = true;
      for (int u = first; ok && u < tiles; u += step) {
        const int64_t m0 = static_cast<int64_t>(u % p.tok_tiles) * C::kTokens + kLanes * side;
        const int nb = min(u / p.tok_tiles * (C::kCols / 128) + (lane & 1), nb_last);
        const float* sw = p.a.w_scale + static_cast<int64_t>(nb) * p.kb_total;
        ScaleRows<kLanes> rows(p, m0, lane);
        rows.fetch(p, kb0 >> 2);
        for (int g = kb0 >> 2; ok && 4 * g < kb1; ++g) {
          rows.advance();
          if (4 * (g + 1) < kb1) rows.fetch(p, g + 1);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (4 * g + j < kb0 || 4 * g + j >= kb1) continue;
            const float w = sw[4 * g + j];
            if (!mbar_wait(&acc_full[it & 1u], ((it >> 1) & 1u) ^ 1u, kErrScale)) {
              ok = false;
              break;
            }
            C::Scales& e = ring[it % R];
#pragma unroll
            for (int i = 0; i < ScaleRows<kLanes>::kPer; ++i) e.sx[lane + 32 * i] = rows.x[i][j];
            if (lane < 2) e.sw[lane] = w;
            mbar_arrive(&acc_full[it & 1u]);
            ++it;
          }
        }
      }
    }
    __syncwarp();
    if (p.splits > 1) cluster_barrier();
    tc_fence_before();
    cluster_barrier();
    if (warp == 1) {
      tc_fence_after();
      tmem_dealloc_pair(tmem, C::kTmemCols);
    }
    return;
  }

  set_max_regs_inc<C::kPromoteRegs>();
  // Promotion: lane 32q + l of the accumulator, columns c0 .. c0 + 127 of the tile.
  const int q = warp & 3, cg = (warp - 4) >> 2;
  const int c0 = cg * C::kColsPerThread;
  const int row = 32 * q + lane;
  constexpr int N2 = C::kColsPerThread / 2, kChunk = 32, kChunks = C::kColsPerThread / kChunk;
  static_assert(kChunks % 2 == 0, "a block's last chunk and the next one's first alternate");
  const uint32_t taddr = tmem + (static_cast<uint32_t>(32 * q) << 16) + c0;
  const uint32_t release0 = map_to_rank(smem_u32(&acc_empty[0]), lead);
  const uint32_t release1 = map_to_rank(smem_u32(&acc_empty[1]), lead);
  uint8_t* out = smem + C::kOutOff + (warp - 4) * C::kOutBytes;
  uint64_t acc[N2];
  uint32_t d[2][kChunk];
  int64_t m = 0, n0 = 0;
  uint32_t it = 0;
  bool ok = true;
  // Adds chunk c, pairs j0 .. j1, of a block's sums times the block's scale.
  auto add = [&](const uint32_t(&v)[kChunk], int c, int j0, int j1, uint64_t s2) {
#pragma unroll
    for (int j = j0; j < j1; ++j)
      acc[kChunk / 2 * c + j] =
          fma_f32x2(f32x2(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1])), s2,
                    acc[kChunk / 2 * c + j]);
  };
  for (int u = first; ok && u < tiles; u += step) {
    m = static_cast<int64_t>(u % p.tok_tiles) * C::kTokens + kLanes * side + row;
    n0 = static_cast<int64_t>(u / p.tok_tiles) * C::kCols;
#pragma unroll
    for (int i = 0; i < N2; ++i) acc[i] = 0;
    // Votes keep the warp together: tcgen05.ld is a warp-wide instruction.
    ok = __all_sync(0xffffffffu, mbar_wait(&acc_full[it & 1u], (it >> 1) & 1u, kErrPromote));
    if (!ok) break;
    tc_fence_after();
    tmem_ld(taddr + (it & 1u) * C::kCols, d[0]);
    // Chunks of 32 columns in one stream over the blocks: the next chunk is fetched, across the
    // end of a block too, while one is added.
    for (int kb = kb0; kb < kb1; ++kb, ++it) {
      const uint32_t b = it & 1u;
      const float sc = ring[it % R].sx[row] * ring[it % R].sw[cg];
      const uint64_t s2 = f32x2(sc, sc);
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        tmem_ld_wait(d[c & 1]);
        if (c + 1 < kChunks) {
          tmem_ld(taddr + b * C::kCols + kChunk * (c + 1), d[(c + 1) & 1]);
          add(d[c & 1], c, 0, kChunk / 2, s2);
        } else {
          // The buffer and the scales are in registers: release both.
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_remote(b ? release1 : release0);
          if (kb + 1 < kb1) {
            const uint32_t ph = ((it + 1) >> 1) & 1u;
            const bool ready = mbar_try_wait(&acc_full[b ^ 1u], ph);
            add(d[c & 1], c, 0, kChunk / 4, s2);
            ok = __all_sync(0xffffffffu,
                            ready || mbar_wait_slow(&acc_full[b ^ 1u], ph, kErrPromote));
            if (!ok) break;
            tc_fence_after();
            tmem_ld(taddr + (b ^ 1u) * C::kCols, d[0]);
            add(d[c & 1], c, kChunk / 4, kChunk / 2, s2);
          } else {
            add(d[c & 1], c, 0, kChunk / 2, s2);
          }
        }
      }
      if (!ok) break;
    }
    if (ok && p.splits == 1) {
      if (p.a.bias != nullptr) {
#pragma unroll
        for (int k = 0; k < C::kColsPerThread / 32; ++k) {
          const float mine = bias_of<T>(p.a, n0 + c0 + 32 * k + lane);
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float2 f = split_f32x2(acc[16 * k + j]);
            acc[16 * k + j] = f32x2(f.x + __shfl_sync(0xffffffffu, mine, 2 * j),
                                    f.y + __shfl_sync(0xffffffffu, mine, 2 * j + 1));
          }
        }
      }
      // The previous tile's copy out of the staging area is done; TMA writes this one (clipped at
      // M and N) while the warp goes on.
      if (lane == 0) tma_store_read_wait();
      __syncwarp();
      stage_row<T, C::kColsPerThread>(out, lane, [&](int i) {
        const float2 f = split_f32x2(acc[i / 2]);
        return i & 1 ? f.y : f.x;
      });
      if (p.tma_out) {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0 && m < p.a.M)
#pragma unroll
          for (int t = 0; t < C::kColsPerThread / C::kOutCols; ++t)
            if (n0 + c0 + t * C::kOutCols < p.a.N)
              tma_store_2d(&tm_y, out + t * C::kOutTile, static_cast<int>(n0) + c0 + t * C::kOutCols,
                           static_cast<int>(m));
      } else {
        __syncwarp();
        copy_rows<T, C::kColsPerThread>(p.a, out, m - lane, n0 + c0, false, lane);
        __syncwarp();
      }
    }
  }
  if (lane == 0) tma_store_read_wait();
  __syncwarp();

  if (p.splits > 1) {
    // Partial tiles in the (drained) stages. Units of 32 columns are dealt to the shares, and a
    // share's to its two warps of a quadrant, which sum them over the shares in an order of the
    // unit's own (its owner's share first, so that the CTAs do not all read the same one at a
    // time).
#pragma unroll
    for (int i = 0; i < N2 / 2; ++i) {
      const float2 f = split_f32x2(acc[2 * i]), g = split_f32x2(acc[2 * i + 1]);
      *reinterpret_cast<float4*>(smem + part_at(row, c0 / 4 + i)) =
          make_float4(f.x, f.y, g.x, g.y);
    }
    __syncwarp();
    cluster_barrier();
    for (int unit = share + cg * p.splits; unit < C::kCols / 32; unit += 2 * p.splits) {
      float v[32];
#pragma unroll
      for (int e = 0; e < 32; ++e) v[e] = 0.f;
#pragma unroll 2
      for (int k = 0; k < p.splits; ++k) {
        const int from = share + k < p.splits ? share + k : share + k - p.splits;
        const uint32_t at = map_to_rank(smem_u32(smem), 2 * from + side);
        float4 w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = ld_cluster_v4(at + part_at(row, 8 * unit + e));
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[4 * e] += w[e].x;
          v[4 * e + 1] += w[e].y;
          v[4 * e + 2] += w[e].z;
          v[4 * e + 3] += w[e].w;
        }
      }
      if (p.a.bias != nullptr) {
        const float mine = bias_of<T>(p.a, n0 + 32 * unit + lane);
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] += __shfl_sync(0xffffffffu, mine, e);
      }
      stage_row<T, 32>(out, lane, [&](int i) { return v[i]; });
      __syncwarp();
      copy_rows<T, 32>(p.a, out, m - lane, n0 + 32 * unit, p.tma_out != 0, lane);
      __syncwarp();
    }
  }
  tc_fence_before();
  cluster_barrier();  // no CTA leaves, or frees its TMEM, while the other one needs it
}

// ------------------------------------------------------------------ weight rows as lanes

template <int kCols>
struct Swap {
  static constexpr int kThreads = 256;
  static constexpr int kABytes = kLanes * kBlockK;
  static constexpr int kBBytes = kCols * kBlockK;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kAccs = 4;
  static constexpr int kTmemCols = kAccs * kCols;
  using Scales = ScaleEntry<kCols>;
  static constexpr int kTail = 1024 + kAccs * static_cast<int>(sizeof(Scales)) + 512;
  // More stages than fit 160 KB were slower again (37888 x 3584, 16 tokens: 25.2 us with 160 KB,
  // 25.6 with 112, 27.1 with 220): about 1000 128-byte TMA rows in flight an SM are enough.
  static constexpr int kBudget = 160 * 1024;
  static constexpr int kStages = (kBudget - kTail) / kStageBytes;
  static constexpr int kRingOff = kStages * kStageBytes;
  static constexpr int kBarOff = kRingOff + kAccs * static_cast<int>(sizeof(Scales));
  static constexpr int kSmem = 1024 + kBarOff + 512;
  static_assert(kTmemCols >= 32 && kTmemCols <= 512, "TMEM");
  static_assert(kLanes * kCols * 4 <= kRingOff, "exchange buffer");
};

// Output column `m` (a token) .. of one weight row n, bias added: 32 lanes write 32 neighbours.
template <typename T>
__device__ __forceinline__ void store_token(const W8A8Args& a, int64_t m, int64_t n, float v,
                                            float bias) {
  if (m < a.M) narrow(v + bias, reinterpret_cast<T*>(a.y) + m * a.ldy + n);
}

template <int kCols, typename T>
__global__ void __launch_bounds__(Swap<kCols>::kThreads, 1)
    w8a8_swap_kernel(const __grid_constant__ CUtensorMap tm_w,
                     const __grid_constant__ CUtensorMap tm_x,
                     const __grid_constant__ CUtensorMap, const TcArgs p) {
  using C = Swap<kCols>;
  constexpr int S = C::kStages, R = C::kAccs;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align_smem(smem_raw);
  typename C::Scales* ring = reinterpret_cast<typename C::Scales*>(smem + C::kRingOff);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kBarOff);
  uint64_t* empty = full + S;          // the MMAs that read the stage completed
  uint64_t* acc_full = empty + S;      // a block's sums are in TMEM
  uint64_t* acc_empty = acc_full + R;  // its buffer and scale entry have been read
  uint64_t* sc_full = acc_empty + R;   // the block's scales are in the ring
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sc_full + R);
  static_assert((2 * S + 3 * R) * 8 + 8 <= 512, "barriers");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int r = 0; r < R; ++r) {
      mbar_init(&acc_full[r], 1);
      mbar_init(&acc_empty[r], 4);
      mbar_init(&sc_full[r], 32);
    }
    fence_barrier_init();
    prefetch_tmap(&tm_w);
    prefetch_tmap(&tm_x);
  }
  if (warp == 1) tmem_alloc(tmem_slot, C::kTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // The activations (and y) may belong to the preceding kernel on the stream.
  pdl_begin();

  // This CTA's tiles, and its share of K in each: with splits > 1 a cluster has one tile.
  const int share = p.splits > 1 ? static_cast<int>(cluster_cta_rank()) : 0;
  const int kb0 = kb_begin(p, share), kb1 = kb_begin(p, share + 1);
  const int tiles = p.tok_tiles * p.w_tiles;
  const int first = static_cast<int>(blockIdx.x) / p.splits;
  const int step = static_cast<int>(gridDim.x) / p.splits;

  if (warp == 0 && lane == 0) {
    uint32_t it = 0;
    bool ok = true;
    for (int u = first; ok && u < tiles; u += step) {
      const int m0 = u % p.tok_tiles * kCols, n0 = u / p.tok_tiles * kLanes;
      for (int kb = kb0; kb < kb1; ++kb, ++it) {
        const uint32_t s = it % S;
        if (!mbar_wait(&empty[s], ((it / S) & 1u) ^ 1u, kErrProducer)) {
          ok = false;
          break;
        }
        uint8_t* st = smem + s * C::kStageBytes;
        mbar_expect_tx(&full[s], C::kStageBytes);
        tma_load_2d(st, &tm_w, &full[s], kb * kBlockK, n0);
        tma_load_2d(st + C::kABytes, &tm_x, &full[s], kb * kBlockK, m0);
      }
    }
    // Every armed stage must have landed before the CTA may exit.
    for (uint32_t j = it > S ? it - S : 0; j < it; ++j) mbar_drain(&full[j % S], (j / S) & 1u);
    drain_empty<S>(empty, it);
  } else if (warp == 1 && lane == 0) {
    constexpr uint32_t idesc = idesc_e4m3(kLanes, kCols);
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
    if (!ok && it > 0) mbar_drain(&empty[(it - 1) % S], ((it - 1) / S) & 1u);
  } else if (warp == 2) {
    // A tile's 128 weight rows share one scale, so the entry holds the products sx * sw.
    uint32_t it = 0;
    bool ok = true;
    for (int u = first; ok && u < tiles; u += step) {
      const float* sw = p.a.w_scale + static_cast<int64_t>(u / p.tok_tiles) * p.kb_total;
      ScaleRows<kCols> rows(p, static_cast<int64_t>(u % p.tok_tiles) * kCols, lane);
      rows.fetch(p, kb0 >> 2);
      for (int g = kb0 >> 2; ok && 4 * g < kb1; ++g) {
        rows.advance();
        if (4 * (g + 1) < kb1) rows.fetch(p, g + 1);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (4 * g + j < kb0 || 4 * g + j >= kb1) continue;
          const uint32_t r = it % R;
          const float w = sw[4 * g + j];
          if (!mbar_wait(&acc_empty[r], ((it / R) & 1u) ^ 1u, kErrScale)) {
            ok = false;
            break;
          }
#pragma unroll
          for (int i = 0; i < ScaleRows<kCols>::kPer; ++i)
            if (lane + 32 * i < kCols) ring[r].sx[lane + 32 * i] = rows.x[i][j] * w;
          mbar_arrive(&sc_full[r]);
          ++it;
        }
      }
    }
  }

  // Promotion (warps 4-7): lane 32q + l of the accumulator, all columns.
  const int q = warp & 3, row = 32 * q + lane;
  constexpr int N2 = kCols / 2, kChunk = kCols < 32 ? kCols : 32;
  uint64_t acc[N2];
  int64_t m0 = 0, n = 0;
  float bias = 0.f;
  if (warp >= 4) {
    const uint32_t taddr = tmem + (static_cast<uint32_t>(32 * q) << 16);
    uint32_t it = 0;
    bool ok = true;
    for (int u = first; ok && u < tiles; u += step) {
      m0 = static_cast<int64_t>(u % p.tok_tiles) * kCols;
      n = static_cast<int64_t>(u / p.tok_tiles) * kLanes + row;
      bias = p.a.bias != nullptr && n < p.a.N ? widen(reinterpret_cast<const T*>(p.a.bias)[n])
                                              : 0.f;
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
        const uint64_t* sc = reinterpret_cast<const uint64_t*>(ring[r].sx);
#pragma unroll
        for (int c = 0; c < kCols / kChunk; ++c) {
          uint32_t d[kChunk];
          tmem_ld(taddr + r * kCols + kChunk * c, d);
          tmem_ld_wait(d);
#pragma unroll
          for (int j = 0; j < kChunk / 2; ++j)
            acc[kChunk / 2 * c + j] =
                fma_f32x2(f32x2(__uint_as_float(d[2 * j]), __uint_as_float(d[2 * j + 1])),
                          sc[kChunk / 2 * c + j], acc[kChunk / 2 * c + j]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_empty[r]);
      }
      if (ok && p.splits == 1 && n < p.a.N) {
#pragma unroll
        for (int i = 0; i < N2; ++i) {
          const float2 v = split_f32x2(acc[i]);
          store_token<T>(p.a, m0 + 2 * i, n, v.x, bias);
          store_token<T>(p.a, m0 + 2 * i + 1, n, v.y, bias);
        }
      }
    }
  }

  if (p.splits > 1) {
    // Partial tiles in the (drained) stages; column chunks of 8 are summed by share chunk mod
    // splits, over the shares in order.
    if (warp >= 4) {
#pragma unroll
      for (int i = 0; i < N2 / 2; ++i) {
        const float2 f = split_f32x2(acc[2 * i]), g = split_f32x2(acc[2 * i + 1]);
        *reinterpret_cast<float4*>(smem + part_at(row, i)) =
            make_float4(f.x, f.y, g.x, g.y);
      }
    }
    __syncwarp();
    cluster_barrier();
    if (warp >= 4) {
      for (int c = share; c < kCols / 8; c += p.splits) {
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int k = 0; k < p.splits; ++k) {
          const uint32_t at = map_to_rank(smem_u32(smem), k);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float4 w = ld_cluster_v4(at + part_at(row, 2 * c + e));
            v[4 * e] += w.x;
            v[4 * e + 1] += w.y;
            v[4 * e + 2] += w.z;
            v[4 * e + 3] += w.w;
          }
        }
        if (n < p.a.N) {
#pragma unroll
          for (int e = 0; e < 8; ++e) store_token<T>(p.a, m0 + 8 * c + e, n, v[e], bias);
        }
      }
    }
    __syncwarp();
    cluster_barrier();  // no CTA leaves while a peer reads its shared memory
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

using TcKernel = void (*)(CUtensorMap, CUtensorMap, CUtensorMap, TcArgs);

cudaLaunchConfig_t tc_config(unsigned grid, int threads, int smem, int cluster, cudaStream_t stream,
                             cudaLaunchAttribute (&attr)[2]) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = stream;
  cfg.attrs = attr;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = 2;
  return cfg;
}

// What one kernel needs once per device: its shared-memory limit raised, and how many clusters of
// each size are resident at once (a GPC holds whole clusters only, so it is not SMs / size).
struct TcDevice {
  std::atomic<int> ready{0};
  std::mutex mu;
  int clusters[9] = {};  // [cluster size]
};

int tc_prepare(TcDevice& d, TcKernel kernel, int threads, int smem, int base) {
  if (d.ready.load(std::memory_order_acquire)) return TF_OK;
  std::lock_guard<std::mutex> lock(d.mu);
  if (d.ready.load(std::memory_order_relaxed)) return TF_OK;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  for (int c = base; c <= 8 && e == cudaSuccess; c += base) {
    cudaLaunchAttribute attr[2];
    const cudaLaunchConfig_t cfg =
        tc_config(static_cast<unsigned>(c), threads, smem, c, nullptr, attr);
    e = cudaOccupancyMaxActiveClusters(&d.clusters[c], kernel, &cfg);
  }
  if (e != cudaSuccess) return cuda_failed(e);
  d.ready.store(1, std::memory_order_release);
  return TF_OK;
}

// Estimated time of a launch in ns, fitted to measurements of 1 to 148 blocks of K on this GPU: a
// fixed part (launch, set-up, first bytes from HBM, output of the last tile), the exchange of a
// split, a time per block of the busiest cluster, and one per tile of it after the first (the tile's
// output, and the ring and the sums starting anew).
struct TcCost {
  int fixed, exchange, block, tile;
};

struct TcSplit {
  int splits;
  int64_t ns;
};

// `base`: CTAs that share a tile and a share of K (2 for the pair kernel). The K split with the
// least estimated time; the clusters of a split launch must all be resident at once.
TcSplit tc_split(const TcDevice& d, int base, const TcCost& c, const TcArgs& p) {
  const int64_t tiles = static_cast<int64_t>(p.tok_tiles) * p.w_tiles;
  const int64_t waves = cdiv(tiles, std::max(1, d.clusters[base]));
  TcSplit best{1, c.fixed + waves * p.kb_total * c.block + (waves - 1) * c.tile};
  for (int s = 2; s * base <= 8 && s <= p.kb_total && tiles <= d.clusters[s * base]; ++s) {
    const int64_t ns = c.fixed + c.exchange + cdiv(p.kb_total, s) * c.block;
    if (ns < best.ns) best = TcSplit{s, ns};
  }
  return best;
}

int tc_launch(const TcDevice& d, TcKernel kernel, int threads, int smem, int base,
              const CUtensorMap (&maps)[3], const TcArgs& p, cudaStream_t stream) {
  const int64_t tiles = static_cast<int64_t>(p.tok_tiles) * p.w_tiles;
  const int64_t clusters = p.splits > 1 ? tiles : std::min<int64_t>(tiles, d.clusters[base]);
  cudaLaunchAttribute attr[2];
  const cudaLaunchConfig_t cfg =
      tc_config(static_cast<unsigned>(clusters * base * p.splits), threads, smem,
                base * p.splits, stream, attr);
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, maps[0], maps[1], maps[2], p);
  if (e != cudaSuccess) return cuda_failed(e);
  return TF_OK;
}

bool make_out_map(CUtensorMap* map, const W8A8Args& a, int box_rows, int box_cols) {
  auto fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(a.N), static_cast<cuuint64_t>(a.M)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(a.ldy) * 2};
  cuuint32_t box[2] = {static_cast<cuuint32_t>(box_cols), static_cast<cuuint32_t>(box_rows)};
  cuuint32_t estr[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, a.y, dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr int kMaxDevices = 64;

int current_device(int* dev) {
  const cudaError_t e = cudaGetDevice(dev);
  if (e != cudaSuccess) return cuda_failed(e);
  return *dev < kMaxDevices ? TF_OK : TF_ERR_UNSUPPORTED;
}

bool tile_counts(const W8A8Args& a, int tokens, int rows, TcArgs* p) {
  const int64_t tt = cdiv(a.M, tokens), wt = cdiv(a.N, rows);
  p->a = a;
  p->kb_total = static_cast<int>(cdiv(a.K, kBlockK));
  p->tok_tiles = static_cast<int>(tt);
  p->w_tiles = static_cast<int>(wt);
  p->vec_scales = aligned16(a.x_scale) && a.ld_xs % 4 == 0;
  return tt * wt < 0x7fffffffLL;
}

// A kernel form: its tile counts and K split for these operands on this device, and its launch.
template <typename T>
struct PairForm {
  static constexpr TcCost kCost{5400, 4600, 420, 1600};
  TcDevice* device;
  TcArgs p;
  int64_t ns;

  int plan(const W8A8Args& a, int dev) {
    static TcDevice devices[kMaxDevices];
    device = &devices[dev];
    const int st = tc_prepare(*device, w8a8_pair_kernel<T>, Pair::kThreads, Pair::kSmem, 2);
    if (st != TF_OK) return st;
    if (!tile_counts(a, Pair::kTokens, Pair::kCols, &p)) return TF_ERR_TOO_LARGE;
    const TcSplit s = tc_split(*device, 2, kCost, p);
    p.splits = s.splits;
    ns = s.ns;
    return TF_OK;
  }
  int launch(const W8A8Args& a, cudaStream_t stream) {
    CUtensorMap maps[3];
    if (!make_map(&maps[0], a.xq, a.K, a.M, a.ldx, kLanes) ||
        !make_map(&maps[1], a.wq, a.K, a.N, a.K, Pair::kCols / 2))
      return TF_ERR_ALIGNMENT;
    // The output goes through TMA where its rows allow it, else by plain stores.
    p.tma_out = aligned16(a.y) && a.ldy % 8 == 0;
    maps[2] = maps[0];
    if (p.tma_out && !make_out_map(&maps[2], a, 32, Pair::kOutCols)) return TF_ERR_ALIGNMENT;
    return tc_launch(*device, w8a8_pair_kernel<T>, Pair::kThreads, Pair::kSmem, 2, maps, p,
                     stream);
  }
};

template <int kCols, typename T>
struct SwapForm {
  static constexpr TcCost kCost{4500, 2000, kCols == 64 ? 380 : 300, 2500};
  TcDevice* device;
  TcArgs p;
  int64_t ns;

  int plan(const W8A8Args& a, int dev) {
    using C = Swap<kCols>;
    static TcDevice devices[kMaxDevices];
    device = &devices[dev];
    const int st = tc_prepare(*device, w8a8_swap_kernel<kCols, T>, C::kThreads, C::kSmem, 1);
    if (st != TF_OK) return st;
    if (!tile_counts(a, kCols, kLanes, &p)) return TF_ERR_TOO_LARGE;
    const TcSplit s = tc_split(*device, 1, kCost, p);
    p.splits = s.splits;
    ns = s.ns;
    return TF_OK;
  }
  int launch(const W8A8Args& a, cudaStream_t stream) {
    using C = Swap<kCols>;
    CUtensorMap maps[3];
    if (!make_map(&maps[0], a.wq, a.K, a.N, a.K, kLanes) ||
        !make_map(&maps[1], a.xq, a.K, a.M, a.ldx, kCols))
      return TF_ERR_ALIGNMENT;
    maps[2] = maps[0];  // unused: an output row's 32 neighbours are one plain store
    p.tma_out = 0;
    return tc_launch(*device, w8a8_swap_kernel<kCols, T>, C::kThreads, C::kSmem, 1, maps, p,
                     stream);
  }
};

template <typename Form>
int run_form(const W8A8Args& a, int dev, cudaStream_t stream) {
  Form f;
  const int st = f.plan(a, dev);
  return st == TF_OK ? f.launch(a, stream) : st;
}

// Up to 64 tokens: one token tile with weight rows as lanes. Above, up to 512: whichever of the
// two forms is estimated faster; 64-token tiles fill more SMs and start sooner, pairs read the
// weights once (128 tokens: 3584 x 3584 11.4 against 13.3 us, 37888 x 3584 50 against 36, 37888 x
// 128 14.8 against 8.5). Of 231 products of 72 to 512 tokens, 512 to 37888 rows and K of 128 to
// 18944, the one it takes is at most 9 % slower than the other. Without the time per tile
// it took 64-token tiles that were up to 1.9 times slower where K is 128 or 256.
template <typename T>
int launch_tc(const W8A8Args& a, cudaStream_t stream) {
  int dev = 0;
  int st = current_device(&dev);
  if (st != TF_OK) return st;
  if (a.M <= 16) return run_form<SwapForm<16, T>>(a, dev, stream);
  if (a.M <= 32) return run_form<SwapForm<32, T>>(a, dev, stream);
  if (a.M <= 64) return run_form<SwapForm<64, T>>(a, dev, stream);
  PairForm<T> pair;
  st = pair.plan(a, dev);
  if (st != TF_OK) return st;
  if (a.M <= 512) {
    SwapForm<64, T> swap;
    st = swap.plan(a, dev);
    if (st != TF_OK) return st;
    if (swap.ns < pair.ns) return swap.launch(a, stream);
  }
  return pair.launch(a, stream);
}

}  // namespace

int launch_w8a8_tc(const W8A8Args& a, cudaStream_t stream) {
  return a.dtype == TF_DTYPE_FP16 ? launch_tc<__half>(a, stream)
                                  : launch_tc<__nv_bfloat16>(a, stream);
}

int w8a8_device_error(int* code) {
  const cudaError_t e = cudaMemcpyFromSymbol(code, g_w8a8_error, sizeof(int));
  if (e != cudaSuccess) return cuda_failed(e);
  return TF_OK;
}

int w8a8_reset_device_error() {
  const int zero = 0;
  const cudaError_t e = cudaMemcpyToSymbol(g_w8a8_error, &zero, sizeof(int));
  if (e != cudaSuccess) return cuda_failed(e);
  return TF_OK;
}

}  // namespace tfb
