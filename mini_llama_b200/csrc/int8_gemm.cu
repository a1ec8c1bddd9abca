// int8_gemm.cu — product of int8 rows with a scale for each token and each channel, on
// the tcgen05 tensor cores.
//
//   y[m, n] = (sum_k x[m, k] w[n, k]) sx[m] sw[n] + bias[n]
//
// Sums are exact in 32-bit integers (131071 products of two codes of at most 128 are
// below 2^31), in any order: a row's result does not depend on the rows beside it, on
// how the work is split or on the run. Then three fp32 steps, each rounded once, and
// one rounding to bf16 where that is asked for.
//
// Few tokens (int8_linear_kernel): a CTA takes 128 channels by NT tokens and a share of K.
// One warp loads tiles of 128 bytes along K by TMA (what lies past the matrices' edges
// arrives as zeros) into a ring, one issues the products, channels as the rows of D, so
// that few tokens fill the tensor cores' other side and a warp stores consecutive
// channels. Where the tiles alone leave SMs idle, a cluster of CTAs shares K; each pushes
// its sums to the CTA that owns their tokens and goes: no workspace, one launch. Bound by
// HBM (the weights are read once) behind the start of the stream: one row of 4096 x 4096
// 4.6 us, 5.0 with weights that L2 does not hold, of 4096 x 28672 21.2 (5.5 TB/s), 32 of 8192
// x 10240 14.4 and 18.7 (4.5 TB/s).
//
// Many tokens (int8_linear_pair_kernel): pairs of CTAs, 256 tokens by up to 256 channels.
// Bound by the tensor cores: 4096 x 4096 x 28672 279 to 293 us (3290 to 3450 TOPS, twice the
// measured bf16 rate; in a long run the power cap, 2800), 512 of 4096 x 4096 11.2.
//
// Every wait for a copy, a product or another CTA's sums is bounded: on a timeout the
// waiting thread records MLB_ERR_TIMEOUT in the device's status word
// (mlb_int8_linear_status) and raises the CTA's abort flag, copies and products in flight
// are waited for (bounded), the results of the cluster's tile become NaN, tensor memory is
// released and the CTA exits. Three waits have no limit of their own, as what they wait for
// ends without this CTA. The kernel before on the stream (pdl_wait). The cluster's other CTAs
// at its barriers, which they reach behind bounded waits or the third kind. Tensor memory:
// whoever holds some on this SM releases it without waiting for another CTA to get any. A CTA
// alone (one share of K, or another kernel of this library) waits for no CTA; those of a
// cluster that shares K take 128 of the 512 columns at most and shared memory for no more
// than two on an SM; a pair's CTA leaves no shared memory for any that takes tensor memory
// (asserted below).
#include <cuda.h>
#include <cuda_bf16.h>

#include <algorithm>
#include <type_traits>

#include "paged.cuh"
#include "runtime.cuh"
#include "rows.cuh"
#include "tcgen05.cuh"

namespace mlb {

namespace {

constexpr int kThreads = 128;
constexpr int kTileK = 128;      // bytes along K of a tile
constexpr int kChannels = 128;   // channels of a CTA
constexpr int kMaxStages = 8;
constexpr int kHalf = 110 * 1024;  // shared memory of a CTA where two share an SM
constexpr int kMaxSplit = 8;
constexpr int kMaxK = 131071;
constexpr long long kWaitCycles = 2000000000LL;  // about 1 s

__device__ DeviceStatus g_status;

struct LinearArgs {
  const float* x_scale;
  const float* w_scale;
  const float* bias;
  void* out;
  long long out_stride;
  int rows, n, tiles_k, channel_tiles, stages;
  int ahead;             // tiles of weights that a CTA asks for before its turn
  int split, log_split;  // CTAs that share K, a power of two
  long long wait_cycles;  // limit of a wait
  int never;              // arrivals that the first barrier waits for in vain (self-test)
};

struct Shared {
  uint64_t full[kMaxStages], empty[kMaxStages], done, joined, drain;
  int abort_flag;
  uint32_t tmem;
  float x_scale[128];
  alignas(16) float w_scale[kChannels];
  alignas(16) float bias[kChannels];
};

// A barrier of some warps; arriving at it without waiting.
__device__ __forceinline__ void barrier_sync(int id, int threads) {
  asm volatile("barrier.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ void barrier_arrive(int id, int threads) {
  asm volatile("barrier.arrive %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

__device__ __forceinline__ bool wait(Shared& sh, const LinearArgs& a, uint64_t* bar,
                                     uint32_t parity, int where) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long start = clock64();
  while (!mbar_try_wait(bar, parity)) {
    if (*(volatile int*)&sh.abort_flag) return false;
    if (clock64() - start > a.wait_cycles) {
      atomicExch(&g_status.code, MLB_ERR_TIMEOUT);
      atomicExch(&g_status.where, where);
      *(volatile int*)&sh.abort_flag = 1;
      return false;
    }
  }
  return true;
}
// The wait for the other shares' sums.
__device__ __forceinline__ bool wait_joined(Shared& sh, const LinearArgs& a) {
  if (mbar_try_wait_cluster(&sh.joined, 0)) return true;
  const long long start = clock64();
  while (!mbar_try_wait_cluster(&sh.joined, 0)) {
    if (clock64() - start > a.wait_cycles) {
      atomicExch(&g_status.code, MLB_ERR_TIMEOUT);
      atomicExch(&g_status.where, 1104);
      return false;
    }
  }
  return true;
}
// The last wait for what is in flight, after which there is nothing more to be done.
__device__ __forceinline__ void drain_wait(const LinearArgs& a, uint64_t* bar, uint32_t parity) {
  const long long start = clock64();
  while (!mbar_try_wait(bar, parity) && clock64() - start < a.wait_cycles) {
  }
}

__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void put4(float* p, const float4& v) {
  *reinterpret_cast<float4*>(p) = v;
}
__device__ __forceinline__ void put4(__nv_bfloat16* p, const float4& v) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
}

// A sum with its scales and bias: three roundings, two without a bias.
__device__ __forceinline__ float scaled(int sum, float sx, float sw, float bias, bool biased) {
  const float y = (float)sum * sx;
  return biased ? fmaf(y, sw, bias) : y * sw;
}

// After a wait that gave up: the time that what others have on its way here takes at most.
__device__ __forceinline__ void settle() {
  const long long start = clock64();
  while (clock64() - start < 2000000) {  // 1 ms
  }
}

// Grid: ((token tile * channel tiles) + channel tile) * split + share of K, the shares of
// a tile being a cluster.
template <int NT, class T>
__global__ void __launch_bounds__(kThreads)
    int8_linear_kernel(const __grid_constant__ CUtensorMap w_map,
                       const __grid_constant__ CUtensorMap x_map, const LinearArgs a) {
  constexpr int COLS = NT < 32 ? 32 : NT;
  constexpr int W_BYTES = kChannels * kTileK, X_BYTES = NT * kTileK;
  constexpr int STAGE = W_BYTES + X_BYTES;
  extern __shared__ uint8_t dynamic[];
  __shared__ Shared sh;
  uint8_t* smem = dynamic + (-smem_addr(dynamic) & 1023u);
  const int warp = threadIdx.x >> 5;
  const int share = blockIdx.x & (a.split - 1), tile = blockIdx.x >> a.log_split;
  const int token_tile = tile / a.channel_tiles;
  const int channel0 = (tile - token_tile * a.channel_tiles) * kChannels;
  const int token0 = token_tile * NT;
  // the CTA's tiles along K; a share has one at least
  const int k0 = a.tiles_k * share >> a.log_split;
  const int count = (a.tiles_k * (share + 1) >> a.log_split) - k0;
  // groups of four tokens share, share + split .. are joined here
  const int tokens = min(NT, a.rows - token0);
  const int owned = ((tokens + 3) / 4 - share + a.split - 1) >> a.log_split;

  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    prefetch_map(&w_map);
    prefetch_map(&x_map);
    for (int i = 0; i < a.stages; ++i) {
      mbar_init(&sh.full[i], 1 + a.never);
      mbar_init(&sh.empty[i], 1);
    }
    mbar_init(&sh.done, 1);
    mbar_init(&sh.joined, 1);
    mbar_init(&sh.drain, 1);
    sh.abort_flag = 0;
    fence_mbar_init();
    // what the other shares of this CTA's tokens come to
    if (a.split > 1)
      mbar_arrive_expect_tx(&sh.joined, (uint32_t)(owned * (a.split - 1)) * kChannels * 16);
  }
  if (a.split > 1) cluster_arrive();
  // weights on their way to L2 while the kernel before still runs: what that one may write
  // there is read all the same, as L2 is where every SM's stores come together
  if (warp == 3)
    for (int i = 0; i < min(count, a.ahead); ++i)
      if (elect_one()) tma_prefetch(&w_map, (k0 + i) * kTileK, channel0);
  // The kernel before may have made what is read from here on; and no CTA keeps tensor
  // memory that another one of that kernel might need while it waits for its end.
  pdl_wait();
  // loads need no tensor memory: their warp does not wait for it
  if (warp == 0) {
    __syncwarp();  // the barriers are its first lane's work
    barrier_arrive(2, kThreads);
  } else {
    if (warp == 1) {
      tmem_alloc(&sh.tmem, COLS);
      tmem_relinquish();
    }
    tc_fence_before();
    barrier_sync(2, kThreads);
    tc_fence_after();
  }

  // Loads and products are a whole warp's loops of uniform values, of which one lane
  // issues: as one lane's loops they took 600 cycles a tile of K, more than its copies.
  int issued = 0;
  if (warp == 0) {
    int s = 0, x = k0 * kTileK;
    uint32_t phase = 1;  // the first turn waits for nothing
    for (; issued < count; ++issued, x += kTileK) {
      if (issued >= a.stages &&
          !__all_sync(0xffffffffu, wait(sh, a, &sh.empty[s], phase, 1101)))
        break;
      if (elect_one()) {
        uint8_t* stage = smem + s * STAGE;
        mbar_arrive_expect_tx(&sh.full[s], STAGE);
        tma_load(stage, &w_map, x, channel0, &sh.full[s]);
        tma_load(stage + W_BYTES, &x_map, x, token0, &sh.full[s]);
      }
      __syncwarp();
      if (++s == a.stages) s = 0, phase ^= 1u;
    }
  } else if (warp == 1) {
    const uint32_t idesc = idesc_i8(kChannels, NT), tmem = sh.tmem;
    const uint64_t ring = smem_desc_sw128(smem_addr(smem));
    int s = 0;
    uint32_t phase = 0;
    for (int i = 0; i < count; ++i) {
      if (!__all_sync(0xffffffffu, wait(sh, a, &sh.full[s], phase, 1102))) break;
      tc_fence_after();
      const uint64_t w = ring + (uint32_t)(s * STAGE >> 4), x = w + (W_BYTES >> 4);
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < kTileK / 32; ++k)
          tc_mma_i8(tmem, w + 2 * k, x + 2 * k, idesc, i > 0 || k > 0);
        tc_commit(&sh.empty[s]);
        if (i == count - 1) tc_commit(&sh.done);
      }
      __syncwarp();
      if (++s == a.stages) s = 0, phase ^= 1u;
    }
  }
  __syncwarp();
  const bool biased = a.bias != nullptr;
  if (warp >= 2) {  // what the results are multiplied with, while the products run
    for (int i = threadIdx.x - 64; i < kChannels; i += kThreads - 64) {
      const bool there = channel0 + i < a.n;
      sh.w_scale[i] = there ? a.w_scale[channel0 + i] : 0.0f;
      sh.bias[i] = there && biased ? a.bias[channel0 + i] : 0.0f;
      if (i < NT) sh.x_scale[i] = i < tokens ? a.x_scale[token0 + i] : 0.0f;
    }
  }
  bool ok = __syncthreads_and(wait(sh, a, &sh.done, 0, 1103));
  if (!ok) {
    // nothing is in flight when shared and tensor memory go
    if (threadIdx.x == 0)
      for (int j = max(0, issued - a.stages); j < issued; ++j)
        drain_wait(a, &sh.full[j % a.stages], (uint32_t)(j / a.stages) & 1u);
    if (warp == 1 && elect_one()) {
      tc_commit(&sh.drain);
      drain_wait(a, &sh.drain, 0);
    }
    __syncthreads();
  }
  tc_fence_after();

  T* out = static_cast<T*>(a.out) + (long long)token0 * a.out_stride + channel0;
  const uint32_t lanes = sh.tmem + ((uint32_t)(warp * 32) << 16);
  const int c = threadIdx.x;
  const bool inside = channel0 + c < a.n;
  const float bias = sh.bias[c];
  if (a.split == 1) {
    const float sw = ok ? sh.w_scale[c] : nanf("");
#pragma unroll 1
    for (int t0 = 0; t0 < tokens; t0 += 16) {
      uint32_t d[16];
      tmem_ld16(lanes + t0, d);
      float y[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) y[i] = scaled((int)d[i], sh.x_scale[t0 + i], sw, bias, biased);
      T* o = out + t0 * a.out_stride + c;
#pragma unroll
      for (int i = 0; i < 16; ++i, o += a.out_stride)
        if (inside && t0 + i < tokens) put(o, y[i]);
    }
  } else {
    // every share's sums go to their tokens' owner, behind its ring, as [group][share]
    // [channel][token]: a thread has four tokens of a channel, a warp 512 bytes
    int4* sums = reinterpret_cast<int4*>(smem + a.stages * STAGE);
    cluster_wait();  // every CTA's barrier is there
    if (ok) {
#pragma unroll 1
      for (int t0 = 0; t0 < tokens; t0 += 16) {
        uint32_t d[16];
        tmem_ld16(lanes + t0, d);
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          if (t0 + i < tokens) {
            const int group = (t0 + i) / 4, owner = group & (a.split - 1);
            int4* to = sums + (group - owner + share) * kChannels + c;
            if (owner == share)
              *to = make_int4((int)d[i], (int)d[i + 1], (int)d[i + 2], (int)d[i + 3]);
            else
              st_async4(cluster_address(to, owner), d[i], d[i + 1], d[i + 2], d[i + 3],
                        cluster_address(&sh.joined, owner));
          }
        }
      }
    }
    if (owned > 0) ok = __syncthreads_and(ok && wait_joined(sh, a));
    const float sw = ok ? sh.w_scale[c] : nanf("");
    const auto finish = [&](auto split) {
      constexpr int S = decltype(split)::value, AT_ONCE = S > 4 ? 1 : 2;
#pragma unroll 1
      for (int g0 = 0; g0 < owned; g0 += AT_ONCE) {
        int4 v[AT_ONCE][S];
#pragma unroll
        for (int g = 0; g < AT_ONCE; ++g)
#pragma unroll
          for (int r = 0; r < S; ++r)
            v[g][r] = sums[(min(g0 + g, owned - 1) * S + r) * kChannels + c];
#pragma unroll
        for (int g = 0; g < AT_ONCE; ++g) {
          int sum[4] = {0, 0, 0, 0};
#pragma unroll
          for (int r = 0; r < S; ++r)
            sum[0] += v[g][r].x, sum[1] += v[g][r].y, sum[2] += v[g][r].z, sum[3] += v[g][r].w;
          const int t = ((g0 + g) * S + share) * 4;
          T* o = out + t * a.out_stride + c;
#pragma unroll
          for (int i = 0; i < 4; ++i, o += a.out_stride)
            if (inside && t + i < tokens)
              put(o, scaled(sum[i], sh.x_scale[t + i], sw, bias, biased));
        }
      }
    };
    if (a.split == 2)
      finish(std::integral_constant<int, 2>());
    else if (a.split == 4)
      finish(std::integral_constant<int, 4>());
    else
      finish(std::integral_constant<int, 8>());
    // a CTA whose sums have all arrived may go; another one waits until no CTA sends any
    // more (those that have gone count as there), and for what they have sent
    if (!ok) {
      cluster_sync_all();
      settle();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(sh.tmem, COLS);
  }
}

// ------------------------------------------------------------ many tokens
// A pair of CTAs takes 256 tokens by N channels at a time, tokens as the rows of D: each
// CTA loads its 128 tokens and half of the channels, and the tensor cores of both read
// both halves. Two accumulators in tensor memory: the products of a tile run while the
// one before is turned in shared memory, scaled and stored, 32 channels of a row at once.
// Pairs take tiles in turn, tokens first in groups of kGroup tiles, so that the pairs at
// work share few tiles of either matrix in L2.
//
// Roles (6 warps): 0 loads, 1 tensor memory and (first CTA) products, 2..5 epilogue.

constexpr int kPairThreads = 192;
constexpr int kPairTokens = 256;
constexpr int kGroup = 16;
constexpr int kMaxPairStages = 10;
constexpr int kTurnWords = 36;  // a row of 32 words, its 16-byte pieces in unlike banks

struct PairShared {
  uint64_t full[kMaxPairStages], empty[kMaxPairStages], sum_full[2], sum_empty[2], drain;
  int abort_flag;
  uint32_t tmem;
  alignas(16) float scale[2][256];
  alignas(16) float bias[2][256];
};

template <int N>
struct PairPlan {
  static constexpr int A = 128 * kTileK, B = N / 2 * kTileK;
  static constexpr int STAGE = A + B;
  static constexpr int TURN = 32 * kTurnWords * 4;  // per epilogue warp
  // as many as there is room for: a tile of K is about 1.5 us on its way
  static constexpr int STAGES = std::min<int>(
      kMaxPairStages, (227 * 1024 - (int)sizeof(PairShared) - 1024 - 4 * TURN) / STAGE);
  static constexpr int BYTES = STAGES * STAGE + 4 * TURN + 1024;
};

__device__ __forceinline__ bool wait_pair(PairShared& sh, const LinearArgs& a, uint64_t* bar,
                                          uint32_t parity, int where) {
  if (mbar_try_wait_cluster(bar, parity)) return true;
  const long long start = clock64();
  while (!mbar_try_wait_cluster(bar, parity)) {
    if (*(volatile int*)&sh.abort_flag) return false;
    if (clock64() - start > a.wait_cycles) {
      atomicExch(&g_status.code, MLB_ERR_TIMEOUT);
      atomicExch(&g_status.where, where);
      *(volatile int*)&sh.abort_flag = 1;
      return false;
    }
  }
  return true;
}

template <int N, class T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    int8_linear_pair_kernel(const __grid_constant__ CUtensorMap x_map,
                            const __grid_constant__ CUtensorMap w_map, const LinearArgs a) {
  using P = PairPlan<N>;
  extern __shared__ uint8_t dynamic[];
  __shared__ PairShared sh;
  uint8_t* smem = dynamic + (-smem_addr(dynamic) & 1023u);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = blockIdx.x & 1, pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int token_tiles = (a.rows + kPairTokens - 1) / kPairTokens;
  const int tiles = token_tiles * a.channel_tiles;
  const auto place = [&](int tile, int& token0, int& channel0) {
    const int group = tile / (kGroup * a.channel_tiles);
    const int in_group = min(kGroup, token_tiles - group * kGroup);
    const int r = tile - group * kGroup * a.channel_tiles;
    channel0 = r / in_group * N;
    token0 = (group * kGroup + r % in_group) * kPairTokens + rank * 128;
  };

  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    prefetch_map(&x_map);
    prefetch_map(&w_map);
    for (int i = 0; i < P::STAGES; ++i) {
      mbar_init(&sh.full[i], 1 + a.never);
      mbar_init(&sh.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.sum_full[i], 1);
      mbar_init(&sh.sum_empty[i], 8);  // four warps of each CTA
    }
    mbar_init(&sh.drain, 1);
    sh.abort_flag = 0;
    fence_mbar_init();
  }
  pdl_wait();  // before tensor memory is taken, as above
  if (warp == 1) {
    tmem_alloc_pair(&sh.tmem, 2 * N);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // the other CTA's barriers are there
  tc_fence_after();
  const uint32_t tmem = sh.tmem;

  int issued = 0;
  if (warp == 0) {
    int s = 0;
    uint32_t phase = 1;
    bool ok = true;
    // the first CTA's barriers count the bytes of both
    const uint32_t full = cluster_address(&sh.full[0], 0);
    for (int tile = pair; ok && tile < tiles; tile += pairs) {
      int token0, channel0;
      place(tile, token0, channel0);
      channel0 += rank * (N / 2);
      for (int k = 0; k < a.tiles_k; ++k, ++issued) {
        if (issued >= P::STAGES) {
          ok = __all_sync(0xffffffffu, wait_pair(sh, a, &sh.empty[s], phase, 1111));
          if (!ok) break;
        }
        if (elect_one()) {
          if (rank == 0) mbar_arrive_expect_tx(&sh.full[s], 2 * P::STAGE);
          uint8_t* stage = smem + s * P::STAGE;
          tma_load_pair(stage, &x_map, k * kTileK, token0, full + s * 8);
          tma_load_pair(stage + P::A, &w_map, k * kTileK, channel0, full + s * 8);
        }
        __syncwarp();
        if (++s == P::STAGES) s = 0, phase ^= 1u;
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      const uint32_t idesc = idesc_i8(kPairTokens, N);
      const uint64_t ring = smem_desc_sw128(smem_addr(smem));
      int s = 0, done = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = pair; ok && tile < tiles; tile += pairs, ++done) {
        const int b = done & 1, turn = done >> 1;
        if (turn > 0) ok = wait_pair(sh, a, &sh.sum_empty[b], (uint32_t)(turn - 1) & 1u, 1112);
        if (!__all_sync(0xffffffffu, ok)) break;
        tc_fence_after();
        for (int k = 0; k < a.tiles_k; ++k) {
          ok = __all_sync(0xffffffffu, wait_pair(sh, a, &sh.full[s], phase, 1113));
          if (!ok) break;
          tc_fence_after();
          const uint64_t x = ring + (uint32_t)(s * P::STAGE >> 4), w = x + (P::A >> 4);
          if (elect_one()) {
#pragma unroll
            for (int j = 0; j < kTileK / 32; ++j)
              tc_mma_i8_pair(tmem + b * N, x + 2 * j, w + 2 * j, idesc, k > 0 || j > 0);
            tc_commit_pair(&sh.empty[s]);
          }
          __syncwarp();
          if (++s == P::STAGES) s = 0, phase ^= 1u;
        }
        if (ok && elect_one()) tc_commit_pair(&sh.sum_full[b]);
        __syncwarp();
      }
    }
  } else {
    const int quarter = warp & 3, thread = threadIdx.x - 64;
    int* turn_buf = reinterpret_cast<int*>(smem + P::STAGES * P::STAGE) +
                      quarter * 32 * kTurnWords;
    // when sums are turned, a lane has four channels of every fourth row
    const int c4 = lane % 8 * 4, r4 = lane / 8;
    const bool wide = reinterpret_cast<uintptr_t>(a.out) % (4 * sizeof(T)) == 0 &&
                      a.out_stride % 4 == 0;
    const bool biased = a.bias != nullptr;
    bool ok = true;
    int done = 0;
    for (int tile = pair; tile < tiles; tile += pairs, ++done) {
      int token0, channel0;
      place(tile, token0, channel0);
      const int b = done & 1;
      token0 += quarter * 32;
      // the tile's scales and biases, while its products run; the warps are at most a
      // tile apart, so the buffer of the tile before the last is free
      for (int c = thread; c < N; c += 128) {
        const bool inside = channel0 + c < a.n;
        sh.scale[b][c] = inside ? a.w_scale[channel0 + c] : 0.0f;
        sh.bias[b][c] = inside && biased ? a.bias[channel0 + c] : 0.0f;
      }
      float sx[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        sx[i] = token0 + 4 * i + r4 < a.rows ? a.x_scale[token0 + 4 * i + r4] : 0.0f;
      asm volatile("bar.sync 1, 128;" ::: "memory");
      ok = __all_sync(0xffffffffu,
                      ok && wait_pair(sh, a, &sh.sum_full[b], (uint32_t)(done >> 1) & 1u, 1114));
      tc_fence_after();
      if (!ok) {
#pragma unroll
        for (int i = 0; i < 8; ++i) sx[i] = nanf("");
      }
      const uint32_t sums = tmem + b * N + ((uint32_t)(quarter * 32) << 16);
      const int columns = min(N, (a.n - channel0 + 31) / 32 * 32);
      T* out = static_cast<T*>(a.out) + (long long)token0 * a.out_stride + channel0 + c4;
      const int rows = a.rows - token0;
      uint32_t d[32];
      tmem_ld32_start(sums, d);
#pragma unroll 1
      for (int c0 = 0; c0 < columns; c0 += 32) {
        tmem_ld32_wait(d);
#pragma unroll
        for (int j = 0; j < 32; j += 4)
          *reinterpret_cast<uint4*>(turn_buf + lane * kTurnWords + j) =
              make_uint4(d[j], d[j + 1], d[j + 2], d[j + 3]);
        if (c0 + 32 < columns) {
          tmem_ld32_start(sums + c0 + 32, d);
        } else {  // that was the last read of these sums
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(cluster_address(&sh.sum_empty[b], 0));
        }
        __syncwarp();
        const float4 s = *reinterpret_cast<const float4*>(&sh.scale[b][c0 + c4]);
        const float4 z = *reinterpret_cast<const float4*>(&sh.bias[b][c0 + c4]);
        int4 v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          v[i] = *reinterpret_cast<const int4*>(turn_buf + (4 * i + r4) * kTurnWords + c4);
        float4 y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          y[i] = make_float4(
              scaled(v[i].x, sx[i], s.x, z.x, biased), scaled(v[i].y, sx[i], s.y, z.y, biased),
              scaled(v[i].z, sx[i], s.z, z.z, biased), scaled(v[i].w, sx[i], s.w, z.w, biased));
        T* o = out + r4 * a.out_stride + c0;
        if (wide && rows >= 32 && channel0 + c0 + 32 <= a.n) {
#pragma unroll
          for (int i = 0; i < 8; ++i, o += 4 * a.out_stride) put4(o, y[i]);
        } else {
          const int left = a.n - channel0 - c0 - c4;
#pragma unroll
          for (int i = 0; i < 8; ++i, o += 4 * a.out_stride) {
            const float e[4] = {y[i].x, y[i].y, y[i].z, y[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (4 * i + r4 < rows && j < left) put(o + j, e[j]);
          }
        }
        __syncwarp();
      }
    }
  }

  __syncwarp();
  __syncthreads();
  if (*(volatile int*)&sh.abort_flag) {
    // nothing is in flight when shared and tensor memory go; the second CTA's copies are
    // counted by the first alone, so it gives them time
    if (rank == 0 && threadIdx.x == 0)
      for (int j = max(0, issued - P::STAGES); j < issued; ++j)
        drain_wait(a, &sh.full[j % P::STAGES], (uint32_t)(j / P::STAGES) & 1u);
    if (rank == 0 && warp == 1 && elect_one()) {
      tc_commit_pair(&sh.drain);
      drain_wait(a, &sh.drain, 0);
    }
    if (rank == 1 && threadIdx.x == 0) settle();
    __syncthreads();
  }
  tc_fence_before();
  cluster_sync_all();  // neither CTA's memory goes while the other one's products read it
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 2 * N);
  }
}

// ------------------------------------------------------------------ host side

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                 const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
  static const EncodeTiled f = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    MLB_CUDA(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found));
    if (found != cudaDriverEntryPointSuccess || !p)
      fail(MLB_ERR_CUDA, "Int8Linear: the driver has no tensor maps");
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return f;
}

// Tiles of 128 bytes by `box_rows` of a byte matrix; past its edges lie zeros.
CUtensorMap tile_map(const void* p, long long stride, int rows, int k, int box_rows) {
  CUtensorMap m;
  const cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)stride};
  const cuuint32_t box[2] = {(cuuint32_t)kTileK, (cuuint32_t)box_rows};
  const cuuint32_t unit[2] = {1, 1};
  const CUresult r = encode_tiled()(
      &m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(p), dims, strides, box, unit,
      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    fail(MLB_ERR_CUDA, "Int8Linear: no tensor map for " + std::to_string(rows) + " rows of " +
                           std::to_string(k) + " (error " + std::to_string((int)r) + ")");
  return m;
}

struct Operands {
  const int8_t* x;
  long long x_stride;
  const int8_t* w;
  long long w_stride;
  int k;
};

// How few tokens (tiles of nt) share K: in a power of two of CTAs (as nt is: groups of
// tokens divide evenly), doubled while the tiles leave room on the SMs and a share keeps
// at least 8 tiles of K (4096 x 4096, 32 tiles, in us with 4 shares of 8, 8 of 4 and 2 of
// 16: one token 4.9, 6.5, 6.7, 32 tokens 5.4, 7.0, 7.7). Two CTAs fit on an SM while the sums
// to be joined leave each a ring of two.
struct FewPlan {
  int split, stages, bytes;
};
FewPlan few_plan(int nt, long long tiles, int tiles_k, int sms) {
  const int stage = (kChannels + nt) * kTileK;
  FewPlan p = {1, 0, 0};
  const auto joined = [&](int split) {
    return split > 1 ? std::max(nt / 4, split) * kChannels * 16 : 0;
  };
  const auto two = [&](int split) { return joined(split) + 2 * stage <= kHalf; };
  while (p.split < kMaxSplit && tiles * p.split * 2 <= (two(p.split * 2) ? 2 : 1) * sms &&
         tiles_k / (p.split * 2) >= 8)
    p.split *= 2;
  const int room = (two(p.split) ? 1 : 2) * kHalf - joined(p.split);
  p.stages = std::min({kMaxStages, (tiles_k + p.split - 1) / p.split, room / stage});
  p.bytes = p.stages * stage + joined(p.split) + 1024;
  return p;
}

template <int NT, class T>
void launch_few(const Operands& o, LinearArgs a, int device_id, cudaStream_t stream) {
  constexpr int kMostBytes = 2 * kHalf + 1024;
  static_assert(NT * kChannels * 4 + (kChannels + NT) * kTileK <= 2 * kHalf);
  static_assert(kMostBytes + sizeof(Shared) <= 227 * 1024);
  a.channel_tiles = (a.n + kChannels - 1) / kChannels;
  const long long tiles = (long long)a.channel_tiles * ((a.rows + NT - 1) / NT);
  const FewPlan p = few_plan(NT, tiles, a.tiles_k, sm_count(device_id));
  a.split = p.split;
  for (a.log_split = 0; 1 << a.log_split < a.split;) ++a.log_split;
  a.stages = p.stages;
  // Four tiles of short shares, whose time is mostly their start (weights beyond L2, in us,
  // with / without: one row of 4096 x 4096, 8 tiles a share, 5.7 / 6.3, behind a norm and with
  // it 8.1 / 8.8, of 14336 x 4096, 14 tiles, 12.3 / 13.2 and 18.5 / 19.3, 32 of 4096 x 4096
  // 6.3 / 6.9 and 9.5 / 10.1); eight kept the norm before waiting. None of long ones: 32 of
  // 8192 x 10240, 32 tiles, 19.8 / 19.0 and 25.0 / 24.4, one of 4096 x 28672 21.9 / 21.6 and
  // 25.1 / 25.1.
  a.ahead = (a.tiles_k + p.split - 1) / p.split <= 16 ? 4 : 0;
  allow_smem(int8_linear_kernel<NT, T>, kMostBytes, device_id);
  if (tiles * a.split > 0x7fffffffLL) invalid("Int8Linear: too many rows");
  const CUtensorMap w_map = tile_map(o.w, o.w_stride, a.n, o.k, kChannels);
  const CUtensorMap x_map = tile_map(o.x, o.x_stride, a.rows, o.k, NT);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * a.split));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (size_t)p.bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)a.split;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = a.split > 1 ? 2 : 1;
  MLB_CUDA(cudaLaunchKernelEx(&cfg, int8_linear_kernel<NT, T>, w_map, x_map, a));
}

template <int N, class T>
void launch_pair(const Operands& o, LinearArgs a, int device_id, cudaStream_t stream) {
  using P = PairPlan<N>;
  static_assert(P::BYTES + sizeof(PairShared) <= 227 * 1024);
  // of an SM's 228 KB (1 KB for each CTA is the system's) nothing is left for the smallest CTA
  // that takes tensor memory, one of few tokens with a ring of one: none waits for this one's
  constexpr size_t kSmallest = (kChannels + 16) * kTileK + 1024 + sizeof(Shared);
  static_assert(P::BYTES + sizeof(PairShared) + 1024 + kSmallest + 1024 > 228 * 1024);
  a.channel_tiles = (a.n + N - 1) / N;
  const long long tiles = (long long)a.channel_tiles * ((a.rows + kPairTokens - 1) / kPairTokens);
  if (tiles > 0x7fffffffLL / 2) invalid("Int8Linear: too many rows");
  allow_smem(int8_linear_pair_kernel<N, T>, P::BYTES, device_id);
  const CUtensorMap x_map = tile_map(o.x, o.x_stride, a.rows, o.k, 128);
  const CUtensorMap w_map = tile_map(o.w, o.w_stride, a.n, o.k, N / 2);
  const int pairs = (int)std::min<long long>(tiles, sm_count(device_id) / 2);
  launch_pdl(int8_linear_pair_kernel<N, T>, dim3(2 * pairs), dim3(kPairThreads), P::BYTES, stream,
             true, x_map, w_map, a);
}

// Time of a pair kernel in us: turns of all pairs, each as long as the products of a tile
// of N channels or the storing of the one before, and the ends. It is for the choice of N
// alone. Measured, in us (N 64, 128, 256): 256 tokens of 4096 x 14336 29.2, 18.9, 17.2; 512 of
// 4096 x 4096 17.1, 11.7, 15.9; 1024 29.4, 18.1, 15.7; 4096 of 4096 x 28672 618, 383, 294,
// where it chooses the fastest. It underrates stores where K is short, and does not there:
// 4096 of 288 x 1536 10.6 (chosen), 9.3, 10.2; of 512 x 2048 13.0 (chosen), 11.6, 10.5; of 1024
// x 4096 30.7, 21.1 (chosen), 20.1; 777 of 288 x 1536 6.1 (chosen), 6.0, 8.4.
double pair_time(int n, const LinearArgs& a, int sms) {
  const double k = n == 256 ? 0.28 : 0.19, store = 0.01 * n, ends = n == 256 ? 5.5 : 2.6 + 0.006 * n;
  const long long tiles = (long long)((a.n + n - 1) / n) * ((a.rows + kPairTokens - 1) / kPairTokens);
  const long long turns = (tiles + sms / 2 - 1) / (sms / 2);
  return (double)turns * std::max(k * a.tiles_k, store) + ends;
}
// Of the other one, for tiles of 128 tokens: 96 tokens of 14336 x 4096 17.5; 65 of 4096 x
// 4096 9.2, 128 11.7; 128 of 8192 x 10240 33.
double few_time(const LinearArgs& a, int sms) {
  const long long tiles = (a.n + kChannels - 1) / kChannels;
  const FewPlan p = few_plan(128, tiles, a.tiles_k, sms);
  const long long turns = (tiles * p.split + sms - 1) / sms;
  return (double)turns * 0.36 * a.tiles_k / p.split + 4.0 + 0.035 * a.rows;
}

template <class T>
void dispatch(const Operands& o, LinearArgs a, int device_id, cudaStream_t stream) {
  a.tiles_k = (o.k + kTileK - 1) / kTileK;
  if (a.rows <= 16) return launch_few<16, T>(o, a, device_id, stream);
  if (a.rows <= 32) return launch_few<32, T>(o, a, device_id, stream);
  if (a.rows <= 64) return launch_few<64, T>(o, a, device_id, stream);
  const int sms = sm_count(device_id);
  const double t64 = pair_time(64, a, sms), t128 = pair_time(128, a, sms),
               t256 = pair_time(256, a, sms);
  if (a.rows <= 128 && few_time(a, sms) < std::min({t64, t128, t256}))
    return launch_few<128, T>(o, a, device_id, stream);
  if (t256 <= std::min(t64, t128)) return launch_pair<256, T>(o, a, device_id, stream);
  if (t128 <= t64) return launch_pair<128, T>(o, a, device_id, stream);
  return launch_pair<64, T>(o, a, device_id, stream);
}

void run(const Operands& o, LinearArgs a, int out_type, int device_id, cudaStream_t stream) {
  if (a.wait_cycles == 0) a.wait_cycles = kWaitCycles;
  if (out_type == MLB_ACT_BF16)
    dispatch<__nv_bfloat16>(o, a, device_id, stream);
  else
    dispatch<float>(o, a, device_id, stream);
}

// The last wait of the device that gave up, and forgets it.
DeviceStatus take_status() {
  MLB_CUDA(cudaDeviceSynchronize());
  DeviceStatus s;
  MLB_CUDA(cudaMemcpyFromSymbol(&s, g_status, sizeof(s)));
  const DeviceStatus none = {0, 0};
  MLB_CUDA(cudaMemcpyToSymbol(g_status, &none, sizeof(none)));
  return s;
}

void check_codes(const std::string& who, const char* name, const void* p, long long stride, int k) {
  if (!p) invalid(who + ": null " + name);
  if (stride < k) invalid(who + ": row stride of " + name + " is smaller than a row");
  if (reinterpret_cast<uintptr_t>(p) % 16 != 0 || stride % 16 != 0)
    invalid(who + ": rows of " + name + " must be 16-byte aligned");
  if (stride >= (1LL << 40)) invalid(who + ": row stride of " + name + " must be below 2^40");
}
void check_floats(const std::string& who, const char* name, const void* p) {
  if (!p) invalid(who + ": null " + name);
  if (reinterpret_cast<uintptr_t>(p) % 4 != 0) invalid(who + ": " + name + " is unaligned");
}

}  // namespace

}  // namespace mlb

using namespace mlb;

extern "C" int mlb_int8_linear(const int8_t* x, long long x_stride, const float* x_scale, int rows,
                               int in_features, const int8_t* w, long long w_stride,
                               const float* w_scale, int out_features, const float* bias,
                               int out_type, void* out, long long out_stride, int device_id,
                               void* stream) {
  return guarded([&] {
    const std::string who = "Int8Linear";
    paged_check_act("Int8Linear", out_type);
    if (rows < 0) invalid(who + ": negative row count");
    if (rows > (1 << 30)) invalid(who + ": too many rows");
    if (in_features <= 0 || in_features > kMaxK)
      invalid(who + ": in_features must be 1 to 131071, got " + std::to_string(in_features));
    if (out_features <= 0 || out_features > (1 << 28))
      invalid(who + ": out_features must be 1 to 2^28, got " + std::to_string(out_features));
    if (rows > 0) {
      check_codes(who, "x", x, x_stride, in_features);
      check_codes(who, "w", w, w_stride, in_features);
      check_floats(who, "x_scale", x_scale);
      check_floats(who, "w_scale", w_scale);
      if (bias) check_floats(who, "bias", bias);
      if (!out) invalid(who + ": null out");
      const int es = out_type == MLB_ACT_BF16 ? 2 : 4;
      if (reinterpret_cast<uintptr_t>(out) % es != 0) invalid(who + ": out is unaligned");
      if (out_stride < out_features) invalid(who + ": row stride of out is smaller than a row");
      const auto apart = [&](const char* name, const void* p, wide_int stride, wide_int bytes,
                             int n) {
        if (byte_rows_overlap(out, (wide_int)out_stride * es, (wide_int)out_features * es, rows, p,
                              stride, bytes, n))
          invalid(who + ": out must not overlap " + name);
      };
      apart("x", x, x_stride, in_features, rows);
      apart("w", w, w_stride, in_features, out_features);
      apart("x_scale", x_scale, (wide_int)rows * 4, (wide_int)rows * 4, 1);
      apart("w_scale", w_scale, (wide_int)out_features * 4, (wide_int)out_features * 4, 1);
      if (bias) apart("bias", bias, (wide_int)out_features * 4, (wide_int)out_features * 4, 1);
    }
    DeviceScope scope(device_id);
    if (rows == 0) return;
    LinearArgs a = {};
    a.x_scale = x_scale, a.w_scale = w_scale, a.bias = bias;
    a.out = out, a.out_stride = out_stride, a.rows = rows, a.n = out_features;
    run({x, x_stride, w, w_stride, in_features}, a, out_type, device_id,
        static_cast<cudaStream_t>(stream));
  });
}

extern "C" int mlb_int8_linear_status(int device_id, int* code, int* where) {
  return guarded([&] {
    if (!code || !where) invalid("Int8Linear: null output");
    DeviceScope scope(device_id);
    const DeviceStatus s = take_status();
    *code = s.code;
    *where = s.where;
  });
}

extern "C" int mlb_int8_linear_wait_selftest(int device_id, int rows, double limit_ms, int* code,
                                             int* where, int* nan_rows) {
  return guarded([&] {
    if (!code || !where || !nan_rows) invalid("Int8Linear: null output");
    if (rows < 1 || rows > 1024) invalid("Int8Linear: rows must be 1 to 1024");
    if (!(limit_ms > 0.0) || limit_ms > 1000.0)
      invalid("Int8Linear: limit_ms must be in (0, 1000]");
    DeviceScope scope(device_id);
    int khz = 0;
    MLB_CUDA(cudaDeviceGetAttribute(&khz, cudaDevAttrClockRate, device_id));
    // zeros times zeros, with scales of zero
    constexpr int kIn = 2048, kOut = 256;
    const size_t codes = (size_t)(rows + kOut) * kIn, scales = (size_t)(rows + kOut) * sizeof(float);
    const size_t results = (size_t)rows * kOut * sizeof(float);
    const size_t at_scales = codes, at_out = (at_scales + scales + 15) / 16 * 16;
    DevBuf buf(at_out + results);
    uint8_t* p = static_cast<uint8_t*>(buf.p);
    zero_now(p, at_out + results);
    LinearArgs a = {};
    a.x_scale = reinterpret_cast<const float*>(p + at_scales);
    a.w_scale = a.x_scale + rows;
    a.out = p + at_out;
    a.out_stride = kOut, a.rows = rows, a.n = kOut;
    a.wait_cycles = std::max(1LL, (long long)(limit_ms * (double)khz));
    a.never = 1;
    const int8_t* x = reinterpret_cast<const int8_t*>(p);
    run({x, kIn, x + (size_t)rows * kIn, kIn, kIn}, a, MLB_ACT_F32, device_id, nullptr);
    const DeviceStatus st = take_status();
    std::vector<float> out((size_t)rows * kOut);
    MLB_CUDA(cudaMemcpy(out.data(), p + at_out, results, cudaMemcpyDeviceToHost));
    *nan_rows = 0;
    for (int r = 0; r < rows; ++r)
      *nan_rows += std::all_of(out.begin() + (size_t)r * kOut, out.begin() + (size_t)(r + 1) * kOut,
                               [](float v) { return v != v; });
    *code = st.code;
    *where = st.where;
  });
}
