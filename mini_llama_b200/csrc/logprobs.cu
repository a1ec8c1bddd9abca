// logprobs.cu — log probabilities of given tokens, entropy and the most likely
// alternatives of rows of logits.
//
// With y = (x - m) log2(e), m the largest of a thread's elements so far, one
// pass keeps L = sum 2^y and T = sum 2^y y in fp32; partial sums of another m
// join by L' = f L, T' = f (T + d L), f = 2^d, d the difference of the m in
// units of y. At the end
//   logprob(t) = x_t - m - ln L,  entropy = ln 2 (log2 L - T / L).
// The difference is taken before the product: x log2(e) - m log2(e) as one
// multiply-add would leave the product's rounding in y, which for masked logits
// near the type's lowest value is larger than any y that counts. Elements of
// -inf have probability 0.
//
// The k largest (ties: lower index first): 64-bit keys order value, then index.
// Every thread knows the largest key of its own elements from the pass. The k-th
// largest of the largest keys of 32 groups of threads is a lower bound for the
// k-th largest of all, and every key at or above it lies with a thread whose own
// largest is. So the row is not filtered while it streams: those few threads'
// elements are looked at again and the survivors (about k to 3 k) sorted. Rows that
// leave more survivors than the buffer holds (long runs of repeated logits) are
// searched key by key instead.
//
// A row is one CTA, or a cluster of up to 8 when there are too few rows to fill
// the GPU; a cluster's CTAs take one slice each and rank 0 joins their sums and
// lists through distributed shared memory, in rank order.
//
// Measured: 4095 bf16 rows of 32000, k = 1: 73 us, 3.6 TB/s; 64 fp32 rows of 152064,
// k = 5: 14.8 us, 2.6 TB/s; one fp32 row of 128256, k = 20: 10.5 us. Of the first,
// 20 us are what ends a row (joins, candidates), the rest the pass at 4.7 TB/s, bound
// by issue: about six instructions per element, one of them an exponential. Short calls
// are a chain of latencies: launch, load, join, candidates, cluster. A ring of
// asynchronous copies in place of loads to registers was slower (82 us).
#include <algorithm>

#include "paged.cuh"

namespace mlb {

namespace {

constexpr int kMaxTop = 32;
constexpr int kMaxSurvivors = 1024;

struct LogprobArgs {
  const void* logits;
  long long stride;
  const int* tokens;
  int rows, vocab, top_k;
  float *logprob, *entropy;
  int* top_ids;
  float* top_logprob;
};

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Sum of a set of elements: L, T relative to its largest element m.
struct Sums {
  float m, l, t;
};

// Joins two sets. One without weight (l = 0) has no say; NaN stays NaN.
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b) {
  if (b.l == 0.0f) return a;
  if (a.l == 0.0f) return b;
  Sums r;
  r.m = fmaxf(a.m, b.m);
  const float da = a.m == r.m ? 0.0f : (a.m - r.m) * kLog2e;
  const float db = b.m == r.m ? 0.0f : (b.m - r.m) * kLog2e;
  const float fa = ex2(da), fb = ex2(db);
  r.l = fmaf(fa, a.l, fb * b.l);
  // a weight of 0 leaves nothing, whatever d is
  r.t = (fa == 0.0f ? 0.0f : fa * fmaf(da, a.l, a.t)) + (fb == 0.0f ? 0.0f : fb * fmaf(db, b.l, b.t));
  return r;
}

// The sums of N lanes (a power of two, from lane 0 on), in every one of them.
template <int N>
__device__ __forceinline__ Sums warp_join(Sums s) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = N / 2; o > 0; o >>= 1) {
    Sums u;
    u.m = __shfl_xor_sync(0xffffffffu, s.m, o);
    u.l = __shfl_xor_sync(0xffffffffu, s.l, o);
    u.t = __shfl_xor_sync(0xffffffffu, s.t, o);
    s = lane & o ? join(u, s) : join(s, u);
  }
  return s;
}

// Keys: larger value first, then lower index. 0 is below every element's key.
__device__ __forceinline__ uint64_t key_of(float x, int index) {
  const uint32_t u = __float_as_uint(x == 0.0f ? 0.0f : x);  // -0 and 0 are one value
  const uint32_t o = u & 0x80000000u ? ~u : u | 0x80000000u;
  return (uint64_t)o << 32 | (uint32_t)~index;
}
__device__ __forceinline__ float key_value(uint64_t k) {
  const uint32_t o = (uint32_t)(k >> 32);
  return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
__device__ __forceinline__ int key_index(uint64_t k) { return (int)~(uint32_t)k; }

// A warp's 32 keys sorted in descending order (lane 0 the largest).
__device__ __forceinline__ uint64_t exchange(uint64_t k, int o, bool keep_large) {
  const uint64_t u = __shfl_xor_sync(0xffffffffu, k, o);
  return (k > u) == keep_large ? k : u;
}
__device__ __forceinline__ uint64_t warp_sort(uint64_t k) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int n = 2; n <= 32; n <<= 1)
#pragma unroll
    for (int o = n >> 1; o > 0; o >>= 1)
      k = exchange(k, o, ((lane & o) == 0) == ((lane & n) == 0 || n == 32));
  return k;
}
// The 32 largest of two descending lists, descending; b is read back to front.
__device__ __forceinline__ uint64_t warp_merge(uint64_t a, uint64_t b_reversed) {
  const int lane = threadIdx.x & 31;
  uint64_t k = a > b_reversed ? a : b_reversed;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) k = exchange(k, o, (lane & o) == 0);
  return k;
}

// The largest of a warp's keys.
__device__ __forceinline__ uint64_t warp_top(uint64_t k, uint32_t lanes = 0xffffffffu) {
  const uint32_t hi = __reduce_max_sync(lanes, (uint32_t)(k >> 32));
  const uint32_t lo = __reduce_max_sync(lanes, (uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
  return (uint64_t)hi << 32 | lo;
}

// The 32 largest of one key per thread, descending, in lists[0..31]. Every
// thread of the CTA calls it; lists holds 32 keys per warp.
template <int WARPS>
__device__ __forceinline__ void block_top32(uint64_t key, uint64_t* lists) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  key = warp_sort(key);
  lists[warp * 32 + lane] = key;
  __syncthreads();
#pragma unroll
  for (int half = WARPS / 2; half > 0; half >>= 1) {
    if (warp < half) {
      key = warp_merge(key, lists[(warp + half) * 32 + 31 - lane]);
      lists[warp * 32 + lane] = key;
    }
    __syncthreads();
  }
}

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }

// The elements of one 16-byte vector.
__device__ __forceinline__ void unpack(const uint4& u, float (&e)[4]) {
  e[0] = __uint_as_float(u.x), e[1] = __uint_as_float(u.y);
  e[2] = __uint_as_float(u.z), e[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ void unpack(const uint4& u, float (&e)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    e[2 * i] = __uint_as_float(w[i] << 16);
    e[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory");
}
// Address of this CTA's shared variable p in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t peer_addr(const void* p, uint32_t rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_addr(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ uint64_t peer_u64(uint32_t a) {
  uint64_t v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ float peer_f32(uint32_t a) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a));
  return v;
}

template <class T, int THREADS, int SLICES>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? 6 : 2) logprob_kernel(LogprobArgs a) {
  constexpr int WARPS = THREADS / 32;
  constexpr int VEC = 16 / sizeof(T);
  __shared__ uint64_t lists[WARPS * 32];
  __shared__ uint64_t survivors[kMaxSurvivors];
  __shared__ Sums warp_sums[WARPS];
  __shared__ Sums slice_sums;
  __shared__ uint64_t groups[32];
  __shared__ int winners[THREADS];
  __shared__ int n_winners, n_survivors;

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row = blockIdx.x / SLICES;
  const int rank = SLICES > 1 ? (int)cluster_rank() : 0;
  const T* x = static_cast<const T*>(a.logits) + (long long)row * a.stride;
  const int k = a.top_k;

  // this CTA's slice [i0, i1): up to VEC - 1 single elements, whole vectors, a
  // remainder; slices are cut at multiples of 16 bytes of memory
  const int head_all = min((int)((16 - reinterpret_cast<uintptr_t>(x) % 16) % 16 / sizeof(T)),
                           a.vocab);
  const int vecs_all = (a.vocab - head_all) / VEC;
  const int v0 = (int)((long long)vecs_all * rank / SLICES);
  const int v1 = (int)((long long)vecs_all * (rank + 1) / SLICES);
  const int tail0 = head_all + vecs_all * VEC;
  // single elements: the head in the first slice, the remainder in the last
  const int singles_head = rank == 0 ? head_all : 0;
  const int singles = singles_head + (rank == SLICES - 1 ? a.vocab - tail0 : 0);
  auto single_index = [&](int j) { return j < singles_head ? j : tail0 + j - singles_head; };
  const uint4* vx = reinterpret_cast<const uint4*>(x + head_all) + v0;
  const int nv = v1 - v0, first = head_all + v0 * VEC;

  // the given token's logit, on its way from the start
  float chosen = __uint_as_float(0x7fc00000u);
  if (rank == 0 && threadIdx.x == 0) {
    const int t = a.tokens[row];
    if (t >= 0 && t < a.vocab) chosen = to_f(x[t]);
  }

  Sums s = {-INFINITY, 0.0f, 0.0f};
  float ref = 0.0f;  // s.m, or 0 while that is -inf
  float2 l2 = make_float2(0.f, 0.f), t2 = l2;  // the vectors' sums, even and odd elements
  int at = -1;
  auto raise = [&](float top, int index) {
    s.l += l2.x + l2.y;
    s.t += t2.x + t2.y;
    l2 = t2 = make_float2(0.f, 0.f);
    if (s.l != 0.0f) {
      const float d = (s.m - top) * kLog2e, f = ex2(d);
      s.t = f == 0.0f ? 0.0f : f * fmaf(d, s.l, s.t);
      s.l *= f;
    }
    s.m = top;
    ref = top == -INFINITY ? 0.0f : top;
    at = index;
  };
  auto add_one = [&](float e) {
    const float y = (e - ref) * kLog2e, p = ex2(y);
    s.l += p;
    s.t = fmaf(p, fmaxf(y, -1000.0f), s.t);
  };
  auto add = [&](float e, int index) {
    if (e > s.m || (at < 0 && e == s.m)) raise(e, index);
    add_one(e);
  };
  auto add_vec = [&](const uint4& u, int v) {
    float e[VEC];
    unpack(u, e);
    float mx = e[0];
#pragma unroll
    for (int i = 1; i < VEC; ++i) mx = fmaxf(mx, e[i]);
    if (mx > s.m || (at < 0 && mx == s.m)) {
      int i0 = VEC - 1;
#pragma unroll
      for (int i = VEC - 2; i >= 0; --i) i0 = e[i] == mx ? i : i0;
      raise(mx, first + v * VEC + i0);
    }
#pragma unroll
    for (int i = 0; i < VEC; i += 2) {
      const float2 y = mul2(add2(make_float2(e[i], e[i + 1]), make_float2(-ref, -ref)),
                            make_float2(kLog2e, kLog2e));
      const float2 p = make_float2(ex2(y.x), ex2(y.y));
      l2 = add2(l2, p);
      t2 = fma2(p, make_float2(fmaxf(y.x, -1000.0f), fmaxf(y.y, -1000.0f)), t2);
    }
  };

  for (int j = threadIdx.x; j < singles_head; j += THREADS) add(to_f(x[j]), j);
  constexpr int UNROLL = THREADS == 256 ? 2 : 4;  // vectors on their way per thread
  int v = threadIdx.x;
  for (; v + (UNROLL - 1) * THREADS < nv; v += UNROLL * THREADS) {
    uint4 u[UNROLL];
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) u[i] = __ldg(vx + v + i * THREADS);
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) add_vec(u[i], v + i * THREADS);
  }
  for (; v < nv; v += THREADS) add_vec(__ldg(vx + v), v);
  for (int j = singles_head + threadIdx.x; j < singles; j += THREADS) {
    const int i = single_index(j);
    add(to_f(x[i]), i);
  }

  // sums of the slice
  s.l += l2.x + l2.y;
  s.t += t2.x + t2.y;
  const float best = s.m;
  s = warp_join<32>(s);
  if (lane == 0) warp_sums[warp] = s;
  if (threadIdx.x == 0) n_winners = n_survivors = 0;

  // the slice's k largest
  const uint64_t own = at < 0 ? 0 : key_of(best, at);
  uint64_t top = 0;  // lane i of warp 0: the slice's i-th largest
  if (k == 0) {
    __syncthreads();
  } else {
    // 32 groups of threads, each its largest
    constexpr int GROUP = THREADS / 32;
    static_assert(GROUP == 8 || GROUP == 16, "groups are parts of a warp");
    const uint32_t part = ((1u << GROUP) - 1u) << (lane / GROUP * GROUP);
    const uint64_t most = warp_top(own, part);
    if (lane % GROUP == 0) groups[threadIdx.x / GROUP] = most;
    __syncthreads();
    const uint64_t mine = groups[lane];
    if (k == 1) {
      const uint64_t first_key = warp_top(mine);
      top = lane == 0 ? first_key : 0;
    } else {
      const uint64_t bound = __shfl_sync(0xffffffffu, warp_sort(mine), k - 1);  // 0: few elements
      if (own != 0 && own >= bound && bound != 0)
        winners[atomicAdd(&n_winners, 1)] = threadIdx.x;
      __syncthreads();
      auto push = [&](float e, int index) {
        if (!(e == e)) return;
        const uint64_t key = key_of(e, index);
        if (key < bound) return;
        const int n = atomicAdd(&n_survivors, 1);
        if (n < kMaxSurvivors) survivors[n] = key;
      };
      auto push_vec = [&](int w) {
        float e[VEC];
        unpack(__ldg(vx + w), e);
#pragma unroll
        for (int i = 0; i < VEC; ++i) push(e[i], first + w * VEC + i);
      };
      if (bound == 0) {  // a short slice: all of it
        for (int w = threadIdx.x; w < nv; w += THREADS) push_vec(w);
      } else {
        for (int i = warp; i < n_winners; i += WARPS)
          for (int w = winners[i] + lane * THREADS; w < nv; w += 32 * THREADS) push_vec(w);
      }
      for (int j = threadIdx.x; j < singles; j += THREADS) {
        const int i = single_index(j);
        push(to_f(x[i]), i);
      }
      __syncthreads();
      const int n = n_survivors;
      if (n <= 4 * 32) {
        if (warp == 0)
          for (int j = 0; j < n; j += 32) {
            const uint64_t sorted = warp_sort(j + lane < n ? survivors[j + lane] : 0);
            top = j == 0 ? sorted
                         : warp_merge(top, __shfl_sync(0xffffffffu, sorted, 31 - lane));
          }
      } else if (n <= kMaxSurvivors) {
        for (int j = 0; j < n; j += THREADS) {
          block_top32<WARPS>(j + threadIdx.x < n ? survivors[j + threadIdx.x] : 0, lists);
          if (warp == 0) top = j == 0 ? lists[lane] : warp_merge(top, lists[31 - lane]);
          __syncthreads();
        }
      } else {  // one key per round, each the largest below the one before
        uint64_t last = ~0ull;
        for (int r = 0; r < k; ++r) {
          uint64_t best = 0;
          auto look = [&](float e, int index) {
            if (!(e == e)) return;
            const uint64_t key = key_of(e, index);
            if (key < last && key > best) best = key;
          };
          for (int w = threadIdx.x; w < nv; w += THREADS) {
            float e[VEC];
            unpack(__ldg(vx + w), e);
#pragma unroll
            for (int i = 0; i < VEC; ++i) look(e[i], first + w * VEC + i);
          }
          for (int j = threadIdx.x; j < singles; j += THREADS) {
            const int i = single_index(j);
            look(to_f(x[i]), i);
          }
          block_top32<WARPS>(best, lists);
          last = lists[0];
          if (lane == r) top = last;
          __syncthreads();
        }
      }
    }
  }

  if (warp == 0) {
    s = warp_join<WARPS>(warp_sums[lane % WARPS]);
    if (SLICES > 1 && lane == 0) slice_sums = s;
  }
  if (SLICES > 1) {
    __syncthreads();
    if (warp == 0) lists[lane] = top;
    cluster_sync();
    if (rank == 0 && warp == 0) {
      // lane r joins slice r's sums; the lists come all at once
      uint64_t peer[SLICES];
#pragma unroll
      for (int r = 1; r < SLICES; ++r)
        peer[r] = k > 0 ? peer_u64(peer_addr(lists + 31 - lane, r)) : 0;
      const uint32_t p = peer_addr(&slice_sums, lane % SLICES);
      s.m = peer_f32(p);
      s.l = peer_f32(p + 4);
      s.t = peer_f32(p + 8);
      s = warp_join<SLICES>(s);
      if (k > 0)
#pragma unroll
        for (int r = 1; r < SLICES; ++r) top = warp_merge(top, peer[r]);
    }
    cluster_sync();  // a CTA's shared memory lives until rank 0 has read it
    if (rank != 0) return;
  }
  if (warp != 0) return;
  const float ln_l = logf(s.l);
  const float nan = __uint_as_float(0x7fc00000u);
  if (lane == 0) {
    a.logprob[row] = chosen - s.m - ln_l;
    a.entropy[row] = ln_l - kLn2 * (s.t / s.l);
  }
  if (lane < k) {
    // fewer numbers than k in the row (NaN): no alternative
    a.top_ids[(long long)row * k + lane] = top == 0 ? -1 : key_index(top);
    a.top_logprob[(long long)row * k + lane] = top == 0 ? nan : key_value(top) - s.m - ln_l;
  }
}

template <class T, int THREADS, int SLICES>
void launch(const LogprobArgs& a, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.rows * SLICES);
  cfg.blockDim = dim3(THREADS);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = SLICES;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = SLICES > 1 ? 1 : 0;
  MLB_CUDA(cudaLaunchKernelEx(&cfg, logprob_kernel<T, THREADS, SLICES>, a));
}

template <class T>
void dispatch(const LogprobArgs& a, int slices, cudaStream_t s) {
  switch (slices) {
    case 8: return launch<T, 512, 8>(a, s);
    case 4: return launch<T, 512, 4>(a, s);
    case 2: return launch<T, 512, 2>(a, s);
    default: break;
  }
  // many rows: 256 threads have twice the elements each against the same work at
  // the end
  return launch<T, 256, 1>(a, s);
}

}  // namespace

}  // namespace mlb

using namespace mlb;

extern "C" int mlb_logprobs(int logits_type, const void* logits, long long row_stride, int rows,
                            int vocab, const int* tokens, int top_k, float* logprob,
                            float* entropy, int* top_ids, float* top_logprob, int device_id,
                            void* stream) {
  return guarded([&] {
    paged_check_act("LogProbs", logits_type);
    if (rows < 0) invalid("LogProbs: negative row count");
    if (vocab <= 0) invalid("LogProbs: empty logits");
    if (row_stride < vocab) invalid("LogProbs: row stride is smaller than a row");
    if (top_k < 0 || top_k > kMaxTop || top_k > vocab)
      invalid("LogProbs: top_k must be 0 to " + std::to_string(std::min(kMaxTop, vocab)) +
              ", got " + std::to_string(top_k));
    // the grid's x dimension ends at 2^31 - 1 CTAs
    if (rows > (1 << 27)) invalid("LogProbs: too many rows");
    if (rows > 0) {
      if (!logits || !tokens || !logprob || !entropy || (top_k > 0 && (!top_ids || !top_logprob)))
        invalid("LogProbs: null pointer");
      const int es = logits_type == MLB_ACT_BF16 ? 2 : 4;
      if (reinterpret_cast<uintptr_t>(logits) % es != 0) invalid("LogProbs: logits are unaligned");
    }
    DeviceScope scope(device_id);
    if (rows == 0) return;
    LogprobArgs a;
    a.logits = logits;
    a.stride = row_stride;
    a.tokens = tokens;
    a.rows = rows;
    a.vocab = vocab;
    a.top_k = top_k;
    a.logprob = logprob;
    a.entropy = entropy;
    a.top_ids = top_ids;
    a.top_logprob = top_logprob;
    // CTAs per row: double while the rows alone leave SMs without their two
    // CTAs and a slice keeps at least 4096 elements (8 per thread)
    int slices = 1;
    while (slices < 8 && rows * slices * 2 <= 2 * sm_count(device_id) &&
           vocab / (slices * 2) >= 4096)
      slices *= 2;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (logits_type == MLB_ACT_BF16)
      dispatch<__nv_bfloat16>(a, slices, s);
    else
      dispatch<float>(a, slices, s);
  });
}
