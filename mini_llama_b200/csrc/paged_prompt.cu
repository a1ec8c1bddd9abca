// paged_prompt.cu — causal attention over the paged Q4_0 KV cache for many rows
// per sequence, on the tcgen05 tensor cores.
//
// A CTA takes a tile of (token, head) rows of one sequence and KV head and goes
// through the cache 128 tokens at a time:
//
//   S = Q K^T (128 x 128, fp32 in tensor memory), P = exp(S - ref) as fp16 over S,
//   O += P V (fp32 in tensor memory)
//
// Here, unlike in the decode form, codes are widened to fp16 with their scales,
// once for all rows of the tile, as d q. That is a whole multiple of 2^-24, so small
// scales lose nothing, and is off by at most half an fp16 step (2^-11) otherwise.
// Where a scale reaches 4096 it is d q / 16: for K by token, with its S times 16 (a
// group of such a token whose own scale is below 2^-10 is off by up to 2^-32 of the
// token's largest key), for V by 16 tokens, with their P times 16. P is off by at most
// half a step, too. fp32 calls keep queries, K, V and P as hi + lo pairs and add the
// three products that count. The tensor cores cut off what falls below a sum's last
// bit, so O takes only hi hi, one cut per 16 tokens, and the small products have a sum
// of their own (with one sum results over 700 tokens were off by 1.5e-6, now by 5e-7).
// ref is the row's maximum as of the last time that it was looked for and had risen
// by more than a constant: only then is O brought to the new one.
//
// Roles (13 warps, one CTA per SM):
//   warps 0..3    widen K and V into shared memory (fp32 calls: warps 8..11 too)
//   warps 4..7    softmax of rows 0..127, one thread per row; epilogue
//   warps 8..11   bf16 calls: the same for rows 128..255
//   warp 12       tensor memory; one lane issues the products
// bf16 calls keep two row tiles going, so that the tensor cores work on one while
// the softmax of the other runs, with K and V double-buffered. fp32 calls have one
// row tile and S double-buffered.
//
// Measured: 4096 rows of 32 heads over 8 KV heads of 128 (bf16, one sequence): 187 us,
// 735 TFLOP/s of the products that the mask leaves. A step of 2 x 128 rows x 128 tokens takes
// 4650 cycles where its products alone take 2880: the rest is the softmax, 2050
// cycles per row tile (exponentials, rounding and the loads from tensor memory),
// which two tiles do not hide whole. Steps of 64 tokens (242 us), two threads per row
// (227) and registers moved to the softmax warps (215) were slower.
//
// Every wait is bounded: on a timeout the waiting thread records
// MLB_ERR_TIMEOUT in the device's status word (mlb_paged_attention_status) and
// raises the CTA's abort flag; all roles leave their loops, a warp's lanes together,
// rows without a result become NaN, the products in flight are waited for (bounded),
// tensor memory is released and the CTA exits.
#include <algorithm>
#include <type_traits>

#include "paged.cuh"
#include "runtime.cuh"
#include "tcgen05.cuh"

namespace mlb {

namespace {

constexpr int kTok = 128;  // tokens per step
constexpr int kThreads = 13 * 32;
constexpr int kMmaWarp = 12;
constexpr long long kWaitCycles = 2000000000LL;  // about 1 s
// P = 2^((S - ref) rs + lift), rs >= 0 the row's scale. With P up to 2^11, and 2^15
// with the 16 of large V scales, it stays within fp16, and what fp16 loses below 2^-14
// is 2^-(25 + lift) of a token at ref. A step looks for each row's maximum first, and
// ref follows it when that is more than kRise above. bf16 calls first make P in one pass
// under the ref that there is, and leave it at that unless the step's sum exceeds 2^11
// (128 tokens at ref come to 2^10) or there is something to mask.
// ref is a value of S, and the difference comes before the product: no P is above
// 2^lift at ref's own value, however large the scores are. As S rs - ref rs with the
// second product rounded P is off by up to half a step of ref rs, and from scores of
// 2^28 on 2^11 and more. Below kFar that is 2^-12 of P: there one fused multiply-add
// does, which spares the main path of bf16 calls an addition per two scores (4096 rows
// of 32 heads: 186.6 us, 187.8 with it; 2945 of 8 heads of 64
// behind prefixes: 47.7, 49.2).
constexpr float kRise = 4.0f, kMostP = 2048.0f, kFar = 8192.0f;

constexpr uint32_t kBigV = 1, kBigK = 2;
constexpr uint32_t kLargeScale = 0x6C00u;  // 4096 as fp16

__device__ DeviceStatus g_status;

// Shape of one instantiation: bytes of its parts of shared memory.
template <int G, bool SPLIT>
struct Plan {
  static constexpr int D = 32 * G;
  static constexpr int PT = SPLIT ? 2 : 1;      // hi, lo
  static constexpr int NX = SPLIT ? 1 : 2;      // row tiles
  static constexpr int NS = SPLIT ? 1 : 2;      // K and V buffers
  static constexpr int ND = SPLIT ? 8 : 4;      // widening warps
  static constexpr int ROWS = 128 * NX;
  // operands: 8 x 16-byte core matrices, 128 bytes apart along the contraction
  static constexpr int SBO_D = D / 8 * 128;     // rows of Q and K, contraction D
  // rows of V^T, contraction tokens; 16 bytes more, so that the eight rows of a
  // stored matrix, two of each of four row groups, fall into different banks
  static constexpr int SBO_T = kTok / 8 * 128 + 16;
  static constexpr int Q = 128 / 8 * SBO_D;     // one row tile, one part
  static constexpr int K = kTok / 8 * SBO_D;
  static constexpr int V = D / 8 * SBO_T;
  static constexpr int Q0 = 0;
  static constexpr int K0 = Q0 + NX * PT * Q;
  static constexpr int V0 = K0 + NS * PT * K;
  static constexpr int BYTES = V0 + NS * PT * V;
  // tensor memory columns
  static constexpr int O_COL = 0;               // + 128 x
  static constexpr int S_COL = SPLIT ? 128 : 256;  // + 128 x (bf16), + 128 (step & 1) (fp32)
  static constexpr int OLO_COL = 384;           // fp32: the small products of O
  // P over S: 32 tokens' hi in 16 columns; fp32: their lo in the 16 after them
  static constexpr int P_STEP = SPLIT ? 32 : 16;
};

struct Shared {
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2];
  uint64_t s_full[2], p_full[2], o_done[2], o_last[2], q_full, drain;
  long long warp_sums[kThreads / 32];
  long long base;
  long long wait_cycles;
  int seq;
  int abort_flag;
  uint32_t tmem;
  float row_scale[256];
  // per step & 3, one byte per block: without a page; kBigV with large V scales, kBigK
  // with large K scales, whose tokens are the bits of k_big
  alignas(8) uint8_t absent[4][8];
  alignas(8) uint8_t big[4][8];
  alignas(4) uint16_t k_big[4][8];
};

// Bounded wait of one thread that also gives up when another one did.
__device__ __forceinline__ bool wait(Shared& sh, uint64_t* bar, int phase, int where) {
  if (mbar_try_wait(bar, (uint32_t)phase & 1u)) return true;
  const long long start = clock64();
  while (!mbar_try_wait(bar, (uint32_t)phase & 1u)) {
    if (*(volatile int*)&sh.abort_flag) return false;
    if (clock64() - start > sh.wait_cycles) {
      atomicExch(&g_status.code, MLB_ERR_TIMEOUT);
      atomicExch(&g_status.where, where);
      *(volatile int*)&sh.abort_flag = 1;
      return false;
    }
  }
  return true;
}

// The same for a warp: its lanes go on or give up together, for what follows is for
// whole warps. Out of line where the first try fails: inside, the bf16 softmax lost
// registers to it (4096 rows of 32 heads 192.7 us, so 186.6).
__device__ __noinline__ bool wait_longer(Shared& sh, uint64_t* bar, int phase, int where) {
  return __all_sync(0xffffffffu, wait(sh, bar, phase, where));
}
__device__ __forceinline__ bool wait_warp(Shared& sh, uint64_t* bar, int phase, int where) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, (uint32_t)phase & 1u))) return true;
  return wait_longer(sh, bar, phase, where);
}

template <int G, class T>
__global__ void __launch_bounds__(kThreads, 1) paged_prompt_kernel(PagedAttnArgs a) {
  constexpr bool SPLIT = sizeof(T) == 4;
  using P = Plan<G, SPLIT>;
  constexpr int D = P::D, NX = P::NX, NS = P::NS, PT = P::PT;
  constexpr float kLift = SPLIT ? 11.0f - kRise : 3.0f;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Shared sh;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;

  // the sequence, KV head and row tile of this CTA; later tiles, which see more,
  // come first
  int seq = -1, head = 0, tile = 0;
  SeqWork sw = {};
  if (a.seqs.n_seqs == 1) {  // nothing to look through
    sw = seq_work(a, 0, P::ROWS, kTok, 0);
    if (blockIdx.x >= (long long)sw.tiles * a.cache.kv) return;
    seq = 0;
    head = blockIdx.x % a.cache.kv;
    tile = sw.tiles - 1 - blockIdx.x / a.cache.kv;
  } else {
    long long base = 0;
    if (threadIdx.x == 0) sh.seq = -1;
    __syncthreads();
    for (int s0 = 0; s0 < a.seqs.n_seqs; s0 += kThreads) {
      const int s = s0 + threadIdx.x;
      long long units = 0;
      if (s < a.seqs.n_seqs) {
        const SeqWork w = seq_work(a, s, P::ROWS, kTok, 0);
        units = (long long)w.tiles * a.cache.kv;
      }
      const long long incl = block_scan<kThreads>(units, sh.warp_sums) + base;
      if (blockIdx.x >= incl - units && blockIdx.x < incl) {
        sh.seq = s;
        sh.base = incl - units;
      }
      if (threadIdx.x == kThreads - 1) sh.warp_sums[0] = incl;
      __syncthreads();
      base = sh.warp_sums[0];
      __syncthreads();
      if (base > blockIdx.x) break;
    }
    seq = sh.seq;
    if (seq < 0) return;
    sw = seq_work(a, seq, P::ROWS, kTok, 0);
    const int u = (int)(blockIdx.x - sh.base);
    head = u % a.cache.kv;
    tile = sw.tiles - 1 - u / a.cache.kv;
  }

  // steps that each row tile needs: up to what its last row sees
  const long long rows = (long long)sw.n * a.group, row0 = (long long)tile * P::ROWS;
  int steps[2] = {0, 0};
#pragma unroll
  for (int x = 0; x < NX; ++x) {
    const long long first = row0 + x * 128;
    if (first < rows) {
      const int tok = (int)(min(first + 127, rows - 1) / a.group);
      steps[x] = (seen_by(sw.pos0, tok, sw.len) + kTok - 1) / kTok;
    }
  }
  const int n = max(steps[0], steps[1]);

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.k_full[i], P::ND + a.never);
      mbar_init(&sh.v_full[i], P::ND);
      mbar_init(&sh.k_empty[i], 1);
      mbar_init(&sh.v_empty[i], 1);
      mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.p_full[i], 4);
      mbar_init(&sh.o_done[i], 1);
      mbar_init(&sh.o_last[i], 1);
    }
    mbar_init(&sh.q_full, 4 * NX);
    mbar_init(&sh.drain, 1);
    sh.abort_flag = 0;
    sh.wait_cycles = a.wait_cycles;
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(&sh.tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;

  if (warp < 4 || (SPLIT && warp >= 8 && warp < 12)) {
    // ------------------------------------------------------------- widening
    // K: token kg, chunk kc, so that eight lanes store 128 bytes in a row; V: token
    // pair c of row lane / 4
    const int dw = warp < 4 ? warp : warp - 4;
    const int kg = lane & 7, kc = lane >> 3, c = lane & 3;
    const int bpp = a.cache.page_size / kPagedBlock;
    constexpr int BLOCK = 576 * G;
    constexpr int NB = 8 / P::ND;  // blocks per warp and step
    const __half2 sixteenth = u32_as_h2(0x2C002C00u);
    for (int j = 0; j < n; ++j) {
      const int st = j % NS;
      // this warp's blocks of the step, as they are in memory
      uint32_t kw[NB][2][G], ks[NB][2][G], vw[NB][2][G], vs[NB][2][G];
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const int b = dw * NB + i, bl = j * 8 + b;
        int page = -1;
        if (bl * kPagedBlock < sw.len) {
          const int p = bl / bpp;
          page = a.seqs.table[(size_t)seq * a.seqs.max_pages + p];
          if (page >= a.cache.n_pages) page = -1;
          if (page >= 0) {
            const uint8_t* block =
                a.cache.layer +
                (size_t)((page * a.cache.kv + head) * bpp + (bl - p * bpp)) * BLOCK;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              lds_words<G>(block + (h * 8 + kg) * 16 * G + kc * 4 * G, kw[i][h]);
              lds_words<G>(block + (256 + 128 * h) * G + lane * 4 * G, vw[i][h]);
              lds_words<G>(block + 512 * G + (h * 4 + (kg >> 1)) * 4 * G, ks[i][h]);
              lds_words<G>(block + 544 * G + (h * 4 + c) * 4 * G, vs[i][h]);
            }
          }
        }
        // K: the scale of token kg in both halves
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int w = 0; w < G; ++w)
            ks[i][h][w] = __byte_perm(ks[i][h][w], 0, kg & 1 ? 0x3232 : 0x1010);
        // scales of tokens that are not there: 0, whatever their codes
        if (page < 0 || (bl + 1) * kPagedBlock > sw.len) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int left = page < 0 ? 0 : sw.len - bl * kPagedBlock - h * 8;
            const uint32_t kt = kg < left ? 0xffffffffu : 0u;
            const uint32_t vt =
                (2 * c < left ? 0xffffu : 0u) | (2 * c + 1 < left ? 0xffff0000u : 0u);
#pragma unroll
            for (int w = 0; w < G; ++w) {
              if (page < 0) kw[i][h][w] = vw[i][h][w] = ks[i][h][w] = vs[i][h][w] = 0u;
              ks[i][h][w] &= kt;
              vs[i][h][w] &= vt;
            }
          }
        }
        // large scales: a vote for all of them, the rest only where there are some
        __half2 top = u32_as_h2(0u);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int w = 0; w < G; ++w)
            top = __hmax2(top, __hmax2(u32_as_h2(ks[i][h][w]), u32_as_h2(vs[i][h][w])));
        const uint32_t tb = h2_as_u32(top);
        uint32_t big = 0, k_big = 0;
        if (__any_sync(0xffffffffu, max(tb & 0xffffu, tb >> 16) >= kLargeScale)) {
          __half2 v_top = u32_as_h2(0u);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t k_top = 0;
#pragma unroll
            for (int w = 0; w < G; ++w) {
              k_top = max(k_top, ks[i][h][w]);
              v_top = __hmax2(v_top, u32_as_h2(vs[i][h][w]));
            }
            const bool large = k_top >= kLargeScale << 16;
            // lanes 0..7 stand for eight tokens
            k_big |= (__ballot_sync(0xffffffffu, large) & 0xffu) << (8 * h);
            if (large) {
#pragma unroll
              for (int w = 0; w < G; ++w)
                ks[i][h][w] = h2_as_u32(__hmul2(u32_as_h2(ks[i][h][w]), sixteenth));
            }
          }
          if (k_big) big |= kBigK;
          const uint32_t vb = h2_as_u32(v_top);
          if (__any_sync(0xffffffffu, max(vb & 0xffffu, vb >> 16) >= kLargeScale)) {
            big |= kBigV;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int w = 0; w < G; ++w)
                vs[i][h][w] = h2_as_u32(__hmul2(u32_as_h2(vs[i][h][w]), sixteenth));
          }
        }
        if (lane == 0) {
          sh.absent[j & 3][b] = page < 0;
          sh.big[j & 3][b] = (uint8_t)big;
          sh.k_big[j & 3][b] = (uint16_t)k_big;
        }
      }

      if (j >= NS && !wait_warp(sh, &sh.k_empty[st], j / NS - 1, 1001)) break;
      uint8_t* k0 = smem + P::K0 + st * PT * P::K;
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint8_t* at = k0 + ((dw * NB + i) * 2 + h) * P::SBO_D + kc * 128 + kg * 16;
#pragma unroll
          for (int w = 0; w < G; ++w) {
            uint32_t r[4], x[4];
            codes_f16(kw[i][h][w], r);
            const __half2 d = u32_as_h2(ks[i][h][w]);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = h2_as_u32(__hmul2(u32_as_h2(r[e]), d));
            *reinterpret_cast<uint4*>(at + w * 512) = make_uint4(x[0], x[1], x[2], x[3]);
            if (SPLIT) {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                r[e] = h2_as_u32(__hfma2(u32_as_h2(r[e]), d, __hneg2(u32_as_h2(x[e]))));
              *reinterpret_cast<uint4*>(at + P::K + w * 512) = make_uint4(r[0], r[1], r[2], r[3]);
            }
          }
        }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.k_full[st]);

      if (j >= NS && !wait_warp(sh, &sh.v_empty[st], j / NS - 1, 1002)) break;
      uint8_t* v0 = smem + P::V0 + st * PT * P::V;
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          // lane 8 e + k: row 4 k + e of a group of 32 dimensions
          uint8_t* at = v0 + (kg >> 1) * P::SBO_T + ((dw * NB + i) * 2 + h) * 128 +
                        (4 * (kg & 1) + kc) * 16;
#pragma unroll
          for (int w = 0; w < G; ++w) {
            uint32_t r[4], x[4];
            codes_f16(vw[i][h][w], r);
            const __half2 d = u32_as_h2(vs[i][h][w]);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = h2_as_u32(__hmul2(u32_as_h2(r[e]), d));
            store_matrices(at + w * 4 * P::SBO_T, x);
            if (SPLIT) {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                r[e] = h2_as_u32(__hfma2(u32_as_h2(r[e]), d, __hneg2(u32_as_h2(x[e]))));
              store_matrices(at + P::V + w * 4 * P::SBO_T, r);
            }
          }
        }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.v_full[st]);
    }
  } else if (warp < 12) {
    // -------------------------------------------------------------- softmax
    // first the queries as operand tiles, 8 rows per warp and turn
    {
      const int g = lane >> 2, c = lane & 3;
      const float sign = a.scale_log2 < 0.0f ? -1.0f : 1.0f;
      for (int r0 = (warp - 4) * 8; r0 < P::ROWS; r0 += 4 * NX * 8) {
        const long long flat = row0 + r0 + g;
        const T* row = nullptr;
        if (flat < rows) {
          const int i = (int)(flat / a.group);
          row = static_cast<const T*>(a.q) + (long long)(sw.row0 + i) * a.q_stride +
                (size_t)(head * a.group + (int)(flat - (long long)i * a.group)) * a.cache.head_dim;
        }
        float e[G][8];
        load_query_elements<G, T>(row, a.cache.head_dim, c, e);
        const int sh2 = query_shift<G>(e);
        if (c == 0) sh.row_scale[r0 + g] = pow2(-sh2) * sign * a.scale_log2;
        const float sf = pow2(sh2) * sign;
        uint8_t* at = smem + P::Q0 + (r0 / 128) * PT * P::Q + (r0 % 128) / 8 * P::SBO_D + g * 16;
#pragma unroll
        for (int w = 0; w < G; ++w) {
          uint32_t hi[4], lo[4];
          query_words(e[w], sf, SPLIT, hi, lo);
          *reinterpret_cast<uint4*>(at + (4 * w + c) * 128) =
              make_uint4(hi[0], hi[1], hi[2], hi[3]);
          if (SPLIT)
            *reinterpret_cast<uint4*>(at + P::Q + (4 * w + c) * 128) =
                make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.q_full);
      asm volatile("bar.sync 1, %0;" ::"n"(4 * NX * 32) : "memory");  // row_scale
    }
    const int x = (warp - 4) / 4;
    const int r = x * 128 + (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t o_at = tmem + lanes + P::O_COL + 128 * x;
    const uint32_t olo_at = tmem + lanes + P::OLO_COL;  // fp32
    const long long flat = row0 + r;
    const bool live = flat < rows;
    const int tok = live ? (int)(flat / a.group) : 0;
    // rows of no one hide nothing, so that their warps need not mask
    const int vis = live ? seen_by(sw.pos0, tok, sw.len) : 0x40000000;
    const float rs = sh.row_scale[r];
    const int nx = steps[x];
    float ref = -INFINITY;
    float2 l0 = make_float2(0.f, 0.f), l1 = make_float2(0.f, 0.f);
    bool ok = true;
    for (int j = 0; ok && j < nx; ++j) {
      const int b = SPLIT ? j & 1 : x;
      ok = wait_warp(sh, &sh.s_full[b], SPLIT ? j >> 1 : j, 1003);
      if (!ok) break;
      tc_fence_after();
      const uint32_t s_at = tmem + lanes + P::S_COL + 128 * b;
      const uint64_t absent = *reinterpret_cast<const volatile uint64_t*>(sh.absent[j & 3]);
      const uint64_t big = *reinterpret_cast<const volatile uint64_t*>(sh.big[j & 3]);
      const int left = vis - j * kTok;  // tokens of the step that the row sees
      const bool whole = __all_sync(0xffffffffu, left >= kTok) && absent == 0;
      // mask of 32 tokens: what the row sees of them
      auto seen = [&](int ch) {
        const int v = left - 32 * ch;
        uint32_t m = v >= 32 ? 0xffffffffu : v <= 0 ? 0u : (1u << v) - 1u;
        if (absent >> (16 * ch) & 0xff) m &= 0xffff0000u;
        if (absent >> (16 * ch + 8) & 0xff) m &= 0x0000ffffu;
        return m;
      };

      // bf16, nothing to mask, no large scale, and no ref so large that its product's
      // rounding would tell: P of the whole step in registers under the ref that there is,
      // in one pass over S; not taken if a row's P have become too large
      bool done = false, tried = false;
      if constexpr (!SPLIT) {
        tried = whole && big == 0 && __all_sync(0xffffffffu, fabsf(ref * rs) < kFar);
        if (tried) {
          const float neg = fmaf(-ref, rs, kLift);
          float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
          // 32 tokens on their way while 32 are worked on (products slow the loads
          // down to about the time that this takes)
          uint32_t u[2][32], hi[4][16];
          tmem_ld32_start(s_at, u[0]);
#pragma unroll
          for (int ch = 0; ch < 4; ++ch) {
            tmem_ld32_wait(u[ch & 1]);
            if (ch < 3) tmem_ld32_start(s_at + 32 * (ch + 1), u[(ch + 1) & 1]);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              float2 p = make_float2(__uint_as_float(u[ch & 1][2 * i]),
                                     __uint_as_float(u[ch & 1][2 * i + 1]));
              p = fma2(p, make_float2(rs, rs), make_float2(neg, neg));
              p.x = ex2(p.x);
              p.y = ex2(p.y);
              sum[i & 1] = add2(sum[i & 1], p);
              hi[ch][i] = pack_f16(p.x, p.y);
            }
          }
          // no P above the sum, so none that fp16 does not hold; looking for the maximum
          // as well would cost a sixth of the pass
          done = !__any_sync(0xffffffffu, (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y) > kMostP);
          if (done) {
            l0 = add2(l0, sum[0]);
            l1 = add2(l1, sum[1]);
#pragma unroll
            for (int ch = 0; ch < 4; ++ch) tmem_st16(s_at + P::P_STEP * ch, hi[ch]);
          }
        }
      }

      // otherwise the largest S first, then P as it is made
      if (!done) {
        if (big & 0x0101010101010101ull * kBigK) {  // S of keys stored as d q / 16
#pragma unroll 1
          for (int ch = 0; ch < 4; ++ch) {
            const uint32_t k16 =
                *reinterpret_cast<const volatile uint32_t*>(&sh.k_big[j & 3][2 * ch]);
            float v[32];
            tmem_ld32(s_at + 32 * ch, v);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t u[16];
#pragma unroll
              for (int i = 0; i < 16; ++i)
                u[i] = __float_as_uint(v[16 * h + i] * (k16 >> (16 * h + i) & 1 ? 16.0f : 1.0f));
              tmem_st16(s_at + 32 * ch + 16 * h, u);
            }
          }
          tmem_wait_st();
        }

        float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll 1
        for (int ch = 0; ch < 4; ++ch) {
          float v[32];
          tmem_ld32(s_at + 32 * ch, v);
          const uint32_t m = whole ? 0xffffffffu : seen(ch);
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            m0 = fmaxf(m0, m >> i & 1 ? v[i] : -INFINITY);
            m1 = fmaxf(m1, m >> (i + 1) & 1 ? v[i + 1] : -INFINITY);
          }
        }
        // ref of the rows that rise, their sums and O go to the maximum
        const float mx = fmaxf(m0, m1);
        const bool rise =
            ref == -INFINITY ? mx > ref : tried ? mx > ref : (mx - ref) * rs > kRise;
        if (__any_sync(0xffffffffu, rise)) {
          const float f = !rise ? 1.0f : ref == -INFINITY ? 0.0f : ex2((ref - mx) * rs);
          if (rise) ref = mx;
          if (j > 0) {  // there is an O
            ok = wait_warp(sh, &sh.o_done[x], j - 1, 1004);
            if (!ok) break;
            tc_fence_after();
            l0 = mul2(l0, make_float2(f, f));
            l1 = mul2(l1, make_float2(f, f));
#pragma unroll 1
            for (int ch = 0; ch < PT * G; ++ch) {
              const uint32_t at = ch < G ? o_at + 32 * ch : olo_at + 32 * (ch - G);
              float v[32];
              tmem_ld32(at, v);
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                uint32_t u[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) u[i] = __float_as_uint(v[16 * h + i] * f);
                tmem_st16(at + 16 * h, u);
              }
            }
            tmem_wait_st();
          }
        }

        const float from = ref == -INFINITY ? 0.0f : -ref;
#pragma unroll 1
        for (int ch = 0; ch < 4; ++ch) {
          float v[32];
          tmem_ld32(s_at + 32 * ch, v);
          const uint32_t m = whole ? 0xffffffffu : seen(ch);
          uint32_t hi[16], lo[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float2 p = fma2(add2(make_float2(v[2 * i], v[2 * i + 1]), make_float2(from, from)),
                            make_float2(rs, rs), make_float2(kLift, kLift));
            p.x = m >> (2 * i) & 1 ? ex2(p.x) : 0.0f;
            p.y = m >> (2 * i + 1) & 1 ? ex2(p.y) : 0.0f;
            if (i & 1)
              l1 = add2(l1, p);
            else
              l0 = add2(l0, p);
            const float up = big >> (16 * ch + 8 * (i >> 3)) & kBigV ? 16.0f : 1.0f;
            p = mul2(p, make_float2(up, up));
            hi[i] = pack_f16(p.x, p.y);
            if (SPLIT) {
              const float2 h = __half22float2(u32_as_h2(hi[i]));
              lo[i] = pack_f16(p.x - h.x, p.y - h.y);
            }
          }
          tmem_st16(s_at + P::P_STEP * ch, hi);  // over S that has been read
          if (SPLIT) tmem_st16(s_at + P::P_STEP * ch + 16, lo);
        }
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.p_full[x]);
    }
    if (ok && nx > 0) {
      ok = wait_warp(sh, &sh.o_last[x], 0, 1005);
      tc_fence_after();
    }
    if (ok) {
      const float l = (l0.x + l0.y) + (l1.x + l1.y);
      const float f = l == 0.0f ? 0.0f : 1.0f / l;
      T* out = live ? static_cast<T*>(a.out) + (long long)(sw.row0 + tok) * a.out_stride +
                          (size_t)(head * a.group + (int)(flat - (long long)tok * a.group)) *
                              a.cache.head_dim
                    : nullptr;
#pragma unroll
      for (int ch = 0; ch < G; ++ch) {
        float v[32];
        if (nx > 0) {
          tmem_ld32(o_at + 32 * ch, v);
          if (SPLIT) {
            float u[32];
            tmem_ld32(olo_at + 32 * ch, u);
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] += u[i];
          }
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = 0.0f;
        }
        if (live) {
#pragma unroll
          for (int i = 0; i < 32; i += 8)
            if (32 * ch + i < a.cache.head_dim) {
              store_act4(out + 32 * ch + i, make_float4(v[i] * f, v[i + 1] * f, v[i + 2] * f,
                                                        v[i + 3] * f));
              store_act4(out + 32 * ch + i + 4, make_float4(v[i + 4] * f, v[i + 5] * f,
                                                            v[i + 6] * f, v[i + 7] * f));
            }
        }
      }
      tc_fence_before();
    } else if (live) {  // no result
      const float nan = __uint_as_float(0x7fc00000u);
      T* out = static_cast<T*>(a.out) + (long long)(sw.row0 + tok) * a.out_stride +
               (size_t)(head * a.group + (int)(flat - (long long)tok * a.group)) *
                   a.cache.head_dim;
      for (int d = 0; d < a.cache.head_dim; d += 4)
        store_act4(out + d, make_float4(nan, nan, nan, nan));
    }
  } else if (warp == kMmaWarp && lane == 0) {
    // ------------------------------------------------------------- products
    const uint32_t base = smem_addr(smem);
    const uint32_t id_s = idesc_f16(kTok), id_o = idesc_f16(D);
    // operand descriptors: the high words are alike, the low words step by bytes / 16
    const uint64_t dq = smem_desc(base + P::Q0, P::SBO_D), dv = smem_desc(base + P::V0, P::SBO_T);
    const uint32_t q_lo = (uint32_t)dq, k_lo = (uint32_t)smem_desc(base + P::K0, P::SBO_D);
    const uint32_t v_lo = (uint32_t)dv;
    const uint32_t hi_d = (uint32_t)(dq >> 32), hi_t = (uint32_t)(dv >> 32);
    // S of row tile x, step j
    auto scores = [&](int x, int j) {
      const uint32_t d = tmem + P::S_COL + 128 * (SPLIT ? j & 1 : x);
      const uint32_t q = q_lo + x * (PT * P::Q / 16), k = k_lo + (j % NS) * (PT * P::K / 16);
      // fp32: lo hi and hi lo first, while the sum is small
#pragma unroll
      for (int part = SPLIT ? 2 : 0; part >= 0; --part)
#pragma unroll
        for (int s = 0; s < 2 * G; ++s) {
          const uint32_t aq = q + (part == 1 ? P::Q / 16 : 0) + s * 16;
          const uint32_t bk = k + (part == 2 ? P::K / 16 : 0) + s * 16;
          if (part == (SPLIT ? 2 : 0) && s == 0)
            tc_mma_ss2<false>(d, aq, hi_d, bk, hi_d, id_s);
          else
            tc_mma_ss2<true>(d, aq, hi_d, bk, hi_d, id_s);
        }
    };
    // O of row tile x += P V of step j
    auto values = [&](int x, int j) {
      const uint32_t p = tmem + P::S_COL + 128 * (SPLIT ? j & 1 : x);
      const uint32_t v = v_lo + (j % NS) * (PT * P::V / 16);
#pragma unroll
      for (int part = 0; part < (SPLIT ? 3 : 1); ++part) {
        const uint32_t d = tmem + (part == 0 ? P::O_COL + 128 * x : P::OLO_COL);
#pragma unroll
        for (int s = 0; s < kTok / 16; ++s) {
          const uint32_t ap = p + P::P_STEP * (s / 2) + 8 * (s % 2) + (part == 1 ? 16 : 0);
          const uint32_t bv = v + (part == 2 ? P::V / 16 : 0) + s * 16;
          if (part < 2 && s == 0 && j == 0)
            tc_mma_ts2<false>(d, ap, bv, hi_t, id_o);
          else
            tc_mma_ts2<true>(d, ap, bv, hi_t, id_o);
        }
      }
    };
    bool ok = wait(sh, &sh.q_full, 0, 1011) && (n == 0 || wait(sh, &sh.k_full[0], 0, 1006));
    if (ok && n > 0) {
      tc_fence_after();
#pragma unroll
      for (int x = 0; x < NX; ++x)
        if (steps[x] > 0) {
          scores(x, 0);
          tc_commit(&sh.s_full[x]);
        }
      tc_commit(&sh.k_empty[0]);
    }
    for (int j = 0; ok && j < n; ++j) {
      const int st = j % NS, st1 = (j + 1) % NS;
      if (SPLIT) {
        if (j + 1 < n) {  // over P of step j - 1: its product has to be done
          ok = wait(sh, &sh.k_full[st1], (j + 1) / NS, 1007) &&
               (j == 0 || wait(sh, &sh.o_done[0], j - 1, 1010));
          if (!ok) break;
          tc_fence_after();
          scores(0, j + 1);
          tc_commit(&sh.s_full[(j + 1) & 1]);
          tc_commit(&sh.k_empty[st1]);
        }
        ok = wait(sh, &sh.v_full[st], j / NS, 1008) && wait(sh, &sh.p_full[0], j, 1009);
        if (!ok) break;
        tc_fence_after();
        values(0, j);
        tc_commit(&sh.o_done[0]);
        tc_commit(&sh.v_empty[st]);
        if (j + 1 == n) tc_commit(&sh.o_last[0]);
      } else {
        ok = wait(sh, &sh.v_full[st], j / NS, 1008);
        if (!ok) break;
        bool k_seen = false;
#pragma unroll
        for (int x = 0; x < NX; ++x) {
          if (j < steps[x]) {
            ok = wait(sh, &sh.p_full[x], j, 1009);
            if (!ok) break;
            tc_fence_after();
            values(x, j);
            tc_commit(&sh.o_done[x]);
            if (j + 1 == steps[x]) tc_commit(&sh.o_last[x]);
          }
          if (j + 1 < steps[x]) {
            // over P of step j: products of unlike accumulators need not run in the
            // order of their issue
            ok = (k_seen || wait(sh, &sh.k_full[st1], (j + 1) / NS, 1007)) &&
                 wait(sh, &sh.o_done[x], j, 1010);
            if (!ok) break;
            k_seen = true;
            tc_fence_after();
            scores(x, j + 1);
            tc_commit(&sh.s_full[x]);
          }
        }
        if (!ok) break;
        tc_commit(&sh.v_empty[st]);
        if (j + 1 < n) tc_commit(&sh.k_empty[st1]);
      }
    }
    // nothing is in flight when tensor and shared memory go
    tc_commit(&sh.drain);
    const long long start = clock64();
    while (!mbar_try_wait(&sh.drain, 0) && clock64() - start < sh.wait_cycles) {
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
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

template <int G, class T>
void launch(const PagedAttnArgs& a, int device_id, cudaStream_t stream) {
  using P = Plan<G, sizeof(T) == 4>;
  allow_smem(paged_prompt_kernel<G, T>, P::BYTES, device_id);
  const long long tiles = (long long)a.seqs.n_rows * a.group / P::ROWS + a.seqs.n_seqs;
  const long long grid = tiles * a.cache.kv;
  if (grid > 0x7fffffffLL) invalid("CudaPagedAttention: too many rows");
  paged_prompt_kernel<G, T><<<(unsigned)grid, kThreads, P::BYTES, stream>>>(a);
  MLB_CUDA(cudaGetLastError());
}

template <class T>
void dispatch(const PagedAttnArgs& a, int device_id, cudaStream_t stream) {
  switch (paged_groups(a.cache.head_dim)) {
    case 1: return launch<1, T>(a, device_id, stream);
    case 2: return launch<2, T>(a, device_id, stream);
    case 3: return launch<3, T>(a, device_id, stream);
    default: return launch<4, T>(a, device_id, stream);
  }
}

}  // namespace

void paged_prompt_launch(const PagedAttnArgs& args, int act_type, int device_id,
                         cudaStream_t stream) {
  PagedAttnArgs a = args;
  if (a.wait_cycles == 0) a.wait_cycles = kWaitCycles;
  if (act_type == MLB_ACT_BF16)
    dispatch<__nv_bfloat16>(a, device_id, stream);
  else
    dispatch<float>(a, device_id, stream);
}

}  // namespace mlb

using namespace mlb;

extern "C" int mlb_paged_attention_status(int device_id, int* code, int* where) {
  return guarded([&] {
    if (!code || !where) invalid("CudaPagedAttention: null output");
    DeviceScope scope(device_id);
    const DeviceStatus s = take_status();
    *code = s.code;
    *where = s.where;
  });
}

extern "C" int mlb_paged_attention_wait_selftest(int device_id, int act_type, double limit_ms,
                                                 int* code, int* where, int* nan_rows) {
  return guarded([&] {
    const char* who = "CudaPagedAttention";
    if (!code || !where || !nan_rows) invalid("CudaPagedAttention: null output");
    paged_check_act(who, act_type);
    if (!(limit_ms > 0.0) || limit_ms > 1000.0)
      invalid("CudaPagedAttention: limit_ms must be in (0, 1000]");
    DeviceScope scope(device_id);
    int khz = 0;
    MLB_CUDA(cudaDeviceGetAttribute(&khz, cudaDevAttrClockRate, device_id));
    // one sequence of kRows rows over one page of zeros, one head of 32
    constexpr int kRows = 8, kDim = 32, kPage = kPagedBlock;
    const size_t page = paged_page_bytes(kPage, 1, kDim), rows = kRows * kDim * sizeof(float);
    const int seqs[4] = {0, kRows, kRows, 0};  // row offsets, length, page table
    const size_t at_q = page, at_out = at_q + rows, at_seqs = at_out + rows;
    DevBuf buf(at_seqs + sizeof(seqs));
    uint8_t* p = static_cast<uint8_t*>(buf.p);
    zero_now(p, at_seqs);
    copy_to_device_now(p + at_seqs, seqs, sizeof(seqs));
    const int* s = reinterpret_cast<const int*>(p + at_seqs);
    PagedAttnArgs a = {};
    a.cache = paged_cache(who, p, 1, 1, kPage, 1, kDim, 0);
    a.seqs = paged_seqs(who, kRows, 1, s, s + 2, s + 3, 1, kPage);
    a.q = p + at_q;
    a.out = p + at_out;
    a.q_stride = a.out_stride = kDim;
    a.n_heads = a.group = 1;
    a.scale_log2 = 1.0f;
    a.wait_cycles = std::max(1LL, (long long)(limit_ms * (double)khz));
    a.never = 1;
    paged_prompt_launch(a, act_type, device_id, nullptr);
    const DeviceStatus st = take_status();
    uint32_t out[kRows * kDim];
    MLB_CUDA(cudaMemcpy(out, p + at_out, rows, cudaMemcpyDeviceToHost));
    // a row's elements are NaN if every word holds one (bf16: two, in half the words)
    const int words = act_type == MLB_ACT_BF16 ? kDim / 2 : kDim;
    const uint32_t nan = act_type == MLB_ACT_BF16 ? 0x7fc07fc0u : 0x7fc00000u;
    *nan_rows = 0;
    for (int r = 0; r < kRows; ++r)
      *nan_rows += std::all_of(out + r * words, out + (r + 1) * words,
                               [&](uint32_t w) { return (w & nan) == nan; });
    *code = st.code;
    *where = st.where;
  });
}
