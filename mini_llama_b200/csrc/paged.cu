// paged.cu — append to and read from the paged Q4_0 KV cache.
//
// Append replaces, for many ragged sequences at once, what the single-sequence
// path does per token in three steps: rotate q and k (Rope, src/ops.cc:143-178),
// quantise, write the cache row (CudaKvCache::WriteDevice,
// src/cuda_kv_cache.cc:137-163). Per row at position p and pair (x0, x1) of
// index j:
//
//   x0' = x0 cos a - x1 sin a,  x1' = x0 sin a + x1 cos a,  a = p theta^(-2j/D)
//
// Angle, sine, cosine and rotation are kept in 64 bits and rounded once to
// fp32: at position 1e5 an fp32 angle is off by up to 4e-3 rad, and a key next to a
// code's border would fall on either side of it. Queries, which have no codes, take the
// same angles and the same rotation. Q4_0 codes then follow the reference quantiser's
// fp32 steps bit for bit.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "paged.cuh"
#include "synth.h"

namespace mlb {

namespace {

struct RopeRates {
  double rate[kPagedMaxHeadDim / 2];  // theta^(-2j/D)
};

constexpr int kAppendThreads = 128;
// CTAs per SM: 64 registers, or the 96 that a NeoX key's eight pairs need (left to the
// compiler, 80 to 128 registers: 256 rows 7.1 us instead of 5.7, 15878 rows 82 instead of 78).
constexpr int append_ctas(bool neox) { return neox ? 5 : 8; }
constexpr int kAppendWarps = kAppendThreads / 32;
constexpr int kAppendRows = kAppendWarps;  // rows per CTA of a read at most: one warp looks up each

template <class T>
struct AppendArgs {
  PagedCache cache;
  PagedSeqs seqs;
  const T *q, *k, *v;
  T* q_out;
  long long q_stride, k_stride, v_stride, q_out_stride;
  int n_heads, rope_type;
};

// A lane holds 8 consecutive dimensions of a head, so a head takes 4 G lanes and a
// warp several heads.
__device__ __forceinline__ int heads_per_warp(int g) { return 32 / (4 * g); }

// The sequence and position of a row, and the page that holds it.
struct RowPlace {
  int pos, page, slot;  // pos < 0: of no sequence, or padded; page < 0: not stored
};
__device__ __forceinline__ RowPlace place_of(const PagedCache& c, const PagedSeqs& q, int row) {
  RowPlace r = {-1, -1, 0};
  // while decoding, row s is sequence s: one look instead of a search
  int s = row;
  if (row >= q.n_seqs || q.row_offsets[row] != row || q.row_offsets[row + 1] != row + 1) {
    s = q.n_seqs > 0 ? paged_find_seq(q, row) : -1;
    if (s < 0 || s >= q.n_seqs) return r;
  }
  const long long pos = (long long)q.seq_lens[s] - q.row_offsets[s + 1] + row;
  if (pos < 0 || pos > 0x7fffffff) return r;  // more: offsets that decrease
  r.pos = (int)pos;
  const int logical = r.pos / c.page_size;
  r.slot = r.pos - logical * c.page_size;
  if (logical < q.max_pages) r.page = q.table[(size_t)s * q.max_pages + logical];
  if (r.page >= c.n_pages) r.page = -1;
  return r;
}

// Address of the 16-token block of (page, kv head) that holds `slot`.
__device__ __forceinline__ uint8_t* block_at(const PagedCache& c, int page, int head, int slot) {
  const size_t bb = paged_block_bytes(c.head_dim);
  const int bpp = c.page_size / kPagedBlock;
  return c.layer + (((size_t)page * c.kv + head) * bpp + slot / kPagedBlock) * bb;
}

// Byte offsets in a block of what lane li of a head holds for token tok: K's word,
// the first of V's two half words (the other is 16 G bytes on), the scales.
__device__ __forceinline__ int k_word(int g, int tok, int li) {
  return tok * 16 * g + (li & 3) * 4 * g + (li >> 2) * 4;
}
__device__ __forceinline__ int v_half(int g, int tok, int li) {
  return 256 * g + (tok >> 3) * 128 * g + ((li & 3) * 8 + ((tok & 7) >> 1)) * 4 * g +
         (li >> 2) * 4 + (tok & 1) * 2;
}
__device__ __forceinline__ int scale_half(int g, int tok, int li, bool value) {
  return (value ? 544 : 512) * g + (tok >> 1) * 4 * g + (li >> 2) * 4 + (tok & 1) * 2;
}

// Eight elements as they are in memory (kept so while they are on their way).
template <class T>
struct Raw8 {
  uint4 u[sizeof(T) / 2];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) u[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) u[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  // four from p, four from q
  __device__ __forceinline__ void load(const T* p, const T* q) {
    if constexpr (sizeof(T) == 4) {
      u[0] = *reinterpret_cast<const uint4*>(p);
      u[1] = *reinterpret_cast<const uint4*>(q);
    } else {
      const uint2 a = *reinterpret_cast<const uint2*>(p), b = *reinterpret_cast<const uint2*>(q);
      u[0] = make_uint4(a.x, a.y, b.x, b.y);
    }
  }
  __device__ __forceinline__ void widen(float (&x)[8]) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        x[4 * i] = __uint_as_float(u[i].x), x[4 * i + 1] = __uint_as_float(u[i].y);
        x[4 * i + 2] = __uint_as_float(u[i].z), x[4 * i + 3] = __uint_as_float(u[i].w);
      }
    } else {
      const uint32_t w[4] = {u[0].x, u[0].y, u[0].z, u[0].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  }
};
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&x)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]),
                                            pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
}

__device__ __forceinline__ void store8(float* p, float* q, const float (&x)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  *reinterpret_cast<float4*>(q) = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, __nv_bfloat16* q, const float (&x)[8]) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
  *reinterpret_cast<uint2*>(q) = make_uint2(pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
}

// A query head's eight elements of lane li. NeoX pairs dimension j with j + D/2: there a
// lane holds 4 li .. 4 li + 3 and their partners, so that it needs no other lane (a
// third of the rotation's conversions less; codes need eight dimensions in a row).
template <bool NEOX, class T>
__device__ __forceinline__ void load_query(Raw8<T>& r, const T* head, int head_dim, int li) {
  if constexpr (NEOX)
    r.load(head + 4 * li, head + head_dim / 2 + 4 * li);
  else
    r.load(head + 8 * li);
}
template <bool NEOX, class T>
__device__ __forceinline__ void store_query(T* head, int head_dim, int li, const float (&x)[8]) {
  if constexpr (NEOX)
    store8(head + 4 * li, head + head_dim / 2 + 4 * li, x);
  else
    store8(head + 8 * li, x);
}

// The (cos, sin) pair of a key head's dimension d.
template <bool NEOX>
__device__ __forceinline__ int key_pair(int d, int head_dim) {
  return !NEOX ? d / 2 : d < head_dim / 2 ? d : d - head_dim / 2;
}

// Rotation of a query head's elements as load_query brings them (NeoX: e with e + 4),
// or of eight dimensions in a row in pairs.
template <bool NEOX>
__device__ __forceinline__ void rotate_query(float (&x)[8], const double2 (&turn)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int e = NEOX ? i : 2 * i, f = NEOX ? i + 4 : 2 * i + 1;
    const double2 t = turn[i];
    const double a = x[e], b = x[f];
    x[e] = (float)(a * t.x - b * t.y);
    x[f] = (float)(a * t.y + b * t.x);
  }
}

// Rotation of a key head's dimensions 8 li .. 8 li + 7 by pair(i): without NeoX the
// i-th pair of dimensions, else that of the i-th dimension. lane0 is the first lane of
// the head. All lanes of the warp call it.
template <bool NEOX, class F>
__device__ __forceinline__ void rotate_key(float (&x)[8], int head_dim, int lane0, int li,
                                           F pair) {
  if constexpr (!NEOX) {
    if (8 * li >= head_dim) return;
    const double2 turn[4] = {pair(0), pair(1), pair(2), pair(3)};
    rotate_query<false>(x, turn);
  } else {
    // element e pairs with another lane's e, or e ^ 4 where D/2 is no multiple of 8
    const int half = head_dim / 2;
    const bool cross = half % 8 != 0;
    float o[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int d = 8 * li + e;
      const int from = d < half ? d + half : d - half;
      o[e] = __shfl_sync(0xffffffffu, cross ? x[e ^ 4] : x[e], lane0 + from / 8);
    }
    if (8 * li >= head_dim) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int d = 8 * li + e;
      const bool first = d < half;
      const double2 t = pair(e);
      const double a = x[e], b = o[e];
      x[e] = (float)(a * t.x + (first ? -b : b) * t.y);
    }
  }
}

// Q4_0 of a lane's quarter of a block of 32: its eight codes and the block's scale
// (fp16 bits). The reference quantiser's fp32 steps; its fp16 rounds halves up, which
// for normal numbers is one addition.
__device__ __forceinline__ uint32_t quantise8(const float (&x)[8], uint32_t& scale) {
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(x[i]));
  amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
  amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
  const float want = __fdiv_rn(amax, 7.0f);
  float sd;
  if (want >= 6.103515625e-05f) {  // 2^-14
    // a scale past fp16 stays its largest number: what is stored is always finite
    const uint32_t u = min((__float_as_uint(want) + 0x1000u) >> 13, 0x7bffu + (112u << 10));
    scale = u - (112u << 10);
    sd = __uint_as_float(u << 13);
  } else {
    scale = synth::float_to_half_ref(want);
    sd = synth::half_to_float((uint16_t)scale);
  }
  const float inv = sd == 0.0f ? 0.0f : __frcp_rn(sd);
  uint32_t code = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    // round(v) of v = x / d + 8 with halves up, as floor(v + 1/2): 1.5 * 2^22 + 1/2 + v
    // rounded down to a half leaves twice that in the low bits (v >= 0.99 unless the
    // scale was cut, and then v below 0 counts as 0)
    const float v = fminf(fmaxf(__fadd_rn(__fmul_rn(x[i], inv), 8.0f), 0.0f), 15.0f);
    code |= (__float_as_uint(__fadd_rd(v, 6291456.5f)) >> 1 & 15u) << (4 * i);
  }
  return code;
}

// Codes and scale of lane li of a head's K or V into the token's place in its block.
__device__ __forceinline__ void store_codes(uint8_t* block, int g, int tok, int li, bool value,
                                            uint32_t code, uint32_t scale) {
  if (value) {
    uint8_t* p = block + v_half(g, tok, li);
    *reinterpret_cast<uint16_t*>(p) = (uint16_t)code;
    *reinterpret_cast<uint16_t*>(p + 16 * g) = (uint16_t)(code >> 16);
  } else {
    *reinterpret_cast<uint32_t*>(block + k_word(g, tok, li)) = code;
  }
  if ((li & 3) == 0)
    *reinterpret_cast<uint16_t*>(block + scale_half(g, tok, li, value)) = (uint16_t)scale;
}

// Few rows: one CTA per row (blockIdx.x) and share of the heads (blockIdx.y). The
// warps take turns of some heads of q, k or v each, two of them on their way ahead of
// the one at work and ahead of the row's place and rotation. Bound by that chain of
// latencies: 3.7 us for one row (a launch alone takes 2.5), 5 to 6 us for 64.
template <class T, bool NEOX>
__global__ void __launch_bounds__(kAppendThreads, append_ctas(NEOX))
    paged_append_kernel(AppendArgs<T> a, RopeRates rates) {
  __shared__ double2 cs[kPagedMaxHeadDim / 2];
  __shared__ RowPlace place;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row = blockIdx.x;
  const int D = a.cache.head_dim, g = paged_groups(D);
  const int H = a.n_heads, KV = a.cache.kv;
  const int hpw = heads_per_warp(g), hw = lane / (4 * g), li = lane - hw * 4 * g;
  const bool on = hw < hpw && 8 * li < D;
  // the row's turns: q's, then k's, then v's
  const int tq = (H + hpw - 1) / hpw, tk = (KV + hpw - 1) / hpw, turns = tq + 2 * tk;
  const int step = gridDim.y * kAppendWarps;
  const int first = blockIdx.y * kAppendWarps + warp;
  auto load = [&](Raw8<T>& x, int lt) {
    x.clear();
    if (lt >= turns) return;
    const bool is_q = lt < tq, is_v = lt >= tq + tk;
    const int h = (is_q ? lt : is_v ? lt - tq - tk : lt - tq) * hpw + hw;
    const T* p = (is_q ? a.q : is_v ? a.v : a.k) + h * D +
                 (long long)row * (is_q ? a.q_stride : is_v ? a.v_stride : a.k_stride);
    if (!on || h >= (is_q ? H : KV)) return;
    if (is_q)
      load_query<NEOX>(x, p, D, li);
    else
      x.load(p + 8 * li);
  };
  Raw8<T> raw[2];
  load(raw[0], first);
  load(raw[1], first + step);

  if (warp == 0) {
    const RowPlace p = place_of(a.cache, a.seqs, row);
    if (lane == 0) place = p;
  }
  __syncthreads();
  const RowPlace at = place;
  if (at.pos < 0) return;
  const bool rope = a.rope_type != MLB_ROPE_NONE;
  if (rope) {
    for (int j = threadIdx.x; j < D / 2; j += kAppendThreads) {
      double sn, c;
      sincos((double)at.pos * rates.rate[j], &sn, &c);
      cs[j] = make_double2(c, sn);
    }
    __syncthreads();
  }
  double2 turn[4];  // pairs 4 li .. 4 li + 3
  if (rope && on)
#pragma unroll
    for (int i = 0; i < 4; ++i) turn[i] = cs[4 * li + i];
  for (int t = first; t < turns; t += step) {
    float x[8];
    raw[0].widen(x);
    raw[0] = raw[1];
    load(raw[1], t + 2 * step);
    if (t < tq) {
      const int h = t * hpw + hw;
      if (!on || h >= H) continue;
      if (rope) rotate_query<NEOX>(x, turn);
      store_query<NEOX>(a.q_out + (long long)row * a.q_out_stride + h * D, D, li, x);
      continue;
    }
    if (at.page < 0) continue;
    if (t < tq + tk && rope)  // few keys per warp: from shared memory
      rotate_key<NEOX>(x, D, hw * 4 * g, li, [&](int i) {
        return NEOX ? cs[key_pair<NEOX>(8 * li + i, D)] : turn[i & 3];
      });
    uint32_t scale;
    const uint32_t code = quantise8(x, scale);
    const bool value = t >= tq + tk;
    const int kh = (t - tq - (value ? tk : 0)) * hpw + hw;
    if (kh >= KV || hw >= hpw) continue;
    store_codes(block_at(a.cache, at.page, kh, at.slot), g, at.slot % kPagedBlock, li, value, code,
                scale);
  }
}

// Many rows: one warp per row, so that its place and a lane's rotation are made once
// for all heads, and every address is a step from the one before. 15878 bf16 rows of
// 32 + 8 + 8 heads of 128: 78 us, 3.9 TB/s (the form for few rows with four rows per
// CTA: 119 us). Bound by latency and the conversions to and from 64 bits (four per pair
// of dimensions, 16 a cycle per SM: half of the time on their unit; issue slots 53 %).
template <class T, bool NEOX>
__global__ void __launch_bounds__(kAppendThreads, append_ctas(NEOX))
    paged_append_rows_kernel(AppendArgs<T> a, RopeRates rates) {
  constexpr int AHEAD = sizeof(T) == 2 ? 4 : 2;  // 64 bytes per lane on their way
  __shared__ double2 cs[kAppendWarps][kPagedMaxHeadDim / 2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long row = (long long)blockIdx.x * kAppendWarps + warp;
  if (row >= a.seqs.n_rows) return;
  const int D = a.cache.head_dim, g = paged_groups(D);
  const int H = a.n_heads, KV = a.cache.kv;
  const int hpw = heads_per_warp(g), hw = lane / (4 * g), li = lane - hw * 4 * g;
  const bool on = hw < hpw && 8 * li < D;
  const RowPlace at = place_of(a.cache, a.seqs, (int)row);
  if (at.pos < 0) return;
  const bool rope = a.rope_type != MLB_ROPE_NONE;
  if (rope) {
    for (int j = lane; j < D / 2; j += 32) {
      double sn, c;
      sincos((double)at.pos * rates.rate[j], &sn, &c);
      cs[warp][j] = make_double2(c, sn);
    }
    __syncwarp();
  }
  // f(elements, head) of the row's heads
  auto each = [&](const T* p, int heads, auto query, auto f) {
    constexpr bool QUERY = decltype(query)::value;
    p += hw * D;
    for (int h = hw; h - hw < heads; h += AHEAD * hpw) {
      Raw8<T> raw[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        raw[i].clear();
        if (on && h + i * hpw < heads) {
          if constexpr (QUERY)
            load_query<NEOX>(raw[i], p + i * hpw * D, D, li);
          else
            raw[i].load(p + i * hpw * D + 8 * li);
        }
      }
      p += AHEAD * hpw * D;
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        if (h - hw + i * hpw >= heads) break;
        float x[8];
        raw[i].widen(x);
        f(x, h + i * hpw);
      }
    }
  };
  T* q_out = a.q_out + row * a.q_out_stride;
  double2 turn[4];  // pairs 4 li .. 4 li + 3
  if (rope && on)
#pragma unroll
    for (int i = 0; i < 4; ++i) turn[i] = cs[warp][4 * li + i];
  each(a.q + row * a.q_stride, H, std::true_type{}, [&](float (&x)[8], int h) {
    if (rope) rotate_query<NEOX>(x, turn);
    if (on && h < H) store_query<NEOX>(q_out + h * D, D, li, x);
  });
  if (at.page < 0) return;
  uint8_t* block = block_at(a.cache, at.page, 0, at.slot);
  const size_t head_bytes = block_at(a.cache, 0, 1, 0) - block_at(a.cache, 0, 0, 0);
  const int tok = at.slot % kPagedBlock;
  auto keep = [&](float (&x)[8], int h, bool value) {
    uint32_t scale;
    const uint32_t code = quantise8(x, scale);
    if (hw < hpw && h < KV) store_codes(block + h * head_bytes, g, tok, li, value, code, scale);
  };
  // a NeoX lane's eight pairs are 128 bytes from the next lane's: fetched once for all
  // heads (from shared memory each time: 110 -> 153 us for 8192 fp32 rows of 64 heads)
  double2 key[NEOX ? 8 : 4];
  if (rope && on)
#pragma unroll
    for (int i = 0; i < (NEOX ? 8 : 4); ++i)
      key[i] = NEOX ? cs[warp][key_pair<NEOX>(8 * li + i, D)] : turn[i & 3];
  each(a.k + row * a.k_stride, KV, std::false_type{}, [&](float (&x)[8], int h) {
    if (rope) rotate_key<NEOX>(x, D, hw * 4 * g, li, [&](int i) { return key[i]; });
    keep(x, h, false);
  });
  each(a.v + row * a.v_stride, KV, std::false_type{},
       [&](float (&x)[8], int h) { keep(x, h, true); });
}

// Rows read back as the fp32 values their codes stand for; rows that are not
// stored are zeros. One CTA per `rows` rows and share of the heads, as above.
__global__ void __launch_bounds__(kAppendThreads)
    paged_read_kernel(PagedCache c, PagedSeqs seqs, int rows, float* k_out, float* v_out) {
  __shared__ RowPlace places[kAppendRows];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row0 = blockIdx.x * rows, n_rows = min(rows, seqs.n_rows - row0);
  const int D = c.head_dim, g = paged_groups(D);
  const int hpw = heads_per_warp(g), hw = lane / (4 * g), li = lane - hw * 4 * g;
  if (warp < n_rows) {
    const RowPlace p = place_of(c, seqs, row0 + warp);
    if (lane == 0) places[warp] = p;
  }
  __syncthreads();
  if (hw >= hpw || 8 * li >= D) return;
  const int turns = (2 * c.kv + hpw - 1) / hpw, total = turns * n_rows;
#pragma unroll 4
  for (int it = blockIdx.y * kAppendWarps + warp; it < total; it += gridDim.y * kAppendWarps) {
    const int r = it / turns, h = (it - r * turns) * hpw + hw;
    if (h >= 2 * c.kv) continue;
    const RowPlace at = places[r];
    const bool value = h >= c.kv;
    const int kh = value ? h - c.kv : h, tok = at.slot % kPagedBlock;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 0.0f;
    if (at.pos >= 0 && at.page >= 0) {
      const uint8_t* block = block_at(c, at.page, kh, at.slot);
      uint32_t code;
      if (value) {
        const uint8_t* p = block + v_half(g, tok, li);
        code = *reinterpret_cast<const uint16_t*>(p) |
               (uint32_t) * reinterpret_cast<const uint16_t*>(p + 16 * g) << 16;
      } else {
        code = *reinterpret_cast<const uint32_t*>(block + k_word(g, tok, li));
      }
      const float d = __half2float(
          *reinterpret_cast<const __half*>(block + scale_half(g, tok, li, value)));
      // 2^23 + q as a float has q in its low bits
#pragma unroll
      for (int i = 0; i < 8; ++i)
        x[i] = (__uint_as_float(0x4b000000u | (code >> (4 * i) & 15u)) - 8388616.0f) * d;
    }
    store8((value ? v_out : k_out) + ((size_t)(row0 + r) * c.kv + kh) * D + 8 * li, x);
  }
}

// CTAs per row: one while the rows alone fill the GPU, more (down to one turn per
// warp) when they do not, so that a single token's heads run side by side.
int head_shares(int rows, int heads, int head_dim, int sms) {
  const int turn = kAppendWarps * (32 / (4 * paged_groups(head_dim)));
  const int most = (heads + turn - 1) / turn;
  return std::max(1, std::min(most, 8 * sms / std::max(rows, 1)));
}

bool many_rows(int rows, int sms) { return rows >= 8 * sms; }

template <class T>
void launch_append(const PagedCache& c, const PagedSeqs& s, const void* k, long long k_stride,
                   const void* v, long long v_stride, const void* q, long long q_stride,
                   int n_heads, void* q_out, long long q_out_stride, float theta, int rope_type,
                   int device_id, cudaStream_t stream) {
  AppendArgs<T> a;
  a.cache = c;
  a.seqs = s;
  a.q = static_cast<const T*>(q);
  a.k = static_cast<const T*>(k);
  a.v = static_cast<const T*>(v);
  a.q_out = static_cast<T*>(q_out);
  a.q_stride = q_stride;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.q_out_stride = q_out_stride;
  a.n_heads = n_heads;
  a.rope_type = rope_type;
  RopeRates r = {};
  if (rope_type != MLB_ROPE_NONE)
    for (int j = 0; j < c.head_dim / 2; ++j)
      r.rate[j] = std::pow((double)theta, -2.0 * j / c.head_dim);
  // a warp per row once that gives every scheduler two: 32 bf16 heads, NeoX, few / many
  // us: 512 rows 10.7 / 11.0, 1024 15.8 / 12.3, 4096 45 / 29; without NeoX 1024 rows
  // 9.8 / 10.8, 2048 15.8 / 15.0, 4096 27.8 / 24.2
  const int sms = sm_count(device_id);
  const bool neox = rope_type == MLB_ROPE_NEOX;
  if (many_rows(s.n_rows, sms)) {
    auto kernel = neox ? paged_append_rows_kernel<T, true> : paged_append_rows_kernel<T, false>;
    kernel<<<(s.n_rows + kAppendWarps - 1) / kAppendWarps, kAppendThreads, 0, stream>>>(a, r);
  } else {
    const int shares = head_shares(s.n_rows, n_heads + 2 * c.kv, c.head_dim, sms);
    auto kernel = neox ? paged_append_kernel<T, true> : paged_append_kernel<T, false>;
    kernel<<<dim3(s.n_rows, shares), kAppendThreads, 0, stream>>>(a, r);
  }
  MLB_CUDA(cudaGetLastError());
}

}  // namespace

}  // namespace mlb

using namespace mlb;

extern "C" int mlb_paged_kv_page_bytes(int page_size, int n_kv_heads, int head_dim,
                                       size_t* bytes) {
  return guarded([&] {
    if (!bytes) invalid("mlb_paged_kv_page_bytes: null output");
    paged_check_shape("mlb_paged_kv_page_bytes", page_size, n_kv_heads, head_dim);
    *bytes = paged_page_bytes(page_size, n_kv_heads, head_dim);
  });
}

extern "C" int mlb_paged_kv_append(void* pages, int n_layers, int n_pages, int page_size,
                                   int n_kv_heads, int head_dim, int layer, int act_type,
                                   const void* k, long long k_stride, const void* v,
                                   long long v_stride, const void* q, long long q_stride,
                                   int n_heads, void* q_out, long long q_out_stride, int n_rows,
                                   int n_seqs, const int* row_offsets, const int* seq_lens,
                                   const int* page_table, int max_pages, float theta,
                                   int rope_type, int device_id, void* stream) {
  return guarded([&] {
    const char* who = "CudaPagedKvCache";
    const PagedCache c =
        paged_cache(who, pages, n_layers, n_pages, page_size, n_kv_heads, head_dim, layer);
    const PagedSeqs s = paged_seqs(who, n_rows, n_seqs, row_offsets, seq_lens, page_table,
                                   max_pages, page_size);
    paged_check_act(who, act_type);
    if (rope_type != MLB_ROPE_NONE && rope_type != MLB_ROPE_NORMAL && rope_type != MLB_ROPE_NEOX)
      invalid("CudaPagedKvCache: unknown rope type " + std::to_string(rope_type));
    if (rope_type != MLB_ROPE_NONE && (!(theta > 0.0f) || !std::isfinite(theta)))
      invalid("Rope: theta must be finite and positive");
    if (n_heads < 0) invalid("CudaPagedKvCache: negative head count");
    if (n_rows > 0) {
      paged_check_rows(who, "k", k, k_stride, n_kv_heads, head_dim, act_type);
      paged_check_rows(who, "v", v, v_stride, n_kv_heads, head_dim, act_type);
      if (n_heads > 0) {
        paged_check_rows(who, "q", q, q_stride, n_heads, head_dim, act_type);
        paged_check_rows(who, "q_out", q_out, q_out_stride, n_heads, head_dim, act_type);
        // a row's q is read by the lanes that write it; other rows have no such order
        const long long row = (long long)n_heads * head_dim;
        const long long kv_row = (long long)n_kv_heads * head_dim;
        const bool in_place = q == q_out && (q_stride == q_out_stride || n_rows == 1);
        if (!in_place && rows_overlap(q, q_stride, row, q_out, q_out_stride, row, n_rows, act_type))
          invalid("CudaPagedKvCache: q_out must be q itself or not overlap it");
        if (rows_overlap(k, k_stride, kv_row, q_out, q_out_stride, row, n_rows, act_type) ||
            rows_overlap(v, v_stride, kv_row, q_out, q_out_stride, row, n_rows, act_type))
          invalid("CudaPagedKvCache: q_out must not overlap k or v");
      }
    }
    DeviceScope scope(device_id);
    if (n_rows == 0 || n_seqs == 0) return;
    (act_type == MLB_ACT_BF16 ? launch_append<__nv_bfloat16> : launch_append<float>)(
        c, s, k, k_stride, v, v_stride, q, q_stride, n_heads, q_out, q_out_stride, theta,
        rope_type, device_id, static_cast<cudaStream_t>(stream));
  });
}

extern "C" int mlb_paged_kv_read(const void* pages, int n_layers, int n_pages, int page_size,
                                 int n_kv_heads, int head_dim, int layer, int n_rows, int n_seqs,
                                 const int* row_offsets, const int* seq_lens,
                                 const int* page_table, int max_pages, float* k_out, float* v_out,
                                 int device_id, void* stream) {
  return guarded([&] {
    const char* who = "CudaPagedKvCache";
    const PagedCache c = paged_cache(who, const_cast<void*>(pages), n_layers, n_pages, page_size,
                                     n_kv_heads, head_dim, layer);
    const PagedSeqs s = paged_seqs(who, n_rows, n_seqs, row_offsets, seq_lens, page_table,
                                   max_pages, page_size);
    if (n_rows > 0) {
      const long long stride = (long long)n_kv_heads * head_dim;
      paged_check_rows(who, "k_out", k_out, stride, n_kv_heads, head_dim, MLB_ACT_F32);
      paged_check_rows(who, "v_out", v_out, stride, n_kv_heads, head_dim, MLB_ACT_F32);
      if (rows_overlap(k_out, stride, stride, v_out, stride, stride, n_rows, MLB_ACT_F32))
        invalid("CudaPagedKvCache: k_out and v_out must not overlap");
    }
    DeviceScope scope(device_id);
    if (n_rows == 0) return;
    const int sms = sm_count(device_id);
    const int rows = many_rows(n_rows, sms) ? kAppendRows : 1;
    const int shares = head_shares(n_rows, 2 * n_kv_heads, head_dim, sms);
    paged_read_kernel<<<dim3((n_rows + rows - 1) / rows, shares), kAppendThreads, 0,
                        static_cast<cudaStream_t>(stream)>>>(c, s, rows, k_out, v_out);
    MLB_CUDA(cudaGetLastError());
  });
}
