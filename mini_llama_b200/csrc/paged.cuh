// paged.cuh — the paged Q4_0 KV cache: its layout and the argument checks and
// device helpers that the append, read and attention kernels share.
//
// A page holds page_size tokens (whole blocks of 16) of every KV head. Per
// (page, KV head) the 16-token blocks follow one another, each 576 * G bytes,
// G = ceil(head_dim / 32) quantisation groups per row (dimensions past head_dim
// are stored as zeros):
//
//   [0, 256 G)      K codes: token t at 16 G t; in it chunk c of 4 (4 G bytes),
//                   word w = dims 32 w + 8 c + 0..7, one nibble each, lowest first
//   [256 G, 512 G)  V codes: word w of slot (t >> 3, g, (t & 7) >> 1) holds dims
//                   32 w + 4 g + 0..3 of token t (t even: low half, odd: high half)
//   [512 G, 544 G)  K scales (fp16): word w of token pair t >> 1, half t & 1
//   [544 G, 576 G)  V scales, the same
//
// Every lane of a warp finds its mma.sync m16n8k16 fragments of one block in G
// consecutive words of each part (lane = 4 g + c: K operand column g, V operand
// row g, contraction / token pair c), so a block goes from memory to the tensor
// cores without a shuffle, and no byte is shared by two tokens, so an append
// never has to merge with what is there.
//
// A code q stands for (q - 8) * d, the GGUF Q4_0 block of the reference
// (include/mini_llama/quantized_tensor.h:26-44), quantised with the steps of its
// QuantizeToQ40 (src/quant.cc:201-276).
#pragma once

#include <cuda_bf16.h>

#include <map>
#include <mutex>
#include <string>
#include <utility>

#include "common.cuh"

namespace mlb {

constexpr int kPagedBlock = 16;  // tokens per block
constexpr int kPagedMaxHeadDim = 128;

// One layer of a cache (fewer than 2^31 blocks) and the sequences of a call.
struct PagedSeqs {
  const int* row_offsets;  // [n_seqs + 1]
  const int* seq_lens;     // [n_seqs], the call's rows included
  const int* table;        // [n_seqs, max_pages]
  int n_seqs, max_pages, n_rows;
};
struct PagedCache {
  uint8_t* layer;  // first page of the layer
  int n_pages, page_size, kv, head_dim;
};

__host__ __device__ inline int paged_groups(int head_dim) { return (head_dim + 31) / 32; }
__host__ __device__ inline size_t paged_block_bytes(int head_dim) {
  return (size_t)576 * paged_groups(head_dim);
}
__host__ __device__ inline size_t paged_page_bytes(int page_size, int kv, int head_dim) {
  return (size_t)(page_size / kPagedBlock) * kv * paged_block_bytes(head_dim);
}

// Shape checks shared by the entry points.
inline void paged_check_shape(const char* who, int page_size, int kv, int head_dim) {
  const std::string w = who;
  if (page_size <= 0 || page_size % kPagedBlock != 0)
    invalid(w + ": page_size must be a positive multiple of 16, got " + std::to_string(page_size));
  if (kv <= 0) invalid(w + ": n_kv_heads must be positive");
  if (head_dim <= 0 || head_dim % 8 != 0 || head_dim > kPagedMaxHeadDim)
    invalid(w + ": head_dim must be a multiple of 8 up to 128, got " + std::to_string(head_dim));
}

inline PagedCache paged_cache(const char* who, void* pages, int n_layers, int n_pages,
                              int page_size, int kv, int head_dim, int layer) {
  const std::string w = who;
  if (!pages || n_layers <= 0 || n_pages <= 0) invalid(w + ": paged KV cache is empty");
  paged_check_shape(who, page_size, kv, head_dim);
  if (layer < 0 || layer >= n_layers) out_of_range(w + ": layer out of range");
  if (reinterpret_cast<uintptr_t>(pages) % 16 != 0)
    invalid(w + ": pages must be 16-byte aligned");
  if ((long long)n_pages * kv * (page_size / kPagedBlock) >= (1LL << 31))
    invalid(w + ": a layer must have fewer than 2^31 blocks of 16 tokens");
  PagedCache c;
  c.layer = static_cast<uint8_t*>(pages) +
            (size_t)layer * n_pages * paged_page_bytes(page_size, kv, head_dim);
  c.n_pages = n_pages;
  c.page_size = page_size;
  c.kv = kv;
  c.head_dim = head_dim;
  return c;
}

inline PagedSeqs paged_seqs(const char* who, int n_rows, int n_seqs, const int* row_offsets,
                            const int* seq_lens, const int* table, int max_pages, int page_size) {
  const std::string w = who;
  if (n_rows < 0 || n_seqs < 0) invalid(w + ": negative row or sequence count");
  if (max_pages <= 0) invalid(w + ": page_table must have at least one column");
  // positions are 32-bit; leave room for the last tile's rounding up
  if ((long long)max_pages * page_size > 2000000000LL)
    invalid(w + ": page_table covers more than 2e9 positions");
  if (n_rows > 0 && n_seqs > 0 && (!row_offsets || !seq_lens || !table))
    invalid(w + ": null row_offsets, seq_lens or page_table");
  PagedSeqs s;
  s.row_offsets = row_offsets;
  s.seq_lens = seq_lens;
  s.table = table;
  s.n_seqs = n_seqs;
  s.max_pages = max_pages;
  s.n_rows = n_rows;
  return s;
}

// Rows of `heads` x head_dim elements read or written 16 bytes at a time.
inline void paged_check_rows(const char* who, const char* name, const void* p, long long stride,
                             int heads, int head_dim, int act) {
  const std::string w = who;
  const int es = act == MLB_ACT_BF16 ? 2 : 4;
  if (!p) invalid(w + ": null " + name);
  if (stride < (long long)heads * head_dim)
    invalid(w + ": row stride of " + name + " is smaller than a row");
  if (reinterpret_cast<uintptr_t>(p) % 16 != 0 || stride % (16 / es) != 0)
    invalid(w + ": rows of " + name + " must be 16-byte aligned");
}

// Whether two sets of n rows share a byte: rows of a_row (b_row) elements,
// a_row_stride (b_row_stride) apart, at least a row. Rows side by side in one buffer do not.
inline bool rows_overlap(const void* a, long long a_row_stride, long long a_row, const void* b,
                         long long b_row_stride, long long b_row, int n, int act) {
  using wide = __int128;  // strides are the caller's
  const int es = act == MLB_ACT_BF16 ? 2 : 4;
  const wide a_stride = (wide)a_row_stride * es, b_stride = (wide)b_row_stride * es;
  const wide a_bytes = (wide)a_row * es, b_bytes = (wide)b_row * es;
  const wide d = (wide)reinterpret_cast<uintptr_t>(b) - (wide)reinterpret_cast<uintptr_t>(a);
  const auto floor_div = [](wide x, wide y) { return x / y - (x % y < 0 ? 1 : 0); };
  // rows of b that row i of a meets: those with i a_stride - j b_stride - d in (-a_bytes, b_bytes)
  const auto meets = [&](wide at, wide j0, wide j1) {
    const wide lo = floor_div(at - d - b_bytes, b_stride) + 1;
    const wide hi = floor_div(at - d + a_bytes - 1, b_stride);
    return (lo > j0 ? lo : j0) <= (hi < j1 ? hi : j1);
  };
  if (n <= 0) return false;
  // of equal strides only the difference of the rows counts
  if (a_stride == b_stride) return meets(0, -(wide)(n - 1), n - 1);
  if (d >= (wide)(n - 1) * a_stride + a_bytes || -d >= (wide)(n - 1) * b_stride + b_bytes)
    return false;
  for (int i = 0; i < n; ++i)
    if (meets((wide)i * a_stride, 0, n - 1)) return true;
  return false;
}

inline void paged_check_act(const char* who, int act) {
  if (act != MLB_ACT_F32 && act != MLB_ACT_BF16)
    invalid(std::string(who) + ": unknown activation type " + std::to_string(act));
}

// Lets a kernel use `bytes` of dynamic shared memory, once per kernel and device.
template <class K>
inline void allow_smem(K kernel, size_t bytes, int device_id) {
  static std::mutex mu;
  static std::map<std::pair<const void*, int>, bool> seen;
  std::lock_guard<std::mutex> lock(mu);
  bool& s = seen[{reinterpret_cast<const void*>(kernel), device_id}];
  if (s) return;
  MLB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
  s = true;
}

// Arguments of the attention kernels.
struct PagedAttnArgs {
  PagedCache cache;
  PagedSeqs seqs;
  const void* q;
  void* out;
  long long q_stride, out_stride;
  int n_heads, group;
  float scale_log2;  // scale * log2(e)
  bool whole;        // decode form: no unit is cut between CTAs (and neither of these is used)
  int4* split;       // decode form, per CTA: {parts, first record, head, tile}, {row0, rows}
  float* partial;    // decode form, per CTA: two records of R x (32 G) + 2 R floats
  long long wait_cycles;  // prompt form: limit of a wait
  int never;              // prompt form: arrivals that K's barriers wait for in vain (self-test)
};

// Prompt form (paged_prompt.cu): many rows per sequence.
void paged_prompt_launch(const PagedAttnArgs& a, int act_type, int device_id, cudaStream_t stream);

#if defined(__CUDACC__)

// One activation row's four elements from dimension d0 as fp32 (fp32 rows: one
// 16-byte load; bf16 rows: one 8-byte load).
__device__ __forceinline__ float4 load_act4(const float* p) {
  return *reinterpret_cast<const float4*>(p);
}
__device__ __forceinline__ float4 load_act4(const __nv_bfloat16* p) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u),
                     __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ void store_act4(float* p, const float4& v) {
  *reinterpret_cast<float4*>(p) = v;
}
__device__ __forceinline__ void store_act4(__nv_bfloat16* p, const float4& v) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
}

__device__ __forceinline__ void store_act2(float* p, float x, float y) {
  *reinterpret_cast<float2*>(p) = make_float2(x, y);
}
__device__ __forceinline__ void store_act2(__nv_bfloat16* p, float x, float y) {
  *reinterpret_cast<uint32_t*>(p) = pack_bf16(x, y);
}

// The sequence that row r belongs to: the last s with row_offsets[s] <= r, found
// by the whole warp 32 probes at a time. Negative or n_seqs: none.
__device__ __forceinline__ int paged_find_seq(const PagedSeqs& q, int r) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = q.n_seqs + 1;
  while (true) {
    const int step = (n + 31) / 32;
    const int i = lane * step;
    const bool le = i < n && q.row_offsets[lo + i] <= r;
    const int cnt = __popc(__ballot_sync(0xffffffffu, le));
    if (cnt == 0) return lo - 1;
    lo += (cnt - 1) * step;
    if (step == 1) return lo;
    n = min(step, n - (cnt - 1) * step);
  }
}

__device__ __forceinline__ uint32_t hsub2_u(uint32_t x, uint32_t y) {
  return h2_as_u32(__hsub2(u32_as_h2(x), u32_as_h2(y)));
}

// Eight 4-bit codes of a word as fp16 pairs (nibble i, nibble i + 4), minus 8.
// 1024 + q and 1024 + 16 q are exact fp16; the second form saves a shift.
__device__ __forceinline__ void codes_f16(uint32_t x, uint32_t (&r)[4]) {
  const uint32_t magic = 0x64006400u, bias = 0x64086408u;  // 1024, 1032
  const __half2 sixteenth = u32_as_h2(0x2C002C00u), m72 = u32_as_h2(0xD480D480u);
  const uint32_t y = x >> 8;
  r[0] = hsub2_u(lop3_and_or(x, 0x000F000Fu, magic), bias);
  r[1] = h2_as_u32(__hfma2(u32_as_h2(lop3_and_or(x, 0x00F000F0u, magic)), sixteenth, m72));
  r[2] = hsub2_u(lop3_and_or(y, 0x000F000Fu, magic), bias);
  r[3] = h2_as_u32(__hfma2(u32_as_h2(lop3_and_or(y, 0x00F000F0u, magic)), sixteenth, m72));
}

// Two fp32 at a time.
__device__ __forceinline__ float2 fma2(const float2& a, const float2& b, const float2& c) {
  float2 r;
  asm("{\n .reg .b64 a, b, c, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n"
      " mov.b64 c, {%6, %7};\n fma.rn.f32x2 d, a, b, c;\n mov.b64 {%0, %1}, d;\n}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 add2(const float2& a, const float2& b) {
  float2 r;
  asm("{\n .reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n"
      " add.rn.f32x2 d, a, b;\n mov.b64 {%0, %1}, d;\n}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 mul2(const float2& a, const float2& b) {
  float2 r;
  asm("{\n .reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n"
      " mul.rn.f32x2 d, a, b;\n mov.b64 {%0, %1}, d;\n}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}

__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Words of a query row: 8 dimensions from d0, zeros past head_dim.
template <class T>
__device__ __forceinline__ void load_q8(const T* p, float (&e)[8]) {
  const float4 a = load_act4(p), b = load_act4(p + 4);
  e[0] = a.x, e[1] = a.y, e[2] = a.z, e[3] = a.w;
  e[4] = b.x, e[5] = b.y, e[6] = b.z, e[7] = b.w;
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  return h2_as_u32(__floats2half2_rn(lo, hi));
}

// G consecutive 32-bit words of memory.
template <int G>
__device__ __forceinline__ void lds_words(const uint8_t* p, uint32_t (&w)[G]) {
  if constexpr (G == 4) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
  } else if constexpr (G == 2) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    w[0] = u.x, w[1] = u.y;
  } else {
#pragma unroll
    for (int i = 0; i < G; ++i) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
  }
}

// One row's query elements of this lane, dims 32 w + 8 c + 0..7 (zeros past head_dim
// and without a row).
template <int G, class T>
__device__ __forceinline__ void load_query_elements(const T* row, int head_dim, int c,
                                                    float (&e)[G][8]) {
#pragma unroll
  for (int w = 0; w < G; ++w) {
#pragma unroll
    for (int i = 0; i < 8; ++i) e[w][i] = 0.0f;
    const int d0 = 32 * w + 8 * c;
    if (row && d0 < head_dim) load_q8(row + d0, e[w]);
  }
}
// The exponent of the power of two that brings the row's largest element near 2^13.
template <int G>
__device__ __forceinline__ int query_shift(const float (&e)[G][8]) {
  float amax = 0.0f;
#pragma unroll
  for (int w = 0; w < G; ++w)
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(e[w][i]));
  amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
  amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
  const int ex = (int)(__float_as_uint(amax) >> 23);
  // zero rows, subnormal rows and infinities stay as they are
  return (ex == 0 || ex == 255) ? 0 : min(max(13 - (ex - 127), -126), 126);
}

// Eight elements times sf as fp16 words, word i = elements (i, i + 4), and for split
// what they leave.
__device__ __forceinline__ void query_words(const float (&e)[8], float sf, bool split,
                                            uint32_t (&hi)[4], uint32_t (&lo)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float x = e[i] * sf, y = e[i + 4] * sf;
    hi[i] = pack_f16(x, y);
    lo[i] = 0u;
    if (split) {
      const float2 h = __half22float2(u32_as_h2(hi[i]));
      lo[i] = pack_f16(x - h.x, y - h.y);
    }
  }
}

// What a sequence asks for: its rows in tiles of tile_rows (token, head) rows, its
// length in chunks of chunk_tokens, and what its units, one per (KV head, tile), take
// up in the runs: their chunks and unit_slots more, or 1 where they stay whole.
// Lengths and offsets are cut to what the page table and the call hold; pos0, the
// position of row row0, is not.
struct SeqWork {
  int len, n, row0, tiles, chunks, slots;
  long long pos0, cost;
};
// Positions that row row0 + i sees.
__device__ __forceinline__ int seen_by(long long pos0, int i, int len) {
  return (int)max(min(pos0 + i + 1, (long long)len), 0LL);
}

__device__ __forceinline__ SeqWork seq_work(const PagedAttnArgs& a, int s, int tile_rows,
                                            int chunk_tokens, int unit_slots) {
  SeqWork w;
  const int cap = a.seqs.max_pages * a.cache.page_size;
  const int len = a.seqs.seq_lens[s], row1 = a.seqs.row_offsets[s + 1];
  w.len = min(max(len, 0), cap);
  w.row0 = max(a.seqs.row_offsets[s], 0);
  w.n = max(min(max(row1, 0), a.seqs.n_rows) - w.row0, 0);  // no difference wraps
  w.pos0 = (long long)len - row1 + w.row0;
  w.tiles = (int)(((long long)w.n * a.group + tile_rows - 1) / tile_rows);
  w.chunks = max(1, (w.len + chunk_tokens - 1) / chunk_tokens);
  w.slots = a.whole ? 1 : w.chunks + unit_slots;
  w.cost = (long long)w.tiles * a.cache.kv * w.slots;
  return w;
}

// Inclusive block-wide scan of one value per thread; warp_sums: one per warp.
template <int THREADS>
__device__ __forceinline__ long long block_scan(long long v, long long* warp_sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  for (int w = 0; w < warp; ++w) v += warp_sums[w];
  __syncthreads();
  return v;
}
#endif  // __CUDACC__

}  // namespace mlb
