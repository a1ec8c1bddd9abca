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

#include <string>

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
  if (reinterpret_cast<uintptr_t>(p) % 16 != 0 || (stride * es) % 16 != 0)
    invalid(w + ": rows of " + name + " must be 16-byte aligned");
}

inline void paged_check_act(const char* who, int act) {
  if (act != MLB_ACT_F32 && act != MLB_ACT_BF16)
    invalid(std::string(who) + ": unknown activation type " + std::to_string(act));
}

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

#endif  // __CUDACC__

}  // namespace mlb
