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
// fp32: at position 1e5 an fp32 angle is off by up to 4e-3 rad, and a value next
// to a code's border would fall on either side of it. Q4_0 codes then follow the
// reference quantiser's fp32 steps bit for bit.
#include <cmath>

#include "paged.cuh"
#include "synth.h"

namespace mlb {

namespace {

struct RopeRates {
  double rate[kPagedMaxHeadDim / 2];  // theta^(-2j/D)
};

constexpr int kAppendThreads = 256;

template <class T>
struct AppendArgs {
  PagedCache cache;
  PagedSeqs seqs;
  const T *q, *k, *v;
  T* q_out;
  long long q_stride, k_stride, v_stride, q_out_stride;
  int n_heads, rope_type;
};

// Address of the 16-token block of (page, kv head) that holds `slot`.
__device__ __forceinline__ uint8_t* block_at(const PagedCache& c, int page, int head, int slot) {
  const size_t bb = paged_block_bytes(c.head_dim);
  const int bpp = c.page_size / kPagedBlock;
  return c.layer + (((size_t)page * c.kv + head) * bpp + slot / kPagedBlock) * bb;
}

// One row's four values of this lane -> codes and, in the first lane of each
// group of 8, the scale.
__device__ __forceinline__ void store_q4(uint8_t* block, bool value, int g, int tok, int lane,
                                         const float4& x) {
  float amax = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  // a scale past fp16 stays its largest number: what is stored is always finite
  const uint16_t d = min((int)synth::float_to_half_ref(__fdiv_rn(amax, 7.0f)), 0x7bff);
  const float sd = synth::half_to_float(d);
  const float inv = sd == 0.0f ? 0.0f : __fdiv_rn(1.0f, sd);
  const float e[4] = {x.x, x.y, x.z, x.w};
  uint32_t code = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int q = synth::clampi((int)roundf(__fadd_rn(__fmul_rn(e[i], inv), 8.0f)), 0, 15);
    code |= (uint32_t)q << (4 * i);
  }
  const int w = lane >> 3;
  if (w >= g) return;
  uint8_t* at;
  if (!value) {
    at = block + (size_t)tok * 16 * g + ((lane & 7) >> 1) * 4 * g + w * 4 + (lane & 1) * 2;
  } else {
    at = block + 256 * g + (tok >> 3) * 128 * g + ((lane & 7) * 4 + ((tok & 7) >> 1)) * 4 * g +
         w * 4 + (tok & 1) * 2;
  }
  *reinterpret_cast<uint16_t*>(at) = (uint16_t)code;
  if ((lane & 7) == 0)
    *reinterpret_cast<uint16_t*>(block + (value ? 544 : 512) * g + (tok >> 1) * 4 * g + w * 4 +
                                 (tok & 1) * 2) = d;
}

// Rotation of this lane's dimensions 4 lane .. 4 lane + 3 with (cos, sin) pairs cs.
__device__ __forceinline__ float4 rotate4(const float4& x, int rope_type, int head_dim, int lane,
                                          const double2* cs) {
  if (rope_type == MLB_ROPE_NORMAL) {
    if (4 * lane >= head_dim) return x;
    const double2 a = cs[2 * lane], b = cs[2 * lane + 1];
    const double x0 = x.x, x1 = x.y, x2 = x.z, x3 = x.w;
    return make_float4((float)(x0 * a.x - x1 * a.y), (float)(x0 * a.y + x1 * a.x),
                       (float)(x2 * b.x - x3 * b.y), (float)(x2 * b.y + x3 * b.x));
  }
  // NeoX: dimension j pairs with j + D/2, D/8 lanes away
  const int hl = head_dim / 8;
  const bool first = lane < hl;
  const int src = first ? lane + hl : lane - hl;
  float4 o;
  o.x = __shfl_sync(0xffffffffu, x.x, src);
  o.y = __shfl_sync(0xffffffffu, x.y, src);
  o.z = __shfl_sync(0xffffffffu, x.z, src);
  o.w = __shfl_sync(0xffffffffu, x.w, src);
  if (4 * lane >= head_dim) return x;
  const double2* t = cs + 4 * (first ? lane : lane - hl);
  const double sg = first ? -1.0 : 1.0;
  return make_float4((float)(x.x * t[0].x + sg * o.x * t[0].y),
                     (float)(x.y * t[1].x + sg * o.y * t[1].y),
                     (float)(x.z * t[2].x + sg * o.z * t[2].y),
                     (float)(x.w * t[3].x + sg * o.w * t[3].y));
}

// One CTA per row (blockIdx.x) and share of the heads (blockIdx.y); one warp
// per (row, head), four dimensions per lane.
template <class T>
__global__ void __launch_bounds__(kAppendThreads)
    paged_append_kernel(AppendArgs<T> a, RopeRates rates) {
  __shared__ double2 cs[kPagedMaxHeadDim / 2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row = blockIdx.x;
  const int D = a.cache.head_dim;
  const int s = paged_find_seq(a.seqs, row);
  if (s < 0 || s >= a.seqs.n_seqs) return;
  const int pos = a.seqs.seq_lens[s] - a.seqs.row_offsets[s + 1] + row;
  if (pos < 0) return;
  if (a.rope_type != MLB_ROPE_NONE) {
    for (int j = threadIdx.x; j < D / 2; j += kAppendThreads) {
      double sn, c;
      sincos((double)pos * rates.rate[j], &sn, &c);
      cs[j] = make_double2(c, sn);
    }
    __syncthreads();
  }
  const int logical = pos / a.cache.page_size;
  const int slot = pos - logical * a.cache.page_size;
  int page = -1;
  if (logical < a.seqs.max_pages) page = a.seqs.table[(size_t)s * a.seqs.max_pages + logical];
  const bool stored = page >= 0 && page < a.cache.n_pages;
  const int g = paged_groups(D), tok = slot % kPagedBlock;
  const int KV = a.cache.kv, heads = a.n_heads + 2 * KV;
  const bool on = 4 * lane < D;
  const int nw = kAppendThreads / 32;
  for (int h = blockIdx.y * nw + warp; h < heads; h += gridDim.y * nw) {
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (h < a.n_heads) {
      if (on) x = load_act4(a.q + row * a.q_stride + (size_t)h * D + 4 * lane);
      if (a.rope_type != MLB_ROPE_NONE) x = rotate4(x, a.rope_type, D, lane, cs);
      if (on) store_act4(a.q_out + row * a.q_out_stride + (size_t)h * D + 4 * lane, x);
      continue;
    }
    if (!stored) continue;
    const bool value = h >= a.n_heads + KV;
    const int kh = h - a.n_heads - (value ? KV : 0);
    if (on)
      x = load_act4((value ? a.v + row * a.v_stride : a.k + row * a.k_stride) + (size_t)kh * D +
                    4 * lane);
    if (!value && a.rope_type != MLB_ROPE_NONE) x = rotate4(x, a.rope_type, D, lane, cs);
    store_q4(block_at(a.cache, page, kh, slot), value, g, tok, lane, x);
  }
}

// Rows read back as the fp32 values their codes stand for; rows that are not
// stored are zeros.
__global__ void __launch_bounds__(kAppendThreads)
    paged_read_kernel(PagedCache c, PagedSeqs seqs, float* k_out, float* v_out) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row = blockIdx.x;
  const int D = c.head_dim;
  const int s = seqs.n_seqs > 0 ? paged_find_seq(seqs, row) : -1;
  int page = -1, slot = 0;
  if (s >= 0 && s < seqs.n_seqs) {
    const int pos = seqs.seq_lens[s] - seqs.row_offsets[s + 1] + row;
    const int logical = pos / c.page_size;
    slot = pos - logical * c.page_size;
    if (pos >= 0 && logical < seqs.max_pages)
      page = seqs.table[(size_t)s * seqs.max_pages + logical];
  }
  const bool stored = page >= 0 && page < c.n_pages;
  const int g = paged_groups(D), tok = slot % kPagedBlock, w = lane >> 3;
  const int nw = kAppendThreads / 32;
  if (4 * lane >= D) return;
  for (int h = blockIdx.y * nw + warp; h < 2 * c.kv; h += gridDim.y * nw) {
    const bool value = h >= c.kv;
    const int kh = value ? h - c.kv : h;
    float* out = (value ? v_out : k_out) + ((size_t)row * c.kv + kh) * D + 4 * lane;
    if (!stored) {
      store_act4(out, make_float4(0.f, 0.f, 0.f, 0.f));
      continue;
    }
    const uint8_t* block = block_at(c, page, kh, slot);
    const uint8_t* at =
        value ? block + 256 * g + (tok >> 3) * 128 * g +
                    ((lane & 7) * 4 + ((tok & 7) >> 1)) * 4 * g + w * 4 + (tok & 1) * 2
              : block + (size_t)tok * 16 * g + ((lane & 7) >> 1) * 4 * g + w * 4 + (lane & 1) * 2;
    const uint32_t code = *reinterpret_cast<const uint16_t*>(at);
    const float d = __half2float(*reinterpret_cast<const __half*>(
        block + (value ? 544 : 512) * g + (tok >> 1) * 4 * g + w * 4 + (tok & 1) * 2));
    float4 x;
    x.x = (float)((int)(code & 15) - 8) * d;
    x.y = (float)((int)(code >> 4 & 15) - 8) * d;
    x.z = (float)((int)(code >> 8 & 15) - 8) * d;
    x.w = (float)((int)(code >> 12 & 15) - 8) * d;
    store_act4(out, x);
  }
}

// CTAs per row: one while the rows alone fill the GPU, more (down to one head
// per warp) when they do not, so that a single token's heads run side by side.
int head_shares(int rows, int heads, int sms) {
  const int most = (heads + kAppendThreads / 32 - 1) / (kAppendThreads / 32);
  return std::max(1, std::min(most, 4 * sms / std::max(rows, 1)));
}

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
  const int shares = head_shares(s.n_rows, n_heads + 2 * c.kv, sm_count(device_id));
  paged_append_kernel<T><<<dim3(s.n_rows, shares), kAppendThreads, 0, stream>>>(a, r);
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
    }
    DeviceScope scope(device_id);
    if (n_rows == 0) return;
    const int shares = head_shares(n_rows, 2 * n_kv_heads, sm_count(device_id));
    paged_read_kernel<<<dim3(n_rows, shares), kAppendThreads, 0,
                        static_cast<cudaStream_t>(stream)>>>(c, s, k_out, v_out);
    MLB_CUDA(cudaGetLastError());
  });
}
