// rope_rows.cu — rotation of queries and keys of many rows to positions of their own:
// both layouts, the first rotary_dim of head_dim dimensions, frequencies from a table
// (which scaled frequencies for long contexts are made into on the host).
//
//   (a, b) -> g (a cos x - b sin x, a sin x + b cos x),  x = position * frequency[i]
//
// for the pairs (2i, 2i + 1) or (i, i + rotary_dim / 2). The angle's turns, position *
// frequency / 2 pi, are taken in 64 bits, where the whole ones are dropped without loss;
// sine and cosine of what is left are fp32's, so far positions cost no accuracy and no
// 64-bit sine. They are the same for all heads: a CTA takes a row, makes them once in
// shared memory and goes through its heads 16 bytes at a time, what is not turned first.
//
// Bound by the chain position - angle - barrier - product, and HBM behind it: 4096 rows of
// 32 + 8 heads of 128 bf16 15.8 us (5.3 TB/s; 17.4 beyond L2), half of each turned 13.3
// (18.3), fp32 28 (6.0 TB/s); one row 2.4 us.
#include <cuda_bf16.h>

#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "paged.cuh"
#include "rows.cuh"

namespace mlb {

namespace {

constexpr int kThreads = 512;  // at most
constexpr int kMaxHeadDim = 1024;  // dimensions whose sines a CTA keeps

struct RopeArgs {
  const void* in[2];  // queries, keys
  void* out[2];
  long long in_stride[2], out_stride[2];
  int heads[2];
  int head_dim, rotary_dim;
  const int* positions;
  const double* frequencies;
  float amplitude;
  bool copy[2];  // dimensions past rotary_dim go to another place
};

template <class T>
__device__ __forceinline__ float widen(T v) {
  if constexpr (sizeof(T) == 4)
    return v;
  else
    return __bfloat162float(v);
}
template <class T, int E>
__device__ __forceinline__ void load(const T* p, float (&v)[E]) {
  if constexpr (E * sizeof(T) == 16) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        v[i] = __uint_as_float(w[i]);
      } else {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = widen(p[i]);
  }
}
template <class T, int E>
__device__ __forceinline__ void store(T* p, const float (&v)[E]) {
  if constexpr (E * sizeof(T) == 16) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4)
        w[i] = __float_as_uint(v[i]);
      else
        w[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      if constexpr (sizeof(T) == 4)
        p[i] = v[i];
      else
        p[i] = __float2bfloat16_rn(v[i]);
    }
  }
}

// body(side, head, unit) for every unit of every head, the threads in turn.
template <class Body>
__device__ __forceinline__ void for_units(const RopeArgs& a, int units, Body body) {
  if (units == 0) return;
  const int threads = blockDim.x;
  const int head_step = threads / units, unit_step = threads - head_step * units;
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    int head = threadIdx.x / units, u = threadIdx.x - head * units;
    while (head < a.heads[side]) {
      body(side, head, u);
      head += head_step;
      u += unit_step;
      if (u >= units) {
        u -= units;
        ++head;
      }
    }
  }
}

// E elements at a time: 16 bytes, or the least that holds a pair (NORMAL: 2) or one
// side of it (NEOX: 1). What is not turned goes first, while the angles are made; then
// units of E elements, NEOX: of the first half, with their partners.
template <class T, int E, bool NEOX>
__global__ void __launch_bounds__(kThreads) rope_rows_kernel(const RopeArgs a) {
  __shared__ float2 turn[kMaxHeadDim / 2];
  const long long row = blockIdx.x;
  const int half = a.rotary_dim / 2;
  const int turned = NEOX ? half / E : (a.rotary_dim + E - 1) / E;
  const int rest0 = NEOX ? a.rotary_dim : turned * E;  // the first dimension that is not
  pdl_launch_dependents();
  pdl_wait();
  const auto in = [&](int side, int head) {
    return static_cast<const T*>(a.in[side]) + row * a.in_stride[side] + head * a.head_dim;
  };
  const auto out = [&](int side, int head) {
    return static_cast<T*>(a.out[side]) + row * a.out_stride[side] + head * a.head_dim;
  };
  const double pos = (double)a.positions[row];
  for (int i = threadIdx.x; i < half; i += blockDim.x) {
    const double t = pos * (a.frequencies[i] * 0.15915494309189533577);  // 1 / (2 pi)
    float s, c;
    sincospif(2.0f * (float)(t - rint(t)), &s, &c);
    turn[i] = make_float2(c * a.amplitude, s * a.amplitude);
  }
  if (a.copy[0] || a.copy[1])
    for_units(a, (a.head_dim - rest0) / E, [&](int side, int head, int u) {
      if (!a.copy[side]) return;
      float p[E];
      load<T, E>(in(side, head) + rest0 + u * E, p);
      store<T, E>(out(side, head) + rest0 + u * E, p);
    });
  __syncthreads();
  for_units(a, turned, [&](int side, int head, int u) {
    const int d = u * E;
    const T* x = in(side, head) + d;
    T* y = out(side, head) + d;
    float p[E];
    load<T, E>(x, p);
    if constexpr (NEOX) {
      float q[E];
      load<T, E>(x + half, q);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const float2 cs = turn[d + i];
        const float lo = fmaf(p[i], cs.x, -(q[i] * cs.y));
        q[i] = fmaf(p[i], cs.y, q[i] * cs.x);
        p[i] = lo;
      }
      store<T, E>(y + half, q);
    } else {
#pragma unroll
      for (int i = 0; i < E; i += 2) {
        if (d + i < a.rotary_dim) {
          const float2 cs = turn[(d + i) / 2];
          const float lo = fmaf(p[i], cs.x, -(p[i + 1] * cs.y));
          p[i + 1] = fmaf(p[i], cs.y, p[i + 1] * cs.x);
          p[i] = lo;
        }
      }
    }
    store<T, E>(y, p);
  });
}

// Threads of a row's CTA: many rows 128, which leaves more of them beside one another
// while their angles are made (4096 rows of 32 + 8 heads bf16 that L2 does not hold, in us,
// 64 / 128 / 192 / 256 threads: 17.9 / 17.4 / 19.2 / 19.0, half of each head 19.2 / 18.3 /
// 21.5 / 22.1), few 512 (one row fp32, 128 / 256 / 512: 4.1 / 2.8 / 2.4); no more than
// there are units.
template <class T, int E>
void launch(const RopeArgs& a, int rows, bool neox, int device_id, cudaStream_t s) {
  const auto kernel =
      neox ? rope_rows_kernel<T, E, true> : rope_rows_kernel<T, (E > 1 ? E : 2), false>;
  const long long units = (long long)(a.heads[0] + a.heads[1]) *
                          (neox ? a.rotary_dim / 2 / E + (a.head_dim - a.rotary_dim) / E
                                : a.head_dim / std::max(E, 2));
  const long long most = rows > 4 * sm_count(device_id) ? 128 : kThreads;
  const int threads = (int)(std::min(most, units) + 31) / 32 * 32;
  launch_pdl(kernel, dim3(rows), dim3(threads), 0, s, true, a);
}

template <class T>
void dispatch(const RopeArgs& a, int rows, bool neox, int device_id, cudaStream_t s) {
  constexpr int E = 16 / (int)sizeof(T);
  bool wide = a.head_dim % E == 0 && (!neox || (a.rotary_dim / 2) % E == 0);
  for (int side = 0; side < 2; ++side) {
    if (a.heads[side] == 0) continue;
    wide = wide && reinterpret_cast<uintptr_t>(a.in[side]) % 16 == 0 &&
           reinterpret_cast<uintptr_t>(a.out[side]) % 16 == 0;
    if (rows > 1) wide = wide && a.in_stride[side] % E == 0 && a.out_stride[side] % E == 0;
  }
  if (wide) return launch<T, E>(a, rows, neox, device_id, s);
  return launch<T, 1>(a, rows, neox, device_id, s);
}

}  // namespace

}  // namespace mlb

using namespace mlb;

extern "C" int mlb_rope_frequencies(int rotary_dim, double theta, int scaling, double factor,
                                    double original_len, double low_freq_factor,
                                    double high_freq_factor, double beta_fast, double beta_slow,
                                    double* frequencies_host, double* amplitude) {
  return guarded([&] {
    const auto positive = [](double v) { return v > 0.0 && std::isfinite(v); };
    if (rotary_dim <= 0 || rotary_dim % 2 != 0 || rotary_dim > kMaxHeadDim)
      invalid("RopeFrequencies: rotary_dim must be even, 2 to 1024, got " +
              std::to_string(rotary_dim));
    if (!positive(theta) || theta <= 1.0)
      invalid("RopeFrequencies: theta must be finite and above 1");
    if (scaling < MLB_ROPE_SCALING_NONE || scaling > MLB_ROPE_SCALING_YARN)
      invalid("RopeFrequencies: unknown scaling " + std::to_string(scaling));
    if (!frequencies_host || !amplitude) invalid("RopeFrequencies: null output");
    const bool by_parts = scaling == MLB_ROPE_SCALING_LLAMA3 || scaling == MLB_ROPE_SCALING_YARN;
    if (scaling != MLB_ROPE_SCALING_NONE && !positive(factor))
      invalid("RopeFrequencies: factor must be finite and positive");
    if (by_parts && !positive(original_len))
      invalid("RopeFrequencies: original_len must be finite and positive");
    if (scaling == MLB_ROPE_SCALING_LLAMA3 &&
        !(positive(low_freq_factor) && positive(high_freq_factor) &&
          low_freq_factor < high_freq_factor))
      invalid("RopeFrequencies: low_freq_factor must be positive and below high_freq_factor");
    if (scaling == MLB_ROPE_SCALING_YARN &&
        !(positive(beta_slow) && positive(beta_fast) && beta_slow <= beta_fast))
      invalid("RopeFrequencies: beta_slow must be positive and at most beta_fast");

    const double two_pi = 6.283185307179586477;
    // pair (as a real number) that makes `turns` turns over the original length
    const auto pair_of = [&](double turns) {
      return rotary_dim * std::log(original_len / (turns * two_pi)) / (2.0 * std::log(theta));
    };
    double first = 0.0, last = 0.0;
    *amplitude = 1.0;
    if (scaling == MLB_ROPE_SCALING_YARN) {
      first = std::max(std::floor(pair_of(beta_fast)), 0.0);
      last = std::min(std::ceil(pair_of(beta_slow)), (double)(rotary_dim - 1));
      if (factor > 1.0) *amplitude = 0.1 * std::log(factor) + 1.0;
    }
    for (int i = 0; i < rotary_dim / 2; ++i) {
      const double f = std::pow(theta, -2.0 * i / rotary_dim);
      double kept = 1.0;  // how much of f itself, the rest is f / factor
      if (scaling == MLB_ROPE_SCALING_LINEAR) kept = 0.0;
      if (scaling == MLB_ROPE_SCALING_LLAMA3)
        kept = (original_len * f / two_pi - low_freq_factor) / (high_freq_factor - low_freq_factor);
      if (scaling == MLB_ROPE_SCALING_YARN) kept = 1.0 - (i - first) / std::max(last - first, 0.001);
      kept = std::min(1.0, std::max(0.0, kept));
      frequencies_host[i] = scaling == MLB_ROPE_SCALING_NONE ? f : f / factor * (1.0 - kept) + f * kept;
    }
  });
}

extern "C" int mlb_rope_rows(int act_type, const void* q, long long q_stride, int n_heads,
                             const void* k, long long k_stride, int n_kv_heads, int head_dim,
                             int rotary_dim, const int* positions, const double* frequencies,
                             float amplitude, int rope_type, int n_rows, void* q_out,
                             long long q_out_stride, void* k_out, long long k_out_stride,
                             int device_id, void* stream) {
  return guarded([&] {
    const std::string who = "RopeRows";
    paged_check_act("RopeRows", act_type);
    if (rope_type != MLB_ROPE_NORMAL && rope_type != MLB_ROPE_NEOX)
      invalid(who + ": unknown rope type " + std::to_string(rope_type));
    if (n_rows < 0) invalid(who + ": negative row count");
    if (n_heads < 0 || n_kv_heads < 0) invalid(who + ": negative head count");
    if (head_dim <= 0 || head_dim % 2 != 0 || head_dim > kMaxHeadDim)
      invalid(who + ": head_dim must be even, 2 to 1024, got " + std::to_string(head_dim));
    if (rotary_dim <= 0 || rotary_dim % 2 != 0 || rotary_dim > head_dim)
      invalid(who + ": rotary_dim must be even, 2 to head_dim, got " + std::to_string(rotary_dim));
    if (!std::isfinite(amplitude)) invalid(who + ": amplitude must be finite");
    const bool any = n_rows > 0 && (n_heads > 0 || n_kv_heads > 0);
    if (!any) {
      DeviceScope scope(device_id);
      return;
    }
    if (!positions || !frequencies) invalid(who + ": null positions or frequencies");
    if (reinterpret_cast<uintptr_t>(positions) % 4 != 0 ||
        reinterpret_cast<uintptr_t>(frequencies) % 8 != 0)
      invalid(who + ": positions or frequencies are unaligned");
    const int es = act_type == MLB_ACT_BF16 ? 2 : 4;
    RopeArgs a = {{q, k}, {q_out, k_out}, {q_stride, k_stride}, {q_out_stride, k_out_stride},
                  {n_heads, n_kv_heads}, head_dim, rotary_dim, positions, frequencies, amplitude,
                  {false, false}};
    const char* names[2][2] = {{"q", "q_out"}, {"k", "k_out"}};
    for (int side = 0; side < 2; ++side) {
      if (a.heads[side] == 0) continue;
      const long long row = (long long)a.heads[side] * head_dim;
      if (row > 0x7fffffffLL) invalid(who + ": rows have more than 2^31 elements");
      const void* p[2] = {a.in[side], a.out[side]};
      const long long stride[2] = {a.in_stride[side], a.out_stride[side]};
      for (int o = 0; o < 2; ++o) {
        if (!p[o]) invalid(who + ": null " + names[side][o]);
        if (stride[o] < row)
          invalid(who + ": row stride of " + names[side][o] + " is smaller than a row");
        if (reinterpret_cast<uintptr_t>(p[o]) % es != 0)
          invalid(who + ": " + names[side][o] + " is unaligned");
      }
      a.copy[side] = p[0] != p[1];
    }
    // an output lies over its own input exactly, or over no byte that is read or written
    for (int o = 0; o < 2; ++o) {
      if (a.heads[o] == 0) continue;
      const wide_int out_bytes = (wide_int)a.heads[o] * head_dim * es;
      const auto apart = [&](const char* name, const void* p, wide_int stride, wide_int bytes,
                             int rows) {
        if (byte_rows_overlap(a.out[o], (wide_int)a.out_stride[o] * es, out_bytes, n_rows, p,
                              stride, bytes, rows))
          invalid(who + ": " + names[o][1] + " must not overlap " + name);
      };
      for (int i = 0; i < 2; ++i) {
        if (a.heads[i] == 0) continue;
        const wide_int bytes = (wide_int)a.heads[i] * head_dim * es;
        const bool same = i == o && a.in[i] == a.out[o] &&
                          (a.in_stride[i] == a.out_stride[o] || n_rows == 1);
        if (!same) apart(names[i][0], a.in[i], (wide_int)a.in_stride[i] * es, bytes, n_rows);
        if (i != o) apart(names[i][1], a.out[i], (wide_int)a.out_stride[i] * es, bytes, n_rows);
      }
      apart("positions", positions, (wide_int)n_rows * 4, (wide_int)n_rows * 4, 1);
      apart("frequencies", frequencies, (wide_int)rotary_dim * 4, (wide_int)rotary_dim * 4, 1);
    }
    DeviceScope scope(device_id);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (act_type == MLB_ACT_BF16)
      dispatch<__nv_bfloat16>(a, n_rows, rope_type == MLB_ROPE_NEOX, device_id, s);
    else
      dispatch<float>(a, n_rows, rope_type == MLB_ROPE_NEOX, device_id, s);
  });
}
