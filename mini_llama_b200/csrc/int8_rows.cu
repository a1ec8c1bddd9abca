// int8_rows.cu — rows of activations or weights as int8 codes with one scale each:
// as they are, after RMSNorm (with the residual's addition), or SiLU(gate) * up; and
// codes back as the values that they stand for.
//
//   A = max |t|,  code = rint(127 t / A) (ties to even),  scale = A / 127
//
// for a row of values t. RMSNorm's root is a factor of the whole row, so it cancels in
// the codes: they are those of t = h w, h the (rounded) sum, and the root enters the
// scale alone. One pass over the row in registers therefore yields both the sum of
// squares and the maximum, and one reduction joins them.
//
// Codes are those of 64-bit arithmetic. Computed in fp32 (v = t 127 / A), a value next
// to a code's border could fall on either side of it, so the fp32 result is taken only
// where it is further from the border than its error bound, and the few others (about
// 2 in 10^5 after a norm) are computed again in 64 bits, from the inputs. That
// needs A in 64 bits too: the threads that hold a value within the bound of the fp32
// maximum compute theirs again. Rows whose fp32 sums or maxima leave the range where
// those bounds hold (below 1e-30, not finite) are done in 64 bits throughout.
//
// A row with a NaN or an infinity among its values, or a scale past fp32's largest
// number, gets the scale NaN: every product of it is NaN, whatever its codes.
//
// Bound by HBM for many rows, by the chain load - reduction - store for few.
#include <cuda_bf16.h>

#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "paged.cuh"
#include "rows.cuh"

namespace mlb {

namespace {

enum Kind { kPlain, kNorm, kNormAdd, kSilu };

struct RowsArgs {
  const void* x;  // kSilu: gate
  long long x_stride;
  const void* y;  // kNormAdd: the residual, kSilu: up
  long long y_stride;
  const float* w;
  void* sum;
  long long sum_stride;
  int8_t* codes;
  long long codes_stride;
  float* scales;
  int rows, n;
  float eps;
};

constexpr int kHeld = 32;  // values that a thread holds at most
constexpr float kSmallest = 1e-30f;
// Relative error bounds of v. After a norm: t, the maximum (rounded from 64 bits), 127
// over it and the product of both are off by 2^-24 each, 2^-22 together. SiLU: expf and
// the quotient are off by 2 ulp (2^-22) each, the sum and the product of t by 2^-24, and
// what comes after t by 3 2^-24: 1.63 2^-21 together.
template <Kind K>
constexpr float kBound = K == kSilu ? 0x1p-20f : 0x1p-21f;

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// E consecutive elements, zeros past `left`.
template <bool ALIGNED, class T, int E>
__device__ __forceinline__ void load_elements(const T* p, int left, float (&v)[E]) {
  if (ALIGNED && left >= E) {
#pragma unroll
    for (int i = 0; i < E; i += 16 / (int)sizeof(T)) {
      const uint4 u = *reinterpret_cast<const uint4*>(p + i);
      const uint32_t words[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 4) {
          v[i + j] = __uint_as_float(words[j]);
        } else {
          v[i + 2 * j] = __uint_as_float(words[j] << 16);
          v[i + 2 * j + 1] = __uint_as_float(words[j] & 0xffff0000u);
        }
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < E; ++i) v[i] = i < left ? to_float(p[i]) : 0.0f;
}

__device__ __forceinline__ void store_one(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_one(__nv_bfloat16* p, float v) {
  *p = __float2bfloat16_rn(v);
}
template <bool ALIGNED, class T, int E>
__device__ __forceinline__ void store_elements(T* p, int left, const float (&v)[E]) {
  if (ALIGNED && left >= E) {
    uint32_t words[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (sizeof(T) == 4)
        words[j] = __float_as_uint(v[j]);
      else
        words[j] = pack_bf16(v[2 * j], v[2 * j + 1]);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(words[0], words[1], words[2], words[3]);
    return;
  }
#pragma unroll
  for (int i = 0; i < E; ++i)
    if (i < left) store_one(p + i, v[i]);
}

// |x| and |y|'s larger, NaN if one is.
__device__ __forceinline__ float max_abs(float x, float y) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(fabsf(y)));
  return r;
}

// SiLU(g) * u.
__device__ __forceinline__ float silu_mul(float g, float u) {
  return __fdividef(g, 1.0f + expf(-g)) * u;
}
__device__ __noinline__ double silu_mul64(float g, float u) {
  return (double)g / (1.0 + exp(-(double)g)) * (double)u;
}

// One value of the row in 64 bits, from memory. After kNormAdd's pass h is what this
// thread has stored in the sum (which may lie over the residual).
template <Kind K, class T>
__device__ __forceinline__ double value64(const RowsArgs& a, long long row, int i) {
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  if constexpr (K == kPlain) return (double)to_float(x[i]);
  if constexpr (K == kNorm) return (double)to_float(x[i]) * (double)a.w[i];
  if constexpr (K == kNormAdd) {
    const T* h = static_cast<const T*>(a.sum) + row * a.sum_stride;
    return (double)to_float(h[i]) * (double)a.w[i];
  }
  if constexpr (K == kSilu) {
    const T* y = static_cast<const T*>(a.y) + row * a.y_stride;
    return silu_mul64(to_float(x[i]), to_float(y[i]));
  }
}
template <Kind K, class T>
__device__ __forceinline__ double square64(const RowsArgs& a, long long row, int i) {
  if constexpr (K == kNorm) {
    const double h = (double)to_float((static_cast<const T*>(a.x) + row * a.x_stride)[i]);
    return h * h;
  }
  if constexpr (K == kNormAdd) {
    const T* p = static_cast<const T*>(a.sum) + row * a.sum_stride;
    const double h = (double)to_float(p[i]);
    return h * h;
  }
  return 0.0;
}

__device__ __forceinline__ int code64(double t, double top) {
  return (int)rint(t * 127.0 / top);
}

struct Shared {
  float2 part[32];  // per warp: sum of squares, maximum
  double part64[32];
  unsigned long long top;  // bits of the 64-bit maximum
};

// Block-wide sum and maximum of one double per thread each (top: NaN above all).
__device__ __forceinline__ void block_sum_max64(double& sum, double& top, Shared& sh) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (threadIdx.x == 0) sh.top = 0;
  __syncthreads();
  if (lane == 0) sh.part64[warp] = sum;
  atomicMax(&sh.top, (unsigned long long)__double_as_longlong(top));
  __syncthreads();
  sum = 0.0;
  for (int i = 0; i < warps; ++i) sum += sh.part64[i];
  top = __longlong_as_double((long long)sh.top);
  __syncthreads();
}

// A row in 64 bits throughout.
template <Kind K, class T, int E>
__device__ __noinline__ void row64(const RowsArgs& a, long long row, Shared& sh) {
  const int step = (int)blockDim.x * E;
  double sum = 0.0, top = 0.0;
  for (int base = threadIdx.x * E; base < a.n; base += step)
    for (int i = base; i < min(base + E, a.n); ++i) {
      const double t = fabs(value64<K, T>(a, row, i));
      sum += square64<K, T>(a, row, i);
      if (t > top || t != t) top = t != t ? __longlong_as_double(0x7ff8000000000000LL) : t;
    }
  block_sum_max64(sum, top, sh);
  double root = 1.0;
  if (K == kNorm || K == kNormAdd) root = 1.0 / sqrt(sum / a.n + (double)a.eps);
  float scale = top == 0.0 ? 0.0f : (float)(top * root / 127.0);
  if (!(fabsf(scale) <= 3.402823466e38f) || !(top <= 1.7976931348623157e308)) scale = nanf("");
  int8_t* codes = a.codes + row * a.codes_stride;
  const bool none = scale != scale || top == 0.0;
  for (int base = threadIdx.x * E; base < a.n; base += step)
    for (int i = base; i < min(base + E, a.n); ++i)
      codes[i] = none ? 0 : (int8_t)code64(value64<K, T>(a, row, i), top);
  if (threadIdx.x == 0) a.scales[row] = scale;
}

// One CTA per row; thread j has elements (v blockDim + j) E + 0 .. E - 1. NV > 0: v < NV
// covers the row and values stay in registers; NV = 0: rows of any length, computed
// twice. ALIGNED: rows start at 16-byte boundaries.
template <Kind K, class T, int NV, bool ALIGNED, int THREADS>
__global__ void __launch_bounds__(THREADS) int8_rows_kernel(const RowsArgs a) {
  constexpr int E = 16 / (int)sizeof(T);
  constexpr bool NORM = K == kNorm || K == kNormAdd;
  __shared__ Shared sh;
  const long long row = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  const T* y = static_cast<const T*>(a.y) + row * a.y_stride;
  const int step = (int)blockDim.x * E;
  const int nv = NV > 0 ? NV : (a.n + step - 1) / step;

  // E values of the row in fp32, their squares' sum added to ss
  const auto values = [&](int base, float (&t)[E], float& ss, bool first) {
    const int left = a.n - base;
    if (left <= 0) {
#pragma unroll
      for (int i = 0; i < E; ++i) t[i] = 0.0f;
      return;
    }
    if constexpr (K == kNormAdd) {
      T* sum = static_cast<T*>(a.sum) + row * a.sum_stride;
      if (!first) {
        load_elements<ALIGNED>(sum + base, left, t);
      } else {
        float r[E];
        load_elements<ALIGNED>(x + base, left, t);
        load_elements<ALIGNED>(y + base, left, r);
#pragma unroll
        for (int i = 0; i < E; ++i) {
          t[i] += r[i];
          if constexpr (sizeof(T) == 2) t[i] = to_float(__float2bfloat16_rn(t[i]));
        }
        store_elements<ALIGNED>(sum + base, left, t);
      }
    } else {
      load_elements<ALIGNED>(x + base, left, t);
    }
    if constexpr (NORM) {
      float w[E];
      load_elements<true>(a.w + base, left, w);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        ss = fmaf(t[i], t[i], ss);
        t[i] *= w[i];
      }
    }
    if constexpr (K == kSilu) {
      float u[E];
      load_elements<ALIGNED>(y + base, left, u);
#pragma unroll
      for (int i = 0; i < E; ++i) t[i] = silu_mul(t[i], u[i]);
    }
  };

  float held[NV > 0 ? NV : 1][E];
  float ss = 0.0f, top = 0.0f;
#pragma unroll
  for (int v = 0; v < nv; ++v) {
    float(&t)[E] = held[NV > 0 ? v : 0];
    values((v * (int)blockDim.x + (int)threadIdx.x) * E, t, ss, true);
#pragma unroll
    for (int i = 0; i < E; ++i) top = max_abs(top, t[i]);
  }
  const float mine = top;
  top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
  if (NORM) ss = warp_sum(ss);
  if (lane == 0) sh.part[warp] = make_float2(ss, top);
  if (threadIdx.x == 0) sh.top = 0;
  __syncthreads();
  ss = 0.0f;
  uint32_t bits = 0;
  if (warps <= 8) {
    for (int i = 0; i < warps; ++i) {
      const float2 p = sh.part[i];
      ss += p.x;
      bits = max(bits, __float_as_uint(p.y));
    }
  } else {
    const float2 p = lane < warps ? sh.part[lane] : make_float2(0.0f, 0.0f);
    if (NORM) ss = warp_sum(p.x);
    bits = __reduce_max_sync(0xffffffffu, __float_as_uint(p.y));
  }
  top = __uint_as_float(bits);
  // the bounds hold for neither (block-uniform; NaN fails the comparisons)
  if (!(top >= kSmallest && top <= 3e38f) || (NORM && !(ss >= kSmallest && ss <= 3e38f))) {
    row64<K, T, E>(a, row, sh);
    return;
  }

  // the maximum in 64 bits: of the values that may be it
  double top64 = (double)top;
  if (K != kPlain) {
    const float near = top * (1.0f - 2.0f * kBound<K>);
    if (mine >= near) {
      for (int v = 0; v < nv; ++v) {
        const int base = (v * (int)blockDim.x + (int)threadIdx.x) * E;
        for (int i = base; i < min(base + E, a.n); ++i) {
          const double t = fabs(value64<K, T>(a, row, i));
          if (t >= (double)near)
            atomicMax(&sh.top, (unsigned long long)__double_as_longlong(t));
        }
      }
    }
    __syncthreads();
    top64 = __longlong_as_double((long long)sh.top);
  }

  const float inv = __fdiv_rn(127.0f, (float)top64);
  int8_t* codes = a.codes + row * a.codes_stride;
#pragma unroll
  for (int v = 0; v < nv; ++v) {
    const int base = (v * (int)blockDim.x + (int)threadIdx.x) * E;
    float(&t)[E] = held[NV > 0 ? v : 0];
    if (NV == 0) {
      float unused = 0.0f;
      values(base, t, unused, false);
    }
    uint32_t c[E];
    float worst = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float q = t[i] * inv;
      const float r = q + 12582912.0f;  // 1.5 * 2^23: the nearest whole number in the low bits
      const float d = q - (r - 12582912.0f);
      c[i] = __float_as_uint(r);
      worst = fmaxf(worst, fmaf(fabsf(q), kBound<K>, fabsf(d)));
    }
    if (worst > 0.5f) {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const float q = t[i] * inv;
        const float d = q - (__uint_as_float(c[i]) - 12582912.0f);
        if (fmaf(fabsf(q), kBound<K>, fabsf(d)) > 0.5f && base + i < a.n)
          c[i] = (uint32_t)code64(K == kPlain ? (double)t[i] : value64<K, T>(a, row, base + i),
                                  top64);
      }
    }
    uint32_t words[E / 4];
#pragma unroll
    for (int i = 0; i < E / 4; ++i)
      words[i] = __byte_perm(__byte_perm(c[4 * i], c[4 * i + 1], 0x0040),
                             __byte_perm(c[4 * i + 2], c[4 * i + 3], 0x0040), 0x5410);
    if (base + E <= a.n) {  // rows of codes are 16-byte aligned
      if constexpr (E == 8)
        *reinterpret_cast<uint2*>(codes + base) = make_uint2(words[0], words[1]);
      else
        *reinterpret_cast<uint32_t*>(codes + base) = words[0];
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (base + i < a.n) codes[base + i] = (int8_t)(c[i] & 0xffu);
    }
  }
  if (threadIdx.x == 0) {
    double s = top64 / 127.0;
    if (NORM) s *= 1.0 / sqrt((double)ss / a.n + (double)a.eps);
    const float scale = (float)s;
    a.scales[row] = fabsf(scale) <= 3.402823466e38f ? scale : nanf("");
  }
}

template <Kind K, class T, int NV, bool ALIGNED>
void launch(const RowsArgs& a, int threads, cudaStream_t s) {
  // 1024 threads leave 64 registers each
  if (threads <= 512)
    int8_rows_kernel<K, T, NV, ALIGNED, 512><<<a.rows, threads, 0, s>>>(a);
  else
    int8_rows_kernel<K, T, NV, ALIGNED, 1024><<<a.rows, threads, 0, s>>>(a);
  MLB_CUDA(cudaGetLastError());
}

template <Kind K, class T>
void dispatch(const RowsArgs& a, bool aligned, int device_id, cudaStream_t s) {
  constexpr int E = 16 / (int)sizeof(T), MOST = kHeld / E;
  const auto threads_for = [&](int nv) { return ((a.n + E * nv - 1) / (E * nv) + 31) / 32 * 32; };
  if (threads_for(MOST) > 1024) {
    if (aligned) return launch<K, T, 0, true>(a, 1024, s);
    return launch<K, T, 0, false>(a, 1024, s);
  }
  if (!aligned) return launch<K, T, MOST, false>(a, threads_for(MOST), s);
  // few rows: many threads for each, for the time of one; many: fewer, for less work
  // around their reductions
  const int most = a.rows <= 2 * sm_count(device_id) ? 512 : 256;
  int nv = 1;
  while (nv < MOST && threads_for(nv) > most) nv *= 2;
  const int threads = threads_for(nv);
  if (nv == 1) return launch<K, T, 1, true>(a, threads, s);
  if (nv == 2) return launch<K, T, 2, true>(a, threads, s);
  if (nv == 4) return launch<K, T, 4, true>(a, threads, s);
  if constexpr (MOST >= 8) return launch<K, T, 8, true>(a, threads, s);
}

template <Kind K>
void run_rows(const RowsArgs& a, int act_type, int device_id, void* stream) {
  DeviceScope scope(device_id);
  if (a.rows == 0) return;
  const int es = act_type == MLB_ACT_BF16 ? 2 : 4;
  const auto on16 = [&](const void* p, long long stride) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (a.rows == 1 || stride % (16 / es) == 0);
  };
  const bool aligned = on16(a.x, a.x_stride) && (!a.y || on16(a.y, a.y_stride)) &&
                       (!a.sum || on16(a.sum, a.sum_stride)) &&
                       (!a.w || reinterpret_cast<uintptr_t>(a.w) % 16 == 0);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (act_type == MLB_ACT_BF16)
    dispatch<K, __nv_bfloat16>(a, aligned, device_id, s);
  else
    dispatch<K, float>(a, aligned, device_id, s);
}

// Codes times their row's scale, 16 per thread.
template <class T>
__global__ void __launch_bounds__(256) int8_dequant_kernel(const int8_t* codes, long long stride,
                                                           const float* scales, int rows, int n,
                                                           T* out, long long out_stride,
                                                           bool aligned) {
  const int per_row = (n + 15) / 16;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long row = i / per_row;
  if (row >= rows) return;
  const int base = (int)(i - row * per_row) * 16;
  const float s = scales[row];
  const int8_t* c = codes + row * stride + base;
  T* o = out + row * out_stride + base;
  float v[16];
  if (base + 16 <= n) {
    const uint4 u = *reinterpret_cast<const uint4*>(c);
    const uint32_t words[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 16; ++j)
      v[j] = (float)(int8_t)(words[j >> 2] >> (8 * (j & 3))) * s;
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = base + j < n ? (float)c[j] * s : 0.0f;
  }
  constexpr int E = 16 / (int)sizeof(T);
#pragma unroll
  for (int j = 0; j < 16; j += E) {
    float part[E];
#pragma unroll
    for (int e = 0; e < E; ++e) part[e] = v[j + e];
    if (aligned)
      store_elements<true>(o + j, n - base - j, part);
    else
      store_elements<false>(o + j, n - base - j, part);
  }
}

// ------------------------------------------------------------ argument checks

// Rows of n elements of the activation type, any alignment that the type itself has.
void check_act_rows(const char* who, const char* name, const void* p, long long stride, int n,
                    int act) {
  const std::string w = who;
  if (!p) invalid(w + ": null " + name);
  if (stride < n) invalid(w + ": row stride of " + name + " is smaller than a row");
  if (reinterpret_cast<uintptr_t>(p) % (act == MLB_ACT_BF16 ? 2 : 4) != 0)
    invalid(w + ": " + name + " is unaligned");
}

struct Bytes {  // rows of bytes
  const char* name;
  const void* p;
  wide_int stride, bytes;
  int rows;
};

Bytes act_bytes(const char* name, const void* p, long long stride, int n, int rows, int act) {
  const int es = act == MLB_ACT_BF16 ? 2 : 4;
  return {name, p, (wide_int)stride * es, (wide_int)n * es, rows};
}

void check_apart(const char* who, const Bytes& a, const Bytes& b) {
  if (byte_rows_overlap(a.p, a.stride, a.bytes, a.rows, b.p, b.stride, b.bytes, b.rows))
    invalid(std::string(who) + ": " + a.name + " must not overlap " + b.name);
}

// Sizes and the rows of codes and scales that a call writes; false where there is
// nothing to do.
bool check_codes(const char* who, int act, int rows, int n, const int8_t* codes,
                 long long codes_stride, const float* scales) {
  const std::string w = who;
  paged_check_act(who, act);
  if (rows < 0) invalid(w + ": negative row count");
  if (n <= 0) invalid(w + ": rows must have at least one element");
  if (n > (1 << 30)) invalid(w + ": rows have more than 2^30 elements");
  if (rows == 0) return false;
  if (!codes) invalid(w + ": null codes");
  if (!scales) invalid(w + ": null scales");
  if (codes_stride < n) invalid(w + ": row stride of codes is smaller than a row");
  if (reinterpret_cast<uintptr_t>(codes) % 16 != 0 || codes_stride % 16 != 0)
    invalid(w + ": rows of codes must be 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(scales) % 4 != 0) invalid(w + ": scales are unaligned");
  check_apart(who, {"codes", codes, codes_stride, n, rows}, {"scales", scales, 4, 4, rows});
  return true;
}

// Neither codes nor scales may overlap an operand.
void check_outputs(const char* who, const RowsArgs& a, const Bytes& operand) {
  check_apart(who, {"codes", a.codes, a.codes_stride, a.n, a.rows}, operand);
  check_apart(who, {"scales", a.scales, 4, 4, a.rows}, operand);
}

}  // namespace

}  // namespace mlb

using namespace mlb;

extern "C" int mlb_int8_quantize(int act_type, const void* x, long long x_stride, int rows, int n,
                                 int8_t* codes, long long codes_stride, float* scales,
                                 int device_id, void* stream) {
  return guarded([&] {
    const char* who = "Int8Quantize";
    const bool any = check_codes(who, act_type, rows, n, codes, codes_stride, scales);
    RowsArgs a = {};
    a.x = x, a.x_stride = x_stride, a.codes = codes, a.codes_stride = codes_stride;
    a.scales = scales, a.rows = rows, a.n = n;
    if (any) {
      check_act_rows(who, "x", x, x_stride, n, act_type);
      check_outputs(who, a, act_bytes("x", x, x_stride, n, rows, act_type));
    }
    run_rows<kPlain>(a, act_type, device_id, stream);
  });
}

extern "C" int mlb_rmsnorm_int8(int act_type, const void* x, long long x_stride,
                                const void* residual, long long residual_stride, const float* w,
                                int rows, int n, float eps, void* sum, long long sum_stride,
                                int8_t* codes, long long codes_stride, float* scales,
                                int device_id, void* stream) {
  return guarded([&] {
    const char* who = "RmsNormInt8";
    const bool any = check_codes(who, act_type, rows, n, codes, codes_stride, scales);
    if (!(eps >= 0.0f) || std::isinf(eps)) invalid("RmsNormInt8: eps must be finite and not negative");
    RowsArgs a = {};
    a.x = x, a.x_stride = x_stride, a.y = residual, a.y_stride = residual_stride;
    a.w = w, a.sum = sum, a.sum_stride = sum_stride, a.codes = codes;
    a.codes_stride = codes_stride, a.scales = scales, a.rows = rows, a.n = n, a.eps = eps;
    if (any) {
      check_act_rows(who, "x", x, x_stride, n, act_type);
      if (!w) invalid("RmsNormInt8: null weights");
      if (reinterpret_cast<uintptr_t>(w) % 4 != 0) invalid("RmsNormInt8: weights are unaligned");
      const Bytes bx = act_bytes("x", x, x_stride, n, rows, act_type);
      const Bytes bw = {"weights", w, (wide_int)n * 4, (wide_int)n * 4, 1};
      check_outputs(who, a, bx);
      check_outputs(who, a, bw);
      if (!residual && sum) invalid("RmsNormInt8: a sum without a residual");
      if (residual) {
        check_act_rows(who, "residual", residual, residual_stride, n, act_type);
        check_act_rows(who, "sum", sum, sum_stride, n, act_type);
        const Bytes br = act_bytes("residual", residual, residual_stride, n, rows, act_type);
        const Bytes bs = act_bytes("sum", sum, sum_stride, n, rows, act_type);
        check_outputs(who, a, br);
        check_outputs(who, a, bs);
        check_apart(who, bs, bw);
        // in place, or apart: an element is read before it is written, but only its own
        const auto same = [&](const void* p, long long stride) {
          return sum == p && (sum_stride == stride || rows == 1);
        };
        if (!same(x, x_stride)) check_apart(who, bs, bx);
        if (!same(residual, residual_stride)) check_apart(who, bs, br);
      }
    }
    if (residual)
      run_rows<kNormAdd>(a, act_type, device_id, stream);
    else
      run_rows<kNorm>(a, act_type, device_id, stream);
  });
}

extern "C" int mlb_silu_mul_int8(int act_type, const void* gate, long long gate_stride,
                                 const void* up, long long up_stride, int rows, int n,
                                 int8_t* codes, long long codes_stride, float* scales,
                                 int device_id, void* stream) {
  return guarded([&] {
    const char* who = "SiluMulInt8";
    const bool any = check_codes(who, act_type, rows, n, codes, codes_stride, scales);
    RowsArgs a = {};
    a.x = gate, a.x_stride = gate_stride, a.y = up, a.y_stride = up_stride;
    a.codes = codes, a.codes_stride = codes_stride, a.scales = scales, a.rows = rows, a.n = n;
    if (any) {
      check_act_rows(who, "gate", gate, gate_stride, n, act_type);
      check_act_rows(who, "up", up, up_stride, n, act_type);
      check_outputs(who, a, act_bytes("gate", gate, gate_stride, n, rows, act_type));
      check_outputs(who, a, act_bytes("up", up, up_stride, n, rows, act_type));
    }
    run_rows<kSilu>(a, act_type, device_id, stream);
  });
}

extern "C" int mlb_int8_dequantize(const int8_t* codes, long long codes_stride,
                                   const float* scales, int rows, int n, int out_type, void* out,
                                   long long out_stride, int device_id, void* stream) {
  return guarded([&] {
    const char* who = "Int8Dequantize";
    const bool any = check_codes(who, out_type, rows, n, codes, codes_stride, scales);
    if (any) {
      check_act_rows(who, "out", out, out_stride, n, out_type);
      const Bytes bo = act_bytes("out", out, out_stride, n, rows, out_type);
      check_apart(who, bo, {"codes", codes, codes_stride, n, rows});
      check_apart(who, bo, {"scales", scales, 4, 4, rows});
    }
    DeviceScope scope(device_id);
    if (!any) return;
    const int es = out_type == MLB_ACT_BF16 ? 2 : 4;
    const bool aligned = reinterpret_cast<uintptr_t>(out) % 16 == 0 &&
                         (rows == 1 || out_stride % (16 / es) == 0);
    const long long blocks = ((long long)rows * ((n + 15) / 16) + 255) / 256;
    if (blocks > 0x7fffffffLL) invalid("Int8Dequantize: too many rows");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (out_type == MLB_ACT_BF16)
      int8_dequant_kernel<<<(unsigned)blocks, 256, 0, s>>>(
          codes, codes_stride, scales, rows, n, static_cast<__nv_bfloat16*>(out), out_stride,
          aligned);
    else
      int8_dequant_kernel<<<(unsigned)blocks, 256, 0, s>>>(
          codes, codes_stride, scales, rows, n, static_cast<float*>(out), out_stride, aligned);
    MLB_CUDA(cudaGetLastError());
  });
}
