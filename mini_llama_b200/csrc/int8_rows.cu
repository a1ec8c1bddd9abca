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
// where it is further from the border than its error bound, and the few others (5 in
// 10^5 after a norm, 4 in 10^4 of SiLU) are done again in 64 bits, from the inputs. Those
// need A in 64 bits: the threads that hold a value within the bound of the fp32 maximum
// compute theirs again, while the others go on, and a second barrier later the doubtful
// codes are corrected. Rows whose fp32 sums or maxima leave the range where the bounds
// hold (below 1e-30, not finite, gates below -87) are done in 64 bits throughout.
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
constexpr float kLowestGate = -87.0f;  // e^87 is a normal number, and so is its reciprocal
// Relative error bounds, in units of 2^-24. t: after a norm one product; SiLU: ex2 4 (2
// ulp), the factor that corrects it, the sum and two products 1 each, the reciprocal 2: 10
// together. v: t's, the maximum's (the same), its reciprocal times 127; the last product is
// exact in a fused multiply-add. Kept: a little more, v's times 127 from a code's border.
template <Kind K>
constexpr float kValueBound = (K == kSilu ? 12.0f : 2.0f) * 0x1p-24f;
template <Kind K>
constexpr float kBorder = 0.5f - 127.0f * 0x1p-24f * (K == kSilu ? 24.0f : K == kPlain ? 2.0f : 4.0f);

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

// SiLU(g) * u. e^-g = 2^(hi + lo), -g log2(e) in two parts; 2^lo as 1 + lo ln 2.
__device__ __forceinline__ float silu_mul(float g, float u) {
  const float hi = g * -1.4426950408889634f;
  // what hi's rounding and the constant's (1.92596e-8 beyond fp32) leave, times ln 2
  const float lo = fmaf(g, -1.4426950408889634f, -hi) * 0.6931471805599453f + g * -1.33497e-8f;
  float e = ex2(hi), r;
  e = fmaf(e, lo, e);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return g * r * u;
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
template <Kind K, class T, int NV, bool ALIGNED>
__global__ void __launch_bounds__(1024) int8_rows_kernel(const RowsArgs a) {
  constexpr int E = 16 / (int)sizeof(T);
  constexpr bool NORM = K == kNorm || K == kNormAdd;
  __shared__ Shared sh;
  const long long row = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  const T* y = static_cast<const T*>(a.y) + row * a.y_stride;
  const int step = (int)blockDim.x * E;
  const int nv = NV > 0 ? NV : (a.n + step - 1) / step;
  pdl_launch_dependents();
  pdl_wait();

  // E values of the row in fp32, their squares added to ss; low: the lowest gate
  const auto values = [&](int base, float2 (&t)[E / 2], float2& ss, float& low, bool first) {
    const int left = a.n - base;
    if (left <= 0) {
#pragma unroll
      for (int i = 0; i < E / 2; ++i) t[i] = make_float2(0.0f, 0.0f);
      return;
    }
    float v[E], o[E];
    if (K == kNormAdd && !first) {
      load_elements<ALIGNED>(static_cast<const T*>(a.sum) + row * a.sum_stride + base, left, v);
    } else {
      load_elements<ALIGNED>(x + base, left, v);
      if constexpr (K == kNormAdd || K == kSilu) load_elements<ALIGNED>(y + base, left, o);
    }
    if (K == kNormAdd && first) {
#pragma unroll
      for (int i = 0; i < E; i += 2) {
        const float2 s = add2(make_float2(v[i], v[i + 1]), make_float2(o[i], o[i + 1]));
        v[i] = s.x, v[i + 1] = s.y;
        if constexpr (sizeof(T) == 2) {
          const uint32_t w = pack_bf16(s.x, s.y);
          v[i] = __uint_as_float(w << 16), v[i + 1] = __uint_as_float(w & 0xffff0000u);
        }
      }
      store_elements<ALIGNED>(static_cast<T*>(a.sum) + row * a.sum_stride + base, left, v);
    }
    if constexpr (NORM) load_elements<true>(a.w + base, left, o);
#pragma unroll
    for (int i = 0; i < E; i += 2) {
      const float2 p = make_float2(v[i], v[i + 1]);
      if constexpr (NORM) {
        ss = fma2(p, p, ss);
        t[i / 2] = mul2(p, make_float2(o[i], o[i + 1]));
      } else if constexpr (K == kSilu) {
        low = fminf(low, fminf(p.x, p.y));
        t[i / 2] = make_float2(silu_mul(p.x, o[i]), silu_mul(p.y, o[i + 1]));
      } else {
        t[i / 2] = p;
      }
    }
  };

  float2 held[NV > 0 ? NV : 1][E / 2];
  float2 ss2 = make_float2(0.0f, 0.0f);
  float top = 0.0f, low = 0.0f;
#pragma unroll
  for (int v = 0; v < nv; ++v) {
    float2(&t)[E / 2] = held[NV > 0 ? v : 0];
    values((v * (int)blockDim.x + (int)threadIdx.x) * E, t, ss2, low, true);
#pragma unroll
    for (int i = 0; i < E / 2; ++i) top = max_abs(max_abs(top, t[i].x), t[i].y);
  }
  if (K == kSilu && low < kLowestGate) top = nanf("");
  const float mine = top;
  float ss = ss2.x + ss2.y;
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
  const float near = top * (1.0f - 2.0f * kValueBound<K>);
  const auto candidate = [&](int i) {
    const double t = fabs(value64<K, T>(a, row, i));
    atomicMax(&sh.top, (unsigned long long)__double_as_longlong(t));
  };
  if (K != kPlain && mine >= near) {
    if constexpr (NV > 0) {
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < E; ++i)
          if (fabsf(i & 1 ? held[v][i / 2].y : held[v][i / 2].x) >= near)
            candidate((v * (int)blockDim.x + (int)threadIdx.x) * E + i);
    } else {
      for (int v = 0; v < nv; ++v) {
        const int base = (v * (int)blockDim.x + (int)threadIdx.x) * E;
        for (int i = base; i < min(base + E, a.n); ++i)
          if (fabs(value64<K, T>(a, row, i)) >= (double)near) candidate(i);
      }
    }
  }
  const auto top64 = [&] {
    return K == kPlain ? (double)top : __longlong_as_double((long long)sh.top);
  };
  if (NV == 0) __syncthreads();

  const float inv = __fdiv_rn(127.0f, top);
  const float2 inv2 = make_float2(inv, inv);
  const float2 magic = make_float2(12582912.0f, 12582912.0f);  // 1.5 * 2^23
  int8_t* codes = a.codes + row * a.codes_stride;
  uint32_t doubtful = 0;  // bit v E + i
#pragma unroll
  for (int v = 0; v < nv; ++v) {
    const int base = (v * (int)blockDim.x + (int)threadIdx.x) * E;
    float2(&t)[E / 2] = held[NV > 0 ? v : 0];
    if (NV == 0) values(base, t, ss2, low, false);
    uint32_t c[E];
    float2 d[E / 2];
    float worst = 0.0f;
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      const float2 r = fma2(t[i], inv2, magic);  // the nearest whole number in the low bits
      d[i] = fma2(t[i], inv2, fma2(r, make_float2(-1.0f, -1.0f), magic));
      c[2 * i] = __float_as_uint(r.x), c[2 * i + 1] = __float_as_uint(r.y);
      worst = fmaxf(worst, fmaxf(fabsf(d[i].x), fabsf(d[i].y)));
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
    if (worst > kBorder<K>) {
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (fabsf(i & 1 ? d[i / 2].y : d[i / 2].x) > kBorder<K> && base + i < a.n) {
          if constexpr (NV > 0)
            doubtful |= 1u << (v * E + i);
          else
            codes[base + i] = (int8_t)code64(value64<K, T>(a, row, base + i), top64());
        }
    }
  }
  if (K != kPlain && NV > 0) __syncthreads();
  while (NV > 0 && doubtful) {
    const int j = __ffs(doubtful) - 1;
    doubtful &= doubtful - 1;
    const int i = (j / E * (int)blockDim.x + (int)threadIdx.x) * E + j % E;
    codes[i] = (int8_t)code64(value64<K, T>(a, row, i), top64());
  }
  if (threadIdx.x == 0) {
    double s = top64() / 127.0;
    if (NORM) s *= 1.0 / sqrt((double)ss / a.n + (double)a.eps);
    const float scale = (float)s;
    a.scales[row] = fabsf(scale) <= 3.402823466e38f ? scale : nanf("");
  }
}

template <Kind K, class T, int NV, bool ALIGNED>
void launch(const RowsArgs& a, int threads, cudaStream_t s) {
  launch_pdl(int8_rows_kernel<K, T, NV, ALIGNED>, dim3(a.rows), dim3(threads), 0, s, true, a);
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

// Codes times their row's scale: a CTA takes 4096 codes of a row, a thread four times
// four, so that a warp stores 512 bytes in a row.
constexpr int kDequant = 4096;

template <class T>
__global__ void __launch_bounds__(256) int8_dequant_kernel(const int8_t* codes, long long stride,
                                                           const float* scales, int n, int pieces,
                                                           T* out, long long out_stride,
                                                           bool aligned) {
  pdl_launch_dependents();
  pdl_wait();
  const long long row = blockIdx.x / pieces;
  const int base = (int)(blockIdx.x - row * pieces) * kDequant + threadIdx.x * 4;
  const int8_t* c = codes + row * stride;
  T* o = out + row * out_stride;
  const float s = scales[row];
  char4 q[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int i = base + j * 1024;
    if (i + 4 <= n)
      q[j] = *reinterpret_cast<const char4*>(c + i);
    else
      q[j] = make_char4(i < n ? c[i] : 0, i + 1 < n ? c[i + 1] : 0, i + 2 < n ? c[i + 2] : 0, 0);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int i = base + j * 1024;
    const float v[4] = {q[j].x * s, q[j].y * s, q[j].z * s, q[j].w * s};
    if (aligned && i + 4 <= n) {
      store_act4(o + i, make_float4(v[0], v[1], v[2], v[3]));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < n) store_one(o + i + e, v[e]);
    }
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
    const int pieces = (n + kDequant - 1) / kDequant;
    const long long blocks = (long long)rows * pieces;
    if (blocks > 0x7fffffffLL) invalid("Int8Dequantize: too many rows");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (out_type == MLB_ACT_BF16)
      launch_pdl(int8_dequant_kernel<__nv_bfloat16>, dim3((unsigned)blocks), dim3(256), 0, s, true,
                 codes, codes_stride, scales, n, pieces, static_cast<__nv_bfloat16*>(out),
                 out_stride, aligned);
    else
      launch_pdl(int8_dequant_kernel<float>, dim3((unsigned)blocks), dim3(256), 0, s, true, codes,
                 codes_stride, scales, n, pieces, static_cast<float*>(out), out_stride, aligned);
  });
}
