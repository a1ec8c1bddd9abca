// int8_rows.cu — rows of activations or weights as int8 codes with one scale each:
// as they are, after RMSNorm (with the residual's addition), or SiLU(gate) * up; and
// codes back as the values that they stand for.
//
//   A = max |t|,  code = rint(127 t / A) (ties to even),  scale = A / 127
//
// for a row of values t. RMSNorm's root is a factor of the whole row, so it cancels in
// the codes: they are those of t = h w, h the (rounded) sum, and the root enters the
// scale alone. One pass over the row in registers therefore yields both the sum of
// squares and the maximum. The sum is 64-bit throughout, so that scales keep their accuracy
// in the longest rows, and do not go by how a row is divided among threads, which goes by
// the number of rows (of fp32 sums every fourth scale did; of these one in 2^23 or fewer, whose
// exact value lies within 64-bit rounding of the middle of two fp32 numbers).
//
// Codes are those of 64-bit arithmetic. Computed in fp32 (v = t 127 / A), a value next
// to a code's border could fall on either side of it, so the fp32 result is taken only
// where it is further from the border than its error bound, and the few others (2 in
// 10^5 after a norm, 4 in 10^5 of SiLU) are done again in 64 bits, from the inputs. Those
// need A in 64 bits: the threads that hold a value within the bound of the fp32 maximum
// compute theirs again, while the others go on, and a second barrier later the doubtful
// codes are corrected. Rows whose fp32 maximum leaves the range where the bounds hold
// (below 1e-30, not finite, gates below -87) are done in 64 bits throughout.
//
// A row with a NaN or an infinity among its values, or a scale past fp32's largest
// number, gets the scale NaN: every product of it is NaN, whatever its codes.
//
// Bound by a row's chain (load, reduction, the 64-bit maximum, codes), which 32 warps per
// SM hide in part: 4096 rows of 8192 bf16, norm with residual 44 us (5.4 TB/s), norm 30.6
// (3.3), SiLU product 40 (4.2), as they are 25 (4.0); fp32 79 (5.5), 40.3 (4.2), 52 (5.8),
// 29.6 (5.7). Codes back to values are bound by HBM (26.5 us, 6.3 TB/s). One row of 4096 fp32:
// norm with residual 2.8 us, norm 2.3, SiLU product 2.5, as it is 1.8, back 1.3.
#include <cuda_bf16.h>

#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "paged.cuh"
#include "rows.cuh"
#include "tcgen05.cuh"

namespace mlb {

namespace {

enum Kind { kPlain, kNorm, kNormAdd, kSilu };
enum Form { kAlone, kStream, kShared };  // how CTAs and rows meet, as at the kernel

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
  int log_share;  // 2^log_share CTAs, a cluster, share a row
};

constexpr int kHeld = 32;  // values that a thread holds at most
constexpr int kMostLogShare = 3;
constexpr float kSmallest = 1e-30f;
constexpr float kLowestGate = -87.0f;  // e^87 is a normal number, and so is its reciprocal
constexpr float kUnit = 0x1p-24f;
// Relative error bounds. t: after a norm one product (1 unit); SiLU: ex2 4 (2 ulp), the
// factor that corrects it, the sum and two products 1 each, the reciprocal 2: 10 together.
// A value is taken for the maximum's candidate within twice that, and a little more.
template <Kind K>
constexpr float kNear = 1.0f - (K == kSilu ? 24.0f : 4.0f) * kUnit;
// v: t's, the maximum's (the same) and its reciprocal's times 127 (1); the last product is
// exact in a fused multiply-add. A code is taken where t times that reciprocal a little
// more than so many units up and down comes to the same.
template <Kind K>
constexpr float kDoubt = (K == kSilu ? 24.0f : K == kPlain ? 4.0f : 6.0f) * kUnit;

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// E elements at once: 16 bytes where rows are aligned, one element where they are not.
template <class T, int E>
struct Raw {
  using type = uint4;
  static __device__ __forceinline__ uint4 zero() { return make_uint4(0u, 0u, 0u, 0u); }
};
template <class T>
struct Raw<T, 1> {
  using type = T;
  static __device__ __forceinline__ T zero() { return T(0.0f); }
};
template <class T, int E>
using raw_t = typename Raw<T, E>::type;

template <class T, int E>
__device__ __forceinline__ void widen(const raw_t<T, E>& u, float (&v)[E]) {
  if constexpr (E == 1) {
    v[0] = to_float(u);
  } else {
    const uint32_t words[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (sizeof(T) == 4) {
        v[j] = __uint_as_float(words[j]);
      } else {
        v[2 * j] = __uint_as_float(words[j] << 16);
        v[2 * j + 1] = __uint_as_float(words[j] & 0xffff0000u);
      }
    }
  }
}
// x + r rounded to T. Of two bf16 the fp32 sum rounds to the same bf16 as the exact one:
// it is inexact only where one is below 2^-16 of the other, which is then the result.
__device__ __forceinline__ float add_round(float x, float r) { return x + r; }
__device__ __forceinline__ __nv_bfloat16 add_round(__nv_bfloat16 x, __nv_bfloat16 r) {
  return __hadd(x, r);
}
__device__ __forceinline__ uint32_t add_words(uint32_t x, uint32_t r, float) {
  return __float_as_uint(__uint_as_float(x) + __uint_as_float(r));
}
__device__ __forceinline__ uint32_t add_words(uint32_t x, uint32_t r, __nv_bfloat16) {
  const __nv_bfloat162 s = __hadd2(*reinterpret_cast<const __nv_bfloat162*>(&x),
                                   *reinterpret_cast<const __nv_bfloat162*>(&r));
  return *reinterpret_cast<const uint32_t*>(&s);
}
template <class T, int E>
__device__ __forceinline__ raw_t<T, E> add_raw(const raw_t<T, E>& x, const raw_t<T, E>& r) {
  if constexpr (E == 1)
    return add_round(x, r);
  else
    return make_uint4(add_words(x.x, r.x, T()), add_words(x.y, r.y, T()),
                      add_words(x.z, r.z, T()), add_words(x.w, r.w, T()));
}

__device__ __forceinline__ void store_one(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_one(__nv_bfloat16* p, float v) {
  *p = __float2bfloat16_rn(v);
}

// A slot on its way into shared memory.
__device__ __forceinline__ void fetch_slot(uint4* slot, const void* p) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(slot)), "l"(p)
               : "memory");
}

// |x| and |y|'s larger, NaN if one is.
__device__ __forceinline__ float max_abs(float x, float y) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(fabsf(y)));
  return r;
}

// SiLU(g) * u. e^-g = 2^(hi + lo), -g log2(e) in two parts; 2^lo as 1 + lo ln 2. The
// reciprocal goes to u first: g may be any number, u a large one, and g times the reciprocal
// below the normal numbers, where it loses its bits. The reciprocal times u does so only
// where u is that small: then it is u itself (a reciprocal of 1, to half a step of u), or,
// as g is between -87 and 17, the result is below 1e-36, 0 beside any maximum in range.
__device__ __forceinline__ float silu_mul(float g, float u) {
  const float hi = g * -1.4426950408889634f;
  // what hi's rounding and the constant's (1.92596e-8 beyond fp32) leave, times ln 2
  const float lo = fmaf(g, -1.4426950408889634f, -hi) * 0.6931471805599453f + g * -1.33497e-8f;
  float e = ex2(hi), r;
  e = fmaf(e, lo, e);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return g * (r * u);
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
  float part[32];    // per warp: maximum
  double part64[32];
  unsigned long long top;  // bits of the 64-bit maximum
  float share[1 << kMostLogShare];  // per CTA of the row's: maximum
  double2 share64[1 << kMostLogShare];  // per CTA: maximum and sum of squares in 64 bits
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
template <Kind K, class T>
__device__ __noinline__ void row64(const RowsArgs& a, long long row, Shared& sh) {
  double sum = 0.0, top = 0.0;
  __syncthreads();  // sums and inputs of every thread are there
  for (int i = threadIdx.x; i < a.n; i += blockDim.x) {
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
  for (int i = threadIdx.x; i < a.n; i += blockDim.x)
    codes[i] = none ? 0 : (int8_t)code64(value64<K, T>(a, row, i), top);
  if (threadIdx.x == 0) a.scales[row] = scale;
}

// The maximum of a row from its threads'.
__device__ __forceinline__ float join_row(float top, Shared& sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
  if (lane == 0) sh.part[warp] = top;
  if (threadIdx.x == 0) sh.top = 0;
  __syncthreads();
  uint32_t bits = 0;
  if (warps <= 8) {
    for (int i = 0; i < warps; ++i) bits = max(bits, __float_as_uint(sh.part[i]));
  } else {
    bits = __reduce_max_sync(0xffffffffu, lane < warps ? __float_as_uint(sh.part[lane]) : 0u);
  }
  return __uint_as_float(bits);
}
// The same of a row that CTAs share, from theirs.
__device__ __forceinline__ float join_shares(float top, int rank, int log_share, Shared& sh) {
  cluster_wait();  // every CTA is there
  if (threadIdx.x < 1u << log_share)
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(
                     cluster_address(&sh.share[rank], threadIdx.x)),
                 "f"(top)
                 : "memory");
  cluster_sync_all();
  uint32_t bits = 0;
  for (int i = 0; i < 1 << log_share; ++i) bits = max(bits, __float_as_uint(sh.share[i]));
  return __uint_as_float(bits);
}
// The sum of squares from its threads', which lie in shared memory behind a barrier: one
// warp's work while the others make codes. (Every warp's lanes' by shuffles: 4096 rows of 8192
// as fast, one of 4096 fp32 2.5 us instead of 2.3, 5768 of 12664 bf16 with residual 123
// instead of 111.)
__device__ __forceinline__ double all_squares(const double* squares) {
  const int lane = threadIdx.x & 31;
  const int pairs = blockDim.x / 2;
  const double2* p = reinterpret_cast<const double2*>(squares);
  double2 a = make_double2(0.0, 0.0), b = a;
  for (int i = lane; i < pairs; i += 64) {
    const double2 q = p[i];
    const double2 r = i + 32 < pairs ? p[i + 32] : make_double2(0.0, 0.0);
    a.x += q.x, a.y += q.y, b.x += r.x, b.y += r.y;
  }
  double ss = (a.x + a.y) + (b.x + b.y);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  return ss;
}
// Maximum and sum of squares in 64 bits of a row that CTAs share.
__device__ __forceinline__ void join_shares64(double& top, double& ss, bool keeper, int rank,
                                              int log_share, Shared& sh) {
  const unsigned lane = threadIdx.x & 31;
  if (keeper && lane < 1u << log_share)
    asm volatile("st.shared::cluster.v2.f64 [%0], {%1, %2};" ::"r"(
                     cluster_address(&sh.share64[rank], lane)),
                 "d"(top), "d"(ss)
                 : "memory");
  cluster_sync_all();
  ss = 0.0;
  for (int i = 0; i < 1 << log_share; ++i) {
    top = fmax(top, sh.share64[i].x);
    ss += sh.share64[i].y;
  }
}
// Whether the error bounds hold (NaN fails the comparisons).
__device__ __forceinline__ bool in_range(float top) { return top >= kSmallest && top <= 3e38f; }
template <Kind K, class T>
__device__ __forceinline__ void candidate(const RowsArgs& a, long long row, int i, Shared& sh) {
  const double t = fabs(value64<K, T>(a, row, i));
  atomicMax(&sh.top, (unsigned long long)__double_as_longlong(t));
}
template <Kind K>
__device__ __forceinline__ void store_scale(const RowsArgs& a, long long row, double top, double ss) {
  double s = top / 127.0;
  if (K == kNorm || K == kNormAdd) s *= 1.0 / sqrt(ss / a.n + (double)a.eps);
  const float scale = (float)s;
  a.scales[row] = fabsf(scale) <= 3.402823466e38f ? scale : nanf("");
}

constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23: a sum's low bits are the whole number

// One CTA per row at a time; thread j has elements (v blockDim + j) E + 0 .. E - 1, v < NV,
// which cover the row, and holds their values in registers. E > 1: rows start at 16-byte
// boundaries and have whole units of E. kStream: a CTA takes row after row and has the next
// one on its way, every thread its own elements, in shared memory slots of its own.
// kShared: a cluster takes a row; blockDim above is that of all its CTAs, and what their
// barriers join the cluster's join once more. (As a choice at run time it spilled, for a
// quarter more time of one row of 29568 fp32, norm with residual.)
template <Kind K, class T, int E, int NV, Form F>
__global__ void __launch_bounds__(1024) int8_rows_kernel(const RowsArgs a) {
  constexpr bool NORM = K == kNorm || K == kNormAdd, TWO = K == kNormAdd || K == kSilu;
  constexpr bool STREAM = F == kStream, SHARED = F == kShared;
  static_assert(!STREAM || E > 1);
  using R = raw_t<T, E>;
  __shared__ Shared shared[2];  // of rows in turn: one is read while the next is written
  extern __shared__ uint4 slots[];
  // of a norm: its threads' sums of squares, and the warp that keeps the row's
  constexpr int SLOTS = STREAM ? NV * (TWO ? 2 : 1) : 0;  // of a thread
  double* squares = reinterpret_cast<double*>(slots + SLOTS * (int)blockDim.x);
  const bool keeper = threadIdx.x >> 5 == (NORM ? (blockDim.x >> 5) - 1 : 0);
  const int log_share = SHARED ? a.log_share : 0, rank = blockIdx.x & ((1 << log_share) - 1);
  const int first = (rank * (int)blockDim.x + (int)threadIdx.x) * E;
  const int step = ((int)blockDim.x << log_share) * E;
  if constexpr (SHARED) cluster_arrive();
  const auto fetch = [&](long long row) {
    if (row < a.rows) {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int i = first + v * step;
        uint4* slot = slots + v * (int)blockDim.x + threadIdx.x;
        if (i < a.n) {
          fetch_slot(slot, static_cast<const T*>(a.x) + row * a.x_stride + i);
          if constexpr (TWO)
            fetch_slot(slot + NV * (int)blockDim.x, static_cast<const T*>(a.y) + row * a.y_stride + i);
        }
      }
    }
    cp_async_commit();
  };
  pdl_launch_dependents();
  pdl_wait();
  if constexpr (STREAM) fetch(blockIdx.x);

  int turn = 0;
  for (long long row = blockIdx.x >> log_share; row < a.rows;
       row += gridDim.x >> log_share, turn ^= 1) {
    Shared& sh = shared[turn];
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* y = static_cast<const T*>(a.y) + row * a.y_stride;
    if constexpr (STREAM) cp_async_wait_all();
    float t[NV][E], top = 0.0f, low = 0.0f;
    // Sums of squares, several where the next row's loads hide behind them (in us, 1 / 2 / 4:
    // 4096 rows of 8192 with residual fp32 81 / 82 / 78.5, bf16 45.5 / 43.7 / 43.9; norm of
    // 16384 of 1000 fp32 26.9 / 29.0 / 28.1; where rows are not streamed they spill: 300 of
    // 65536 with residual fp32 78 / 89 / 98)
    constexpr int SUMS = !STREAM ? 1 : sizeof(T) == 2 ? 2 : K == kNormAdd ? 4 : 1;
    double sums[SUMS] = {};
    // a batch is asked for at once: the sums' stores, which may lie over the inputs, would
    // otherwise keep each load behind the one before (2048 rows of 8191, norm with residual, 8 /
    // 16 elements: fp32 79 / 65 us, bf16 85 / 65; 32 spilled)
    constexpr int BATCH = E == 1 ? (NV <= 16 ? NV : 8) : NV < 4 ? NV : 4;
    R asked[2][BATCH];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int i = first + v * step;
      const bool there = i < a.n;
      if (!STREAM && v % BATCH == 0) {
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
          const int j = i + k * step;
          asked[0][k] = asked[1][k] = Raw<T, E>::zero();
          if (j < a.n) {
            asked[0][k] = *reinterpret_cast<const R*>(x + j);
            if constexpr (TWO) asked[1][k] = *reinterpret_cast<const R*>(y + j);
          }
        }
      }
      R u = Raw<T, E>::zero(), o = Raw<T, E>::zero();
      if constexpr (!STREAM) {
        u = asked[0][v % BATCH], o = asked[1][v % BATCH];
      } else if (there) {
        const uint4* slot = slots + v * (int)blockDim.x + threadIdx.x;
        u = *slot;
        if constexpr (TWO) o = slot[NV * (int)blockDim.x];
      }
      if constexpr (K == kNormAdd) {
        u = add_raw<T, E>(u, o);
        if (there)
          *reinterpret_cast<R*>(static_cast<T*>(a.sum) + row * a.sum_stride + i) = u;
      }
      float p[E];
      widen<T, E>(u, p);
      if constexpr (NORM) {
        float w[E];
        if constexpr (E == 1) {
          w[0] = there ? a.w[i] : 0.0f;
        } else {
#pragma unroll
          for (int e = 0; e < E; e += 4) {
            float4 q = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (there) q = *reinterpret_cast<const float4*>(a.w + i + e);
            w[e] = q.x, w[e + 1] = q.y, w[e + 2] = q.z, w[e + 3] = q.w;
          }
        }
        if constexpr (E == 1) {
          sums[0] = fma((double)p[0], (double)p[0], sums[0]);
          t[v][0] = p[0] * w[0];
        } else {
#pragma unroll
          for (int e = 0; e < E; e += 2) {
            const float2 q = make_float2(p[e], p[e + 1]);
            double& s0 = sums[e % SUMS];
            s0 = fma((double)q.x, (double)q.x, s0);
            double& s1 = sums[(e + 1) % SUMS];
            s1 = fma((double)q.y, (double)q.y, s1);
            const float2 m = mul2(q, make_float2(w[e], w[e + 1]));
            t[v][e] = m.x, t[v][e + 1] = m.y;
          }
        }
      } else if constexpr (K == kSilu) {
        float q[E];
        widen<T, E>(o, q);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          low = fminf(low, p[e]);
          t[v][e] = silu_mul(p[e], q[e]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) t[v][e] = p[e];
      }
#pragma unroll
      for (int e = 0; e < E; ++e) top = max_abs(top, t[v][e]);
    }
    // the slots have been read; but for the maximum's candidates, which are nearer there
    // than in memory (SiLU product 44 us so, 40 with the copies after them; with a residual,
    // whose sum is not there, 47 and 48)
    constexpr bool EARLY = STREAM && (K == kPlain || K == kNormAdd);
    if constexpr (EARLY) fetch(row + gridDim.x);
    if (K == kSilu && low < kLowestGate) top = nanf("");
    const float mine = top;
    double ss = sums[0];
#pragma unroll
    for (int i = 1; i < SUMS; ++i) ss += sums[i];
    if constexpr (NORM) squares[threadIdx.x] = ss;
    top = join_row(top, sh);
    if constexpr (SHARED) top = join_shares(top, rank, log_share, sh);
    if (!in_range(top)) {  // the same for all threads of the row
      if constexpr (STREAM && !EARLY) fetch(row + gridDim.x);
      if (rank == 0) row64<K, T>(a, row, sh);
      continue;
    }
    // the maximum in 64 bits: of the values that may be it
    const float near = top * kNear<K>;
    const auto candidate = [&](double value) {
      atomicMax(&sh.top, (unsigned long long)__double_as_longlong(fabs(value)));
    };
    if (K == kNormAdd && mine >= near) {
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (fabsf(t[v][e]) >= near) candidate(value64<K, T>(a, row, first + v * step + e));
    } else if (K != kPlain && mine >= near) {
      uint32_t named = 0;  // bit v E + e
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (fabsf(t[v][e]) >= near) named |= 1u << (v * E + e);
      while (named) {
        const int j = __ffs(named) - 1, i = first + j / E * step + j % E;
        named &= named - 1;
        if constexpr (STREAM) {
          const uint4* slot = slots + j / E * (int)blockDim.x + threadIdx.x;
          const float one = to_float(reinterpret_cast<const T*>(slot)[j % E]);
          if constexpr (K == kSilu) {
            const T* other = reinterpret_cast<const T*>(slot + NV * (int)blockDim.x);
            candidate(silu_mul64(one, to_float(other[j % E])));
          } else {
            candidate((double)one * (double)a.w[i]);
          }
        } else {
          candidate(value64<K, T>(a, row, i));
        }
      }
    }
    if constexpr (STREAM && !EARLY) fetch(row + gridDim.x);
    if (NORM && keeper) ss = all_squares(squares);

    const float inv = __fdiv_rn(127.0f, top);
    const float up = inv * (1.0f + kDoubt<K>), down = inv * (1.0f - kDoubt<K>);
    int8_t* codes = a.codes + row * a.codes_stride;
    uint32_t doubtful = 0;  // bit v E + e
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int i = first + v * step;
      uint32_t c[E], other[E], differ = 0;
      if constexpr (E == 1) {
        c[0] = __float_as_uint(fmaf(t[v][0], up, kMagic));
        other[0] = __float_as_uint(fmaf(t[v][0], down, kMagic));
      } else {
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          const float2 q = make_float2(t[v][e], t[v][e + 1]), m = make_float2(kMagic, kMagic);
          const float2 r = fma2(q, make_float2(up, up), m);
          const float2 s = fma2(q, make_float2(down, down), m);
          c[e] = __float_as_uint(r.x), c[e + 1] = __float_as_uint(r.y);
          other[e] = __float_as_uint(s.x), other[e + 1] = __float_as_uint(s.y);
        }
      }
#pragma unroll
      for (int e = 0; e < E; ++e) differ |= c[e] ^ other[e];
      if (i < a.n) {
        if constexpr (E == 1) {
          codes[i] = (int8_t)(c[0] & 0xffu);
        } else {
          uint32_t words[E / 4];
#pragma unroll
          for (int e = 0; e < E / 4; ++e)
            words[e] = __byte_perm(__byte_perm(c[4 * e], c[4 * e + 1], 0x0040),
                                   __byte_perm(c[4 * e + 2], c[4 * e + 3], 0x0040), 0x5410);
          if constexpr (E == 8)
            *reinterpret_cast<uint2*>(codes + i) = make_uint2(words[0], words[1]);
          else
            *reinterpret_cast<uint32_t*>(codes + i) = words[0];
        }
      }
      if (differ) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (c[e] != other[e]) doubtful |= 1u << (v * E + e);
      }
    }
    if (K != kPlain) __syncthreads();
    double top64 = K == kPlain ? (double)top : __longlong_as_double((long long)sh.top);
    if constexpr (K != kPlain && SHARED) join_shares64(top64, ss, keeper, rank, log_share, sh);
    while (doubtful) {
      const int j = __ffs(doubtful) - 1;
      doubtful &= doubtful - 1;
      const int i = first + j / E * step + j % E;
      codes[i] = (int8_t)code64(value64<K, T>(a, row, i), top64);
    }
    if (rank == 0 && keeper && (threadIdx.x & 31) == 0) store_scale<K>(a, row, top64, ss);
  }
}

// Rows too long for eight CTAs' registers: the same, one element at a time, values computed
// twice. With a residual two CTAs fit on an SM, at 32 registers (300 rows of 300000 fp32 784
// us, one at the 39 that it takes otherwise 1181).
template <Kind K, class T>
__global__ void __launch_bounds__(1024, K == kNormAdd ? 2 : 1)
    int8_long_rows_kernel(const RowsArgs a) {
  constexpr bool NORM = K == kNorm || K == kNormAdd;
  __shared__ Shared sh;
  extern __shared__ uint4 slots[];
  double* squares = reinterpret_cast<double*>(slots);
  const long long row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  const T* y = static_cast<const T*>(a.y) + row * a.y_stride;
  T* sum = static_cast<T*>(a.sum) + row * a.sum_stride;
  pdl_launch_dependents();
  pdl_wait();
  float top = 0.0f;
  double ss = 0.0;
  const auto value = [&](int i, bool again) {
    if constexpr (K == kSilu) {
      const float g = to_float(x[i]);
      return g < kLowestGate ? nanf("") : silu_mul(g, to_float(y[i]));
    }
    T h = K == kNormAdd && again ? sum[i] : x[i];
    if constexpr (K == kNormAdd)
      if (!again) sum[i] = h = add_round(h, y[i]);
    const float f = to_float(h);
    if (NORM && !again) ss = fma((double)f, (double)f, ss);
    return NORM ? f * a.w[i] : f;
  };
  for (int i = threadIdx.x; i < a.n; i += 1024) top = max_abs(top, value(i, false));
  const float mine = top;
  if constexpr (NORM) squares[threadIdx.x] = ss;
  top = join_row(top, sh);
  if (!in_range(top)) {
    row64<K, T>(a, row, sh);
    return;
  }
  const float near = top * kNear<K>;
  if (K != kPlain && mine >= near)
    for (int i = threadIdx.x; i < a.n; i += 1024)
      if (fabsf(value(i, true)) >= near) candidate<K, T>(a, row, i, sh);
  __syncthreads();
  const double top64 = K == kPlain ? (double)top : __longlong_as_double((long long)sh.top);
  const float inv = __fdiv_rn(127.0f, top);
  const float up = inv * (1.0f + kDoubt<K>), down = inv * (1.0f - kDoubt<K>);
  int8_t* codes = a.codes + row * a.codes_stride;
  for (int i = threadIdx.x; i < a.n; i += 1024) {
    const float t = value(i, true);
    const uint32_t c = __float_as_uint(fmaf(t, up, kMagic));
    int code = (int)(int8_t)(c & 0xffu);
    if (c != __float_as_uint(fmaf(t, down, kMagic))) code = code64(value64<K, T>(a, row, i), top64);
    codes[i] = (int8_t)code;
  }
  __syncwarp();
  if (threadIdx.x < 32) {
    if constexpr (NORM) ss = all_squares(squares);
    if (threadIdx.x == 0) store_scale<K>(a, row, top64, ss);
  }
}

constexpr int kSquareBytes = sizeof(double);  // of a norm's thread

template <Kind K, class T, int E, int NV>
void launch(const RowsArgs& a, int threads, int device_id, cudaStream_t s) {
  const int squares = K == kNorm || K == kNormAdd ? threads * kSquareBytes : 0;
  if constexpr (E > 1 && NV > 1) {
    // as many CTAs as 64 registers a thread and their slots leave room for
    const int bytes = threads * NV * 16 * (K == kNormAdd || K == kSilu ? 2 : 1) + squares;
    constexpr int kRoom = 220 * 1024;
    const int per_sm = std::min(1024 / threads, kRoom / (bytes + 2 * (int)sizeof(Shared) + 1024));
    if (a.log_share == 0 && per_sm > 0 && a.rows > per_sm * sm_count(device_id)) {
      const auto kernel = int8_rows_kernel<K, T, E, NV, kStream>;
      allow_smem(kernel, kRoom, device_id);
      return launch_pdl(kernel, dim3(per_sm * sm_count(device_id)), dim3(threads), bytes, s, true, a);
    }
  }
  if (a.log_share == 0)
    return launch_pdl(int8_rows_kernel<K, T, E, NV, kAlone>, dim3(a.rows), dim3(threads), squares, s,
                      true, a);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.rows << a.log_share);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = (size_t)squares;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 1u << a.log_share;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  MLB_CUDA(cudaLaunchKernelEx(&cfg, int8_rows_kernel<K, T, E, NV, kShared>, a));
}

template <Kind K, class T>
void dispatch(RowsArgs a, bool aligned, int device_id, cudaStream_t s) {
  constexpr int E = 16 / (int)sizeof(T);
  // CTAs that share a row: as many as its values take registers of, rather than passing
  // over it twice (norm with residual, norm, SiLU product, as it is, 300 rows of 65536, in
  // us: fp32 178, 90, 186, 53 with one CTA's two passes, 79, 50, 65, 37.5 shared, bf16 142, 81,
  // 129, 28 and 57, 39, 50, 30)
  const auto held = [&](int log_share) {  // threads that hold a row, of each CTA
    return ((a.n + (kHeld << log_share) - 1) / (kHeld << log_share));
  };
  a.log_share = 0;
  while (a.log_share < kMostLogShare && held(a.log_share) > 1024) ++a.log_share;
  if (held(a.log_share) > 1024 || (a.log_share > 0 && a.rows >= 1 << (31 - kMostLogShare)))
    return launch_pdl(int8_long_rows_kernel<K, T>, dim3(a.rows), dim3(1024),
                      K == kNorm || K == kNormAdd ? 1024 * kSquareBytes : 0, s, true, a);
  // Few rows of more than 32 KB: as many as SMs and 2048 elements each allow, if they are
  // four or more of 8192 or less (SiLU product and as it is, alone / shared, in us: one row
  // of 29568 fp32 6.5, 3.8 / 3.8, 2.4, bf16 5.7, 3.2 / 3.7, 2.7; 16 rows 6.9, 3.9 / 4.9, 3.4
  // and 6.1, 3.7 / 4.9, 3.5; one of 14336 fp32 4.4, 2.6 / 3.8, 2.4; in two, 64 of 14336 fp32
  // 4.7, 3.2 / 5.4, 3.5). Norms, which would gain as much (one row of 29568 fp32 with
  // residual 8.7 / 4.2, 16 rows 8.8 / 5.4), are not shared yet.
  if ((K == kPlain || K == kSilu) && (long long)a.n * (int)sizeof(T) > 32768) {
    int log_share = a.log_share;
    while (log_share < kMostLogShare &&
           (long long)a.rows << (log_share + 1) <= sm_count(device_id) &&
           a.n >> (log_share + 1) >= 2048)
      ++log_share;
    if (log_share >= 2 && a.n >> log_share <= 8192) a.log_share = log_share;
  }
  // few rows: up to 512 threads for each, for the time of one; many: 16 elements a thread,
  // or 32 of aligned bf16 rows, for less work around their reductions, where no residual
  // takes registers (4096 rows of 8192, 16 / 32 elements, in us: norm with residual bf16 44
  // / 50, fp32 79 / 98; norm bf16 32.6 / 30.6, fp32 40 / 44; SiLU product bf16 41.6 / 39.6,
  // fp32 52 / 54; as they are bf16 27.6 / 25, fp32 29.6 / 32; 2048 unaligned rows of 8191 bf16,
  // norm with residual 64 / 82, SiLU product 46 / 55, but norm 54 / 48.5)
  const bool few = a.rows <= 2 * sm_count(device_id);
  const auto threads_for = [&](int per) {
    per <<= a.log_share;
    return ((a.n + per - 1) / per + 31) / 32 * 32;
  };
  const bool wide = aligned && sizeof(T) == 2 && K != kNormAdd;
  const int most = few ? 512 : std::min(1024, threads_for(wide ? kHeld : 16));
  int per = aligned ? E : 8;  // elements a thread
  while (per < kHeld && threads_for(per) > most) per *= 2;
  const int threads = threads_for(per);
  if (!aligned) {
    if (per == 8) return launch<K, T, 1, 8>(a, threads, device_id, s);
    if (per == 16) return launch<K, T, 1, 16>(a, threads, device_id, s);
    return launch<K, T, 1, 32>(a, threads, device_id, s);
  }
  if (per == E) return launch<K, T, E, 1>(a, threads, device_id, s);
  if (per == 2 * E) return launch<K, T, E, 2>(a, threads, device_id, s);
  if (per == 4 * E) return launch<K, T, E, 4>(a, threads, device_id, s);
  if constexpr (8 * E <= kHeld) return launch<K, T, E, 8>(a, threads, device_id, s);
}

template <Kind K>
void run_rows(const RowsArgs& a, int act_type, int device_id, void* stream) {
  DeviceScope scope(device_id);
  if (a.rows == 0) return;
  const int es = act_type == MLB_ACT_BF16 ? 2 : 4;
  const auto on16 = [&](const void* p, long long stride) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (a.rows == 1 || stride % (16 / es) == 0);
  };
  const bool aligned = a.n % (16 / es) == 0 && on16(a.x, a.x_stride) && (!a.y || on16(a.y, a.y_stride)) &&
                       (!a.sum || on16(a.sum, a.sum_stride)) &&
                       (!a.w || reinterpret_cast<uintptr_t>(a.w) % 16 == 0);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (act_type == MLB_ACT_BF16)
    dispatch<K, __nv_bfloat16>(a, aligned, device_id, s);
  else
    dispatch<K, float>(a, aligned, device_id, s);
}

// Codes times their row's scale: `across` threads (a power of two) take 16 of each row's
// codes, the others of a CTA the rows below. E codes at a time: four, so that a warp stores
// 512 bytes in a row, or one where rows of results do not start at boundaries of four.
template <class T, int E>
__global__ void __launch_bounds__(256) int8_dequant_kernel(const int8_t* codes, long long stride,
                                                           const float* scales, int rows, int n,
                                                           int log_across, int pieces, T* out,
                                                           long long out_stride) {
  pdl_launch_dependents();
  const int across = 1 << log_across;
  const unsigned down = blockIdx.x / (unsigned)pieces, piece = blockIdx.x - down * pieces;
  const long long row = (long long)down * (256 >> log_across) + (threadIdx.x >> log_across);
  const int first = ((int)threadIdx.x & (across - 1)) * E + (int)piece * 16 * across;
  if (row >= rows) return;
  const int8_t* c = codes + row * stride;
  T* o = out + row * out_stride;
  pdl_wait();
  const float s = scales[row];
  if constexpr (E == 4) {
    char4 q[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = first + j * 4 * across;
      q[j] = make_char4(0, 0, 0, 0);
      if (i + 4 <= n)
        q[j] = *reinterpret_cast<const char4*>(c + i);
      else if (i < n)
        q[j] = make_char4(c[i], i + 1 < n ? c[i + 1] : 0, i + 2 < n ? c[i + 2] : 0, 0);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = first + j * 4 * across;
      const float v[4] = {q[j].x * s, q[j].y * s, q[j].z * s, q[j].w * s};
      if (i + 4 <= n) {
        store_act4(o + i, make_float4(v[0], v[1], v[2], v[3]));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (i + e < n) store_one(o + i + e, v[e]);
      }
    }
  } else {
    int8_t q[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) q[j] = first + j * across < n ? c[first + j * across] : 0;
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (first + j * across < n) store_one(o + first + j * across, q[j] * s);
  }
}

template <class T>
void launch_dequant(const int8_t* codes, long long stride, const float* scales, int rows, int n,
                    T* out, long long out_stride, cudaStream_t s) {
  int log_across = 0;
  while (log_across < 8 && (16 << log_across) < n) ++log_across;
  const int down = 256 >> log_across, pieces = (n + (16 << log_across) - 1) / (16 << log_across);
  const long long blocks = ((long long)rows + down - 1) / down * pieces;
  if (blocks > 0x7fffffffLL) invalid("Int8Dequantize: too many rows");
  const bool aligned = reinterpret_cast<uintptr_t>(out) % (4 * sizeof(T)) == 0 &&
                       (rows == 1 || out_stride % 4 == 0);
  const auto kernel = aligned ? int8_dequant_kernel<T, 4> : int8_dequant_kernel<T, 1>;
  launch_pdl(kernel, dim3((unsigned)blocks), dim3(256), 0, s, true, codes, stride, scales, rows, n,
             log_across, pieces, out, out_stride);
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
  if (n > (1 << 28)) invalid(w + ": rows have more than 2^28 elements");
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
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (out_type == MLB_ACT_BF16)
      launch_dequant(codes, codes_stride, scales, rows, n, static_cast<__nv_bfloat16*>(out),
                     out_stride, s);
    else
      launch_dequant(codes, codes_stride, scales, rows, n, static_cast<float*>(out), out_stride, s);
  });
}
