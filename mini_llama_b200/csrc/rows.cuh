// rows.cuh — checks of row-wise operands shared by the entry points.
#pragma once

#include <stdint.h>

namespace mlb {

using wide_int = __int128;  // strides are the caller's: their bytes may pass 64 bits

// Whether two sets of rows share a byte: n_a (n_b) rows of a_bytes (b_bytes), a_stride
// (b_stride) bytes apart, at least a row. Rows side by side in one buffer do not.
inline bool byte_rows_overlap(const void* a, wide_int a_stride, wide_int a_bytes, int n_a,
                              const void* b, wide_int b_stride, wide_int b_bytes, int n_b) {
  using wide = wide_int;
  if (n_a <= 0 || n_b <= 0 || a_bytes <= 0 || b_bytes <= 0) return false;
  const wide d = (wide)reinterpret_cast<uintptr_t>(b) - (wide)reinterpret_cast<uintptr_t>(a);
  const auto floor_div = [](wide x, wide y) { return x / y - (x % y < 0 ? 1 : 0); };
  // rows of b that row i of a meets: those with i a_stride - j b_stride - d in (-a_bytes, b_bytes)
  const auto meets = [&](wide at, wide j0, wide j1) {
    const wide lo = floor_div(at - d - b_bytes, b_stride) + 1;
    const wide hi = floor_div(at - d + a_bytes - 1, b_stride);
    return (lo > j0 ? lo : j0) <= (hi < j1 ? hi : j1);
  };
  // of equal strides only the difference of the rows counts
  if (a_stride == b_stride) return meets(0, -(wide)(n_a - 1), n_b - 1);
  if (d >= (wide)(n_a - 1) * a_stride + a_bytes || -d >= (wide)(n_b - 1) * b_stride + b_bytes)
    return false;
  for (int i = 0; i < n_a; ++i)
    if (meets((wide)i * a_stride, 0, n_b - 1)) return true;
  return false;
}

}  // namespace mlb
