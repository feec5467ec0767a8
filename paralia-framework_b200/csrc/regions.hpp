// What memory the columns of a matrix take, and whether two matrices share any.
#pragma once
#include <stdint.h>

#include <algorithm>

namespace paralia {

// `cols` runs of `bytes`, `stride` apart (a column-major matrix, or with one column a vector).
struct Region {
  int64_t at, bytes, stride, cols;
};

inline Region region(const void* p, int64_t rows, int64_t cols, int64_t ld, int64_t element_bytes) {
  Region r = {static_cast<int64_t>(reinterpret_cast<uintptr_t>(p)), 0, 0, 0};
  if (!p || rows <= 0 || cols <= 0) return r;
  r.bytes = rows * element_bytes;
  r.cols = cols;
  if (cols == 1) return r;                                    // its leading dimension has no meaning
  if (ld == rows) r = {r.at, r.bytes * cols, 0, 1};           // one run
  else r.stride = ld > INT64_MAX / 2 / element_bytes ? INT64_MAX / 2 : ld * element_bytes;
  return r;
}

// Whether the run [p, p + bytes) touches y, whose columns may start up to `ahead` columns before its first:
// `ahead` more runs that look like its own.
inline bool run_touches(__int128 p, __int128 bytes, const Region& y, int64_t ahead) {
  if (y.cols + ahead == 1) return p < (__int128)y.at + y.bytes && y.at < p + bytes;
  // the first column that ends behind p
  const __int128 past = p - y.at - y.bytes;
  __int128 k = past >= 0 ? past / y.stride + 1 : -((-past - 1) / y.stride);
  k = std::max(k, -(__int128)ahead);
  return k < y.cols && y.at + k * y.stride < p + bytes;
}

inline bool regions_overlap(const Region& a, const Region& b) {
  if (a.cols == 0 || b.cols == 0) return false;
  const __int128 a_end = (__int128)a.at + (__int128)(a.cols - 1) * a.stride + a.bytes;
  const __int128 b_end = (__int128)b.at + (__int128)(b.cols - 1) * b.stride + b.bytes;
  if (a_end <= b.at || b_end <= a.at) return false;
  // Views of one parent lie between each other's columns. With one stride only the difference of the column
  // numbers counts; otherwise each column of the matrix that has fewer is looked at.
  if (a.cols > 1 && a.stride == b.stride) return run_touches(a.at, a.bytes, b, a.cols - 1);
  const Region& x = a.cols <= b.cols ? a : b;
  const Region& y = a.cols <= b.cols ? b : a;
  for (int64_t j = 0; j < x.cols; ++j)
    if (run_touches((__int128)x.at + (__int128)j * x.stride, x.bytes, y, 0)) return true;
  return false;
}

}  // namespace paralia
