// rope_rows.h — whether the 256-lane rows of two tensors share memory.  Plain
// C++, for the C entries and the torch binding alike.

#ifndef WELM_ROPE_ROWS_H_
#define WELM_ROPE_ROWS_H_

#include <cstdint>

#include "welm_rope.h"

namespace {

// Rows of WELM_ROPE_HEAD_DIM two-byte lanes at `at` and the given (not
// negative) strides, in elements, from it.
struct RowSet {
  uintptr_t at;
  int64_t extent[3], stride[3];
};

// Elements from the first lane to behind the last; 0 where there are no rows.
inline __int128 rows_span(const RowSet& r) {
  __int128 span = WELM_ROPE_HEAD_DIM;
  for (int i = 0; i < 3; ++i) {
    if (r.extent[i] <= 0) return 0;
    span += __int128(r.stride[i]) * (r.extent[i] - 1);
  }
  return span;
}

// The dimensions of a RowSet that step, the largest stride first.
struct RowDims {
  int n = 0;
  int64_t extent[3], stride[3];
  explicit RowDims(const RowSet& r) {
    for (int i = 0; i < 3; ++i) {
      if (r.extent[i] <= 1 || r.stride[i] == 0) continue;
      int at = n++;
      for (; at > 0 && stride[at - 1] < r.stride[i]; --at) {
        stride[at] = stride[at - 1];
        extent[at] = extent[at - 1];
      }
      stride[at] = r.stride[i];
      extent[at] = r.extent[i];
    }
  }
};

// Rows i of a's and j of b's largest stride T meet where those of the
// dimensions below do, displaced by d + (j - i) T; only displacements within
// their spans have to be looked at, one or two where rows of equal steps
// interleave.  Exact, unless that takes more than `steps` of them: then true.
template <typename Int>
bool rows_meet_at(const RowDims& a, int ai, Int span_a, const RowDims& b, int bi, Int span_b, Int d, int& steps) {
  if (d >= span_a || -d >= span_b) return false;
  if (ai == a.n && bi == b.n) return true;
  const int64_t sa = ai < a.n ? a.stride[ai] : 0, sb = bi < b.n ? b.stride[bi] : 0;
  const Int step = sa > sb ? sa : sb;
  Int lo = 0, hi = 0;
  if (sa == step) {
    lo = -Int(a.extent[ai] - 1);
    span_a += lo * step;
    ++ai;
  }
  if (sb == step) {
    hi = b.extent[bi] - 1;
    span_b -= hi * step;
    ++bi;
  }
  auto floor_div = [](Int x, Int y) { return x / y - (x % y < 0); };
  const Int first = -floor_div(span_b - 1 + d, step), last = floor_div(span_a - 1 - d, step);
  if (lo < first) lo = first;
  if (hi > last) hi = last;
  for (Int m = lo; m <= hi; ++m) {
    if (--steps < 0 || rows_meet_at(a, ai, span_a, b, bi, span_b, d + m * step, steps)) return true;
  }
  return false;
}

inline bool rows_meet(const RowSet& x, const RowSet& y) {
  const __int128 span_x = rows_span(x), span_y = rows_span(y);
  const __int128 d = (__int128(y.at) - __int128(x.at)) / 2;  // rows begin at even addresses
  if (d >= span_x || -d >= span_y || span_x == 0 || span_y == 0) return false;
  const RowDims a(x), b(y);
  int steps = 4096;
  // the usual case in 64 bits, whose divisions are ten times as fast
  if (((span_x | span_y) >> 61) == 0) return rows_meet_at<int64_t>(a, 0, span_x, b, 0, span_y, d, steps);
  return rows_meet_at<__int128>(a, 0, span_x, b, 0, span_y, d, steps);
}

}  // namespace

#endif  // WELM_ROPE_ROWS_H_
