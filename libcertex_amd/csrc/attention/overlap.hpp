// Whether strided tensors share elements: what a call writes must not be what another of its threads reads or writes.
#pragma once

#include <algorithm>
#include <cstdint>

namespace certex_amd::attention {

/** A dimension: its extent, and its stride in elements (not negative). */
struct dimension {
  int64_t n, stride;
};

/**
 * Whether sum_i stride_i c_i = target for whole numbers c_i of [lo_i, hi_i], not all of them 0 if `moved` is false. Terms
 * are tried from the longest stride on, and of each only the numbers from which the others still reach the target:
 * two or three where the dimensions nest, as those of slices and transposed tensors do. Others end after kTries
 * tries with the answer true.
 */
class stride_equation {
 public:
  void add(int64_t stride, int64_t lo, int64_t hi)
  {
    if (stride != 0 && lo < hi) { t_[n_++] = {stride, lo, hi, 0, 0}; }
  }
  bool solvable(int64_t target, bool moved)
  {
    std::sort(t_, t_ + n_, [](term const& a, term const& b) { return a.stride > b.stride; });
    int64_t lo = 0, hi = 0;  // what the terms behind one reach
    for (int i = n_ - 1; i >= 0; --i) {
      t_[i].rest_lo = lo;
      t_[i].rest_hi = hi;
      lo += t_[i].stride * t_[i].lo;
      hi += t_[i].stride * t_[i].hi;
    }
    left_ = kTries;
    return search(0, target, moved);
  }

 private:
  static constexpr int kTries = 1 << 18;
  struct term {
    int64_t stride, lo, hi, rest_lo, rest_hi;
  };
  term t_[16];
  int n_    = 0;
  int left_ = 0;

  static int64_t floored(int64_t a, int64_t b) { return a / b - (a % b < 0 ? 1 : 0); }
  bool search(int i, int64_t target, bool moved)
  {
    if (--left_ < 0) { return true; }
    if (i == n_) { return target == 0 && moved; }
    term const& t      = t_[i];
    const int64_t from = std::max(t.lo, -floored(t.rest_hi - target, t.stride));
    const int64_t to   = std::min(t.hi, floored(target - t.rest_lo, t.stride));
    for (int64_t c = from; c <= to; ++c) {
      if (search(i + 1, target - c * t.stride, moved || c != 0)) { return true; }
    }
    return false;
  }
};

/** Whether two different elements of a tensor are one in memory. Extents are at least 1. */
inline bool shares_itself(dimension const* d, int n)
{
  stride_equation e;
  bool nested = true;
  for (int i = 0; i < n; ++i) {
    if (d[i].n > 1 && d[i].stride == 0) { return true; }
    e.add(d[i].stride, -(d[i].n - 1), d[i].n - 1);
    int64_t inner = 0;  // reach of the dimensions of shorter strides (of equal ones: both ways)
    for (int j = 0; j < n; ++j) {
      if (j != i && d[j].stride <= d[i].stride) { inner += d[j].stride * (d[j].n - 1); }
    }
    nested = nested && (d[i].n <= 1 || d[i].stride > inner);
  }
  return !nested && e.solvable(0, false);
}

/** Whether an element of a is one of b, whose first lies `distance` elements behind a's. Extents are at least 1. */
inline bool shares(dimension const* a, int na, dimension const* b, int nb, int64_t distance)
{
  int64_t a_reach = 0, b_reach = 0;
  for (int i = 0; i < na; ++i) { a_reach += a[i].stride * (a[i].n - 1); }
  for (int i = 0; i < nb; ++i) { b_reach += b[i].stride * (b[i].n - 1); }
  if (distance > a_reach || -distance > b_reach) { return false; }
  // a's index less b's, where both have a dimension of one stride: one term
  stride_equation e;
  bool used[8] = {};
  for (int i = 0; i < na; ++i) {
    int64_t lo = 0;
    for (int j = 0; j < nb; ++j) {
      if (!used[j] && b[j].stride == a[i].stride) {
        lo      = -(b[j].n - 1);
        used[j] = true;
        break;
      }
    }
    e.add(a[i].stride, lo, a[i].n - 1);
  }
  for (int j = 0; j < nb; ++j) {
    if (!used[j]) { e.add(b[j].stride, -(b[j].n - 1), 0); }
  }
  return e.solvable(distance, true);
}

}  // namespace certex_amd::attention
