// Whether two strided tensors share memory, and whether one holds an element twice.
//
// The addresses of a tensor are base + sum_k i_k s_k + u, 0 <= i_k < n_k, 0 <= u < element size.
// Two tensors meet where a bounded integer equation has a solution:
//   sum_k i_k s_k - sum_k j_k t_k + (u - v) = base_b - base_a
// It is searched term by term, the largest stride first: what the smaller terms can still reach
// bounds each term from both sides, and their greatest common divisor has to divide what is left.
// In views of one tensor (columns, interleaved or transposed parts) each stride passes the reach of
// the smaller ones, so at most three values a term are tried.
#pragma once

#include <c10/util/SmallVector.h>

#include <algorithm>
#include <cstdint>
#include <numeric>
#include <utility>

namespace dtb {

struct MemView {
  uintptr_t base;
  int elem;  // bytes of an element
  c10::SmallVector<long, 6> size, stride;  // stride in bytes
};

struct OverlapTerm {
  long c, lo, hi;  // c x with lo <= x <= hi, c > 0
};

using OverlapTerms = c10::SmallVector<OverlapTerm, 13>;

// Whether sum c x = d has a solution.  Gives up after `budget` steps, and then says yes.
class BoundedSum {
 public:
  explicit BoundedSum(OverlapTerms terms) : t_(std::move(terms)) {
    std::sort(t_.begin(), t_.end(), [](const OverlapTerm& a, const OverlapTerm& b) { return a.c > b.c; });
    size_t m = 0;  // terms of one coefficient are one term
    for (const auto& x : t_) {
      if (m && t_[m - 1].c == x.c) {
        t_[m - 1].lo += x.lo;
        t_[m - 1].hi += x.hi;
      } else {
        t_[m++] = x;
      }
    }
    t_.resize(m);
    lo_.assign(m + 1, 0);
    hi_.assign(m + 1, 0);
    div_.assign(m + 1, 0);
    for (size_t i = m; i-- > 0;) {
      lo_[i] = lo_[i + 1] + t_[i].c * t_[i].lo;
      hi_[i] = hi_[i + 1] + t_[i].c * t_[i].hi;
      div_[i] = std::gcd(div_[i + 1], t_[i].c);
    }
  }
  bool reaches(long d) {
    budget_ = 1 << 16;
    return search(0, d);
  }

 private:
  static long floor_div(long a, long b) { return a / b - (a % b != 0 && a < 0); }
  bool search(size_t i, long d) {
    if (d < lo_[i] || d > hi_[i] || (div_[i] ? d % div_[i] != 0 : d != 0)) return false;
    if (i == t_.size() || --budget_ < 0) return true;
    const OverlapTerm& t = t_[i];
    const long first = std::max(t.lo, -floor_div(hi_[i + 1] - d, t.c)), last = std::min(t.hi, floor_div(d - lo_[i + 1], t.c));
    for (long x = first; x <= last; ++x)
      if (search(i + 1, d - t.c * x)) return true;
    return false;
  }
  OverlapTerms t_;
  c10::SmallVector<long, 14> lo_, hi_, div_;  // of the terms from i on: least and greatest sum, common divisor
  long budget_ = 0;
};

inline bool views_overlap(const MemView& a, const MemView& b) {
  OverlapTerms t;
  for (size_t k = 0; k < a.size.size(); ++k)
    if (a.size[k] > 1 && a.stride[k]) t.push_back({a.stride[k], 0, a.size[k] - 1});
  for (size_t k = 0; k < b.size.size(); ++k)
    if (b.size[k] > 1 && b.stride[k]) t.push_back({b.stride[k], 1 - b.size[k], 0});
  t.push_back({1, 1 - b.elem, a.elem - 1});
  return BoundedSum(std::move(t)).reaches((long)(b.base - a.base));
}

inline bool view_overlaps_itself(const MemView& a) {
  c10::SmallVector<std::pair<long, long>, 6> d;  // stride, size
  for (size_t k = 0; k < a.size.size(); ++k)
    if (a.size[k] > 1) d.push_back({a.stride[k], a.size[k]});
  std::sort(d.begin(), d.end());
  long reach = a.elem;
  bool apart = true;  // each stride passes the reach of the smaller ones
  for (const auto& [s, n] : d) {
    apart = apart && s >= reach;
    reach += s * (n - 1);
  }
  if (apart) return false;
  // two index vectors of one address: they differ first in dimension k, by x >= 1
  for (size_t k = 0; k < d.size(); ++k) {
    if (d[k].first == 0) return true;
    OverlapTerms t{{d[k].first, 1, d[k].second - 1}, {1, 1 - a.elem, a.elem - 1}};
    for (size_t j = k + 1; j < d.size(); ++j) t.push_back({d[j].first, 1 - d[j].second, d[j].second - 1});
    if (BoundedSum(std::move(t)).reaches(0)) return true;
  }
  return false;
}

}  // namespace dtb
