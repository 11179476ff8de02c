// Which memory the tensors of a call lie in (host code).
#pragma once

#include <algorithm>
#include <cstdint>

namespace magma {

// An address that is none of an element's would fault in a kernel.
inline bool on_element(const void* p, size_t size) {
  return reinterpret_cast<uintptr_t>(p) % size == 0;
}

// Positions [n0, n1, n2] of `bytes` contiguous bytes each, `step` bytes apart
// along each dimension (not negative).
struct MemView {
  const void* at = nullptr;  // NULL: no tensor
  int64_t bytes = 0;
  int64_t n[3] = {1, 1, 1};
  int64_t step[3] = {0, 0, 0};
};

namespace memory_views {

using wide = __int128;  // strides of 2^40 elements times 2^31 positions

inline wide end_of(const MemView& v) {
  wide e = (wide) reinterpret_cast<uintptr_t>(v.at) + v.bytes;
  for (int i = 0; i < 3; ++i) e += v.n[i] > 0 ? (wide)v.step[i] * (v.n[i] - 1) : 0;
  return e;
}

struct Term {
  wide step, lo, hi;  // step * c for lo <= c <= hi
};
// Whether d + sum of one value of each term lies in (-below, above), found by
// going through the terms from the largest step down and leaving out what the
// smaller ones cannot make good. `left` bounds the tries: nested strides, as
// views of one tensor have, need a few; where it runs out nothing is proven.
struct Search {
  Term t[6];
  wide rest_lo[7], rest_hi[7];
  int count = 0;
  wide below, above;
  int left = 4096;

  bool reach(int k, wide d) {
    if (d + rest_lo[k] >= above || d + rest_hi[k] <= -below || left-- <= 0) return false;
    if (k == count) return true;
    const Term& x = t[k];
    // d + c step + rest > -below and < above for some value of the rest
    wide c0 = floor_div(-below - rest_hi[k + 1] - d, x.step) + 1;
    wide c1 = -(floor_div(-(above - rest_lo[k + 1] - d), x.step) + 1);
    c0 = std::max(c0, x.lo);
    c1 = std::min(c1, x.hi);
    for (wide c = c0; c <= c1 && left > 0; ++c)
      if (reach(k + 1, d + c * x.step)) return true;
    return false;
  }
  static wide floor_div(wide a, wide b) { return a >= 0 ? a / b : -((-a + b - 1) / b); }
};

}  // namespace memory_views

// Whether some position of x and some position of y share a byte. Views that lie
// between one another, as those of fused projections do, share none.
inline bool share_memory(const MemView& x, const MemView& y) {
  using namespace memory_views;
  if (x.at == nullptr || y.at == nullptr || x.bytes <= 0 || y.bytes <= 0) return false;
  if (end_of(x) <= (wide) reinterpret_cast<uintptr_t>(y.at) ||
      end_of(y) <= (wide) reinterpret_cast<uintptr_t>(x.at))
    return false;
  Search s;
  s.above = x.bytes;  // y begins less than x.bytes behind x,
  s.below = y.bytes;  // and x less than y.bytes behind y
  for (int i = 0; i < 6; ++i) {
    const MemView& v = i < 3 ? x : y;
    const int64_t n = v.n[i % 3];
    const wide step = v.step[i % 3];
    if (n <= 0) return false;
    if (n == 1 || step == 0) continue;
    const wide lo = i < 3 ? -(wide)(n - 1) : 0, hi = i < 3 ? 0 : (wide)(n - 1);
    Term* same = std::find_if(s.t, s.t + s.count, [&](const Term& t) { return t.step == step; });
    if (same == s.t + s.count) s.t[s.count++] = Term{step, lo, hi};
    else same->lo += lo, same->hi += hi;
  }
  std::sort(s.t, s.t + s.count, [](const Term& a, const Term& b) { return a.step > b.step; });
  s.rest_lo[s.count] = s.rest_hi[s.count] = 0;
  for (int k = s.count; k-- > 0;) {
    s.rest_lo[k] = s.rest_lo[k + 1] + s.t[k].step * s.t[k].lo;
    s.rest_hi[k] = s.rest_hi[k + 1] + s.t[k].step * s.t[k].hi;
  }
  return s.reach(0, (wide) reinterpret_cast<uintptr_t>(y.at) - (wide) reinterpret_cast<uintptr_t>(x.at));
}

}  // namespace magma
