// Which tensors of a call share memory: checks of what is written.
#pragma once
#include <ATen/ATen.h>

#include <algorithm>
#include <cstdint>
#include <utility>
#include <vector>

namespace dlvk {
namespace aten {

// Byte range of one tensor.  Column slices of one matrix have ranges that
// interleave without sharing an element: `row` bytes of every `pitch` bytes.
struct Extent {
  uintptr_t lo, hi;
  int64_t row, pitch;  // pitch 0: one dense run
  int64_t index;
};

inline Extent extent_of(const at::Tensor& t, int64_t index) {
  const int64_t es = t.element_size();
  Extent e{reinterpret_cast<uintptr_t>(t.data_ptr()), 0, 0, 0, index};
  if (t.is_contiguous()) {
    e.hi = e.lo + (uintptr_t)(t.numel() * es);
    return e;
  }
  int64_t span = 1, run = 1;
  bool rows = false, regular = true;
  // dimensions from the innermost stride outwards
  std::vector<std::pair<int64_t, int64_t>> dims;  // stride, size
  for (int64_t d = 0; d < t.dim(); ++d)
    if (t.size(d) > 1) dims.emplace_back(t.stride(d), t.size(d));
  std::sort(dims.begin(), dims.end());
  for (const auto& [st, sz] : dims) {
    span += st * (sz - 1);
    if (!rows && st == run) {
      run *= sz;
    } else if (!rows) {
      rows = true;
      e.row = run * es;
      e.pitch = st * es;
      run = st * sz;  // the next dimension continues the rows when its stride is this
    } else {
      regular = regular && st == run;
      run = st * sz;
    }
  }
  e.hi = e.lo + (uintptr_t)(span * es);
  if (!rows || !regular) e.row = e.pitch = 0;
  return e;
}

inline bool share_bytes(const Extent& a, const Extent& b) {
  if (a.hi <= b.lo || b.hi <= a.lo) return false;
  if (a.pitch == 0 || a.pitch != b.pitch) return true;
  const Extent &f = a.lo <= b.lo ? a : b, &l = a.lo <= b.lo ? b : a;
  const int64_t p = a.pitch, d = (int64_t)((l.lo - f.lo) % (uintptr_t)p);
  return d < f.row || d + l.row > p;
}

// Whether two indexes may name one element: each stride has to pass all that
// the smaller ones span.
inline bool may_repeat(const at::Tensor& t) {
  std::vector<std::pair<int64_t, int64_t>> dims;  // stride, size
  for (int64_t d = 0; d < t.dim(); ++d)
    if (t.size(d) > 1) dims.emplace_back(t.stride(d), t.size(d));
  std::sort(dims.begin(), dims.end());
  int64_t span = 1;
  for (const auto& [st, sz] : dims) {
    if (st < span) return true;
    span += st * (sz - 1);
  }
  return false;
}

}  // namespace aten
}  // namespace dlvk
