// Whether two arrays laid out in rows share memory: plain arithmetic on the host, before anything is queued.
#pragma once

#include <algorithm>
#include <cstdint>
#include <vector>

namespace tesm {

// n rows of `width` bytes, `pitch` bytes from row to row (at least the width where there is more than one).
struct RowSpan {
  const void* p = nullptr;
  int64_t n = 0, pitch = 0, width = 0;
};

// Column slices of the same wider rows interleave without sharing a byte, so ranges alone do not tell.
inline bool rows_share(RowSpan a, RowSpan b) {
  if (!a.p || !b.p || a.n <= 0 || b.n <= 0 || a.width <= 0 || b.width <= 0) return false;
  if (a.n > b.n) {
    const RowSpan t = a;
    a = b, b = t;
  }
  // from here on a has no more rows than b; addresses count from b's first byte
  const int64_t at = static_cast<int64_t>(reinterpret_cast<uintptr_t>(a.p)) - static_cast<int64_t>(reinterpret_cast<uintptr_t>(b.p));
  const int64_t a_end = at + (a.n - 1) * a.pitch + a.width, b_end = (b.n - 1) * b.pitch + b.width;
  if (a_end <= 0 || at >= b_end) return false;
  if (b.n == 1) return true;  // (and a.n == 1: two overlapping ranges)
  // Bytes [lo, lo + width) against b's rows: the last row that starts before the end, if it reaches past lo.
  auto hits = [&](int64_t lo) {
    const int64_t end = lo + a.width;
    if (end <= 0 || lo >= b_end) return false;
    const int64_t last = (end - 1) / b.pitch, row = last < b.n ? last : b.n - 1;
    return row * b.pitch + b.width > lo;
  };
  // Rows of one pitch all lie alike against b's where both reach: the first and the last row of a that b's range covers.
  if (a.pitch == b.pitch || a.n == 1) {
    const int64_t past = at < 0 ? (-at) / b.pitch : 0, first = past < a.n ? past : a.n - 1;
    int64_t last = (b_end - 1 - at) / b.pitch;
    if (last >= a.n) last = a.n - 1;
    return hits(at + first * a.pitch) || (first + 1 <= last && hits(at + (first + 1) * a.pitch)) || hits(at + last * a.pitch);
  }
  for (int64_t i = 0; i < a.n; ++i)
    if (hits(at + i * a.pitch)) return true;
  return false;
}

// Whether any two of the arrays share memory (sorted by address here).  Only arrays whose ranges meet are compared, and
// column slices of the same wider rows by their order inside a row.
inline bool any_rows_share(std::vector<RowSpan>& v) {
  auto at = [&](size_t i) { return reinterpret_cast<uintptr_t>(v[i].p); };
  auto end = [&](size_t i) { return at(i) + static_cast<uintptr_t>((v[i].n - 1) * v[i].pitch + v[i].width); };
  v.erase(std::remove_if(v.begin(), v.end(), [](const RowSpan& r) { return !r.p || r.n <= 0 || r.width <= 0; }), v.end());
  std::sort(v.begin(), v.end(), [](const RowSpan& a, const RowSpan& b) { return reinterpret_cast<uintptr_t>(a.p) < reinterpret_cast<uintptr_t>(b.p); });
  for (size_t i = 0, j; i < v.size(); i = j) {
    uintptr_t past = end(i);
    bool slices = true;  // one pitch, each behind the last, all inside one row
    for (j = i + 1; j < v.size() && at(j) < past; ++j) {
      slices = slices && v[j].pitch == v[i].pitch && at(j - 1) + static_cast<uintptr_t>(v[j - 1].width) <= at(j);
      past = std::max(past, end(j));
    }
    if (j == i + 1 || (slices && at(j - 1) + static_cast<uintptr_t>(v[j - 1].width) <= at(i) + static_cast<uintptr_t>(v[i].pitch))) continue;
    for (size_t a = i; a < j; ++a)
      for (size_t b = a + 1; b < j; ++b)
        if (rows_share(v[a], v[b])) return true;
  }
  return false;
}

}  // namespace tesm
