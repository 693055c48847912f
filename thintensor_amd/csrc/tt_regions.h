// What a strided operand touches: the host's checks that no place is written twice, or read by one
// thread while another writes it.
#pragma once

#include <cstdint>
#include <initializer_list>
#include <utility>

namespace tt {

// Runs of `run` bytes along up to three axes.  Axes of one element are dropped, negative steps turned
// around, and the largest step comes first; an axis that stays in place (step 0) is noted and dropped.
struct Region {
  struct Axis {
    int64_t n;
    __int128 step;
  };
  __int128 start = 0, run = 0;
  Axis axes[3];
  int count = 0;
  bool empty = false, in_place = false;

  // `axes_of`: (elements, stride in elements), innermost last; the last one's runs are `length` elements.
  Region(const void* p, int64_t element, int64_t length, std::initializer_list<std::pair<int64_t, int64_t>> axes_of) {
    start = (__int128) reinterpret_cast<uintptr_t>(p);
    run = (__int128)element * length;
    empty = length <= 0;
    for (const auto& a : axes_of) {
      if (a.first <= 0) empty = true;
      if (a.first <= 1) continue;
      __int128 step = (__int128)a.second * element;
      if (step < 0) {
        start += (a.first - 1) * step;
        step = -step;
      }
      if (step == 0) {
        in_place = true;
        continue;
      }
      int at = count++;
      for (; at > 0 && axes[at - 1].step < step; at--) axes[at] = axes[at - 1];
      axes[at] = Axis{a.first, step};
    }
  }
  // from the first byte to past the last one, of the axes from `from` on
  __int128 extent(int from = 0) const {
    __int128 e = run;
    for (int i = from; i < count; i++) e += (axes[i].n - 1) * axes[i].step;
    return e;
  }
  // No byte comes twice: every step passes what the smaller ones reach.
  bool once() const {
    if (empty) return true;
    if (in_place) return false;
    for (int i = 0; i < count; i++)
      if (axes[i].step < extent(i + 1)) return false;
    return true;
  }
  bool same(const Region& o) const {
    if (start != o.start || run != o.run || count != o.count) return false;
    for (int i = 0; i < count; i++)
      if (axes[i].n != o.axes[i].n || axes[i].step != o.axes[i].step) return false;
    return true;
  }
};

// Whether two regions share no byte, with b's axes from j on `gap` bytes behind a's from i on.  Equal steps
// run side by side, so that only the distances of their indexes matter; of unequal ones the larger is
// walked.  What would take more than a few looks counts as shared.
inline bool apart(const Region& a, int i, const Region& b, int j, __int128 gap) {
  constexpr int kLooks = 8;
  const __int128 ea = a.extent(i), eb = b.extent(j);
  if (gap >= ea || gap + eb <= 0) return true;
  if (i == a.count && j == b.count) return false;
  const auto up = [](__int128 x, __int128 s) { return x >= 0 ? (x + s - 1) / s : -(-x / s); };   // ceil(x / s)
  const bool has_a = i < a.count, has_b = j < b.count;
  const bool walk_a = has_a && (!has_b || a.axes[i].step >= b.axes[j].step);
  const bool walk_b = has_b && (!has_a || b.axes[j].step >= a.axes[i].step);
  const __int128 step = walk_a ? a.axes[i].step : b.axes[j].step;
  const int ni = i + (walk_a ? 1 : 0), nj = j + (walk_b ? 1 : 0);
  // k = (index in b) - (index in a), where an axis that is not walked has index 0: the parts share bytes
  // only where -(b's extent) < gap + k step < (a's extent)
  const __int128 pa = a.extent(ni), pb = b.extent(nj);
  __int128 lo = up(1 - pb - gap, step), hi = up(pa - gap, step) - 1;
  const __int128 least = walk_a ? -(__int128)(a.axes[i].n - 1) : 0, most = walk_b ? b.axes[j].n - 1 : 0;
  if (lo < least) lo = least;
  if (hi > most) hi = most;
  if (hi - lo >= kLooks) return false;
  for (__int128 k = lo; k <= hi; k++)
    if (!apart(a, ni, b, nj, gap + k * step)) return false;
  return true;
}
inline bool apart(const Region& a, const Region& b) {
  return a.empty || b.empty || apart(a, 0, b, 0, b.start - a.start);
}

}  // namespace tt
