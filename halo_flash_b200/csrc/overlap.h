// Whether two strided views share memory, and whether a view's own rows do: host checks of the arguments of calls whose
// CTAs write in no order, where shared memory would make the result depend on chance.
//
// A view is a run of bytes repeated along up to three axes. The answer is exact. Two views of one buffer (q, k and v of a
// projection, K and V beside each other in a page) have the same strides, where only the difference of two indices counts
// and a handful of them brings the runs near each other: nanoseconds. Views whose strides differ and whose spans cross are
// walked along the larger stride; the walk is cut off at kOverlapSteps and then counts as "no": nothing that a program
// lays out on purpose comes near that.
#ifndef HALO_B200_OVERLAP_H_
#define HALO_B200_OVERLAP_H_

#include <cstdint>
#include <utility>

namespace halo_b200 {

constexpr unsigned kOverlapSteps = 1u << 16;

struct View {
  using Int = __int128;  // strides and counts that no memory has must not wrap
  struct Axis {
    Int stride, n;
  };
  Int base = 0, run = 0;  // in bytes
  Axis axis[3];           // ascending strides
  int axes = 0;
  bool repeats = false;   // an axis of stride 0 with several entries

  View(const void* p, uint64_t run_bytes) : base(static_cast<Int>(reinterpret_cast<uintptr_t>(p))), run(run_bytes) {}
  // n entries, `stride` elements of `size` bytes apart.
  View& Along(uint64_t n, uint64_t stride, uint64_t size) {
    if (n == 0) run = 0;
    if (n <= 1) return *this;
    if (stride == 0) {
      repeats = true;
      return *this;
    }
    int i = axes++;
    axis[i] = {static_cast<Int>(stride) * size, static_cast<Int>(n)};
    for (; i > 0 && axis[i].stride < axis[i - 1].stride; --i) std::swap(axis[i], axis[i - 1]);
    return *this;
  }
  Int Span() const {
    Int s = run;
    for (int i = 0; i < axes; ++i) s += axis[i].stride * (axis[i].n - 1);
    return s;
  }
  const Axis& Top() const { return axis[axes - 1]; }
  View Without(Int shift) const {  // one entry of the outermost axis, moved
    View v = *this;
    --v.axes;
    v.base += shift;
    return v;
  }
};

namespace overlap_detail {

inline View::Int FloorDiv(View::Int a, View::Int b) { return a >= 0 ? a / b : -((-a + b - 1) / b); }

// The indices i in [lo, hi] at which `v`, moved by i * stride, meets `other`: those with both
// v.base + i stride < other's end and other.base < v's end + i stride.
inline void Near(const View& v, const View& other, View::Int stride, View::Int* lo, View::Int* hi) {
  const View::Int first = FloorDiv(other.base - v.base - v.Span(), stride) + 1;
  const View::Int last = FloorDiv(other.base + other.Span() - v.base - 1, stride);
  if (first > *lo) *lo = first;
  if (last < *hi) *hi = last;
}

inline bool Meet(const View& a, const View& b, unsigned* steps) {
  if (*steps == 0) return false;
  --*steps;
  if (a.base + a.Span() <= b.base || b.base + b.Span() <= a.base) return false;
  if (a.axes == 0 && b.axes == 0) return true;
  if (a.axes > 0 && b.axes > 0 && a.Top().stride == b.Top().stride) {
    const View one = a.Without(0), two = b.Without(0);
    View::Int lo = -(a.Top().n - 1), hi = b.Top().n - 1;  // of b's index less a's
    Near(two, one, a.Top().stride, &lo, &hi);
    for (View::Int i = lo; i <= hi && *steps; ++i)
      if (Meet(one, b.Without(i * a.Top().stride), steps)) return true;
    return false;
  }
  if (a.axes == 0 || (b.axes > 0 && b.Top().stride > a.Top().stride)) return Meet(b, a, steps);
  View::Int lo = 0, hi = a.Top().n - 1;
  Near(a.Without(0), b, a.Top().stride, &lo, &hi);
  for (View::Int i = lo; i <= hi && *steps; ++i)
    if (Meet(a.Without(i * a.Top().stride), b, steps)) return true;
  return false;
}

inline bool MeetsItself(const View& v, unsigned* steps) {
  if (v.axes == 0) return false;
  const View one = v.Without(0);
  const View::Int s = v.Top().stride;
  for (View::Int i = 1; i < v.Top().n && i * s < one.Span() && *steps; ++i)
    if (Meet(one, v.Without(i * s), steps)) return true;
  return MeetsItself(one, steps);
}

}  // namespace overlap_detail

// Two views that share a byte.
inline bool Overlap(const View& a, const View& b) {
  unsigned steps = kOverlapSteps;
  return a.run > 0 && b.run > 0 && overlap_detail::Meet(a, b, &steps);
}
// A view of which two entries share a byte.
inline bool OverlapsItself(const View& v) {
  unsigned steps = kOverlapSteps;
  return v.run > 0 && (v.repeats || overlap_detail::MeetsItself(v, &steps));
}

}  // namespace halo_b200

#endif  // HALO_B200_OVERLAP_H_
