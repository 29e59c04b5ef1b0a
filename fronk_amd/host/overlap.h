// overlap.h - whether two strided arrays, or two elements of one, share memory, exactly, in
// plain C++ so that it is tested on the host.
//
// An array's bytes are its address, plus multiples of its strides, plus 0 .. size - 1 of an
// element. Two share one where their addresses' difference d and some multiples t, within
// bounds, of all strides s of both give d + sum s t within one element's reach. Axes that
// continue each other are one run of bytes first; axes of one stride are one t. Then the
// largest stride's t is tried first, and of each only what the others can still bring within
// reach: where strides are nested, as those of rows and heads are, two values at most.
#pragma once
#include <stddef.h>
#include <stdint.h>

#include <algorithm>

namespace fronk {

constexpr int kAxes = 8;   // of an array, at most

// An array's elements; sizes and strides in elements, strides 0 or more, none empty.
struct Strided {
  uintptr_t at;
  int64_t element, axes;
  const int64_t *sizes, *strides;
};
// Its bytes, with what is between them.
inline uintptr_t reach(const Strided& a) {
  uintptr_t n = a.element;
  for (int64_t i = 0; i < a.axes; ++i) n += (a.sizes[i] - 1) * a.strides[i] * a.element;
  return n;
}

struct Axis {
  int64_t stride, low, high;   // bytes; bounds of its multiple
};
struct Axes {
  Axis axis[2 * kAxes];
  int n = 0;
};

// An array's axes, times `sign`, but for those that continue each other: these are one run, whose bytes are returned.
inline int64_t runs(const Strided& a, int sign, Axes* out) {
  Axes all;
  for (int64_t i = 0; i < a.axes; ++i)
    if (a.sizes[i] > 1 && a.strides[i]) all.axis[all.n++] = {a.strides[i] * a.element, 0, a.sizes[i] - 1};
  std::sort(all.axis, all.axis + all.n, [](const Axis& x, const Axis& y) { return x.stride < y.stride; });
  int64_t run = a.element;
  for (int i = 0; i < all.n; ++i) {
    const Axis x = all.axis[i];
    if (x.stride == run) run *= x.high + 1;
    else out->axis[out->n++] = {x.stride, sign < 0 ? -x.high : 0, sign < 0 ? 0 : x.high};
  }
  return run;
}

// Whether some multiples of axes i and on bring d to within low .. high; not all 0, unless `moved`. `left`
// steps are taken at most; without an answer by then it is yes.
inline bool reaches(const Axes& a, int i, int64_t d, int64_t low, int64_t high, bool moved, int64_t* left) {
  if (i == a.n) return moved && d >= low && d <= high;
  int64_t least = 0, most = 0;   // what the axes behind this one can add
  for (int k = i + 1; k < a.n; ++k) least += a.axis[k].stride * a.axis[k].low, most += a.axis[k].stride * a.axis[k].high;
  auto floor_div = [](int64_t x, int64_t y) { return x / y - (x % y < 0); };
  const int64_t s = a.axis[i].stride;
  const int64_t first = std::max(a.axis[i].low, -floor_div(d + most - low, s)), last = std::min(a.axis[i].high, floor_div(high - least - d, s));
  for (int64_t t = first; t <= last; ++t)
    if (--*left < 0 || reaches(a, i + 1, d + s * t, low, high, moved || t, left)) return true;
  return false;
}

inline bool share(const Strided& a, const Strided& b) {
  if (a.axes > kAxes || b.axes > kAxes) return true;
  if (a.at + reach(a) <= b.at || b.at + reach(b) <= a.at) return false;
  Axes axes;
  const int64_t run_a = runs(a, -1, &axes), run_b = runs(b, 1, &axes);
  std::sort(axes.axis, axes.axis + axes.n, [](const Axis& x, const Axis& y) { return x.stride > y.stride; });
  int n = 0;
  for (int i = 0; i < axes.n; ++i) {
    const Axis x = axes.axis[i];
    if (n && axes.axis[n - 1].stride == x.stride) axes.axis[n - 1].low += x.low, axes.axis[n - 1].high += x.high;
    else axes.axis[n++] = x;
  }
  axes.n = n;
  int64_t left = 1 << 20;
  return reaches(axes, 0, (int64_t)(b.at - a.at), 1 - run_b, run_a - 1, true, &left);
}

// Whether two of an array's elements share memory.
inline bool shares(const Strided& a) {
  if (a.axes > kAxes) return true;
  for (int64_t i = 0; i < a.axes; ++i)
    if (a.sizes[i] > 1 && !a.strides[i]) return true;
  Axes axes;
  const int64_t run = runs(a, 1, &axes);
  std::sort(axes.axis, axes.axis + axes.n, [](const Axis& x, const Axis& y) { return x.stride > y.stride; });
  for (int i = 0; i < axes.n; ++i) axes.axis[i].low = -axes.axis[i].high;
  int64_t left = 1 << 20;
  return reaches(axes, 0, 0, 1 - run, run - 1, false, &left);
}

}  // namespace fronk
