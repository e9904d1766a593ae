// Host-side checks of what the paged cache operators and the draft
// verification write: a view must not reach an element twice, and must share
// none with another one.  Everything in bytes, 128-bit where strides multiply.
#pragma once

#include <algorithm>
#include <cstdint>

namespace persona {
namespace overlap {

using wide = __int128;

// A strided view: up to three dimensions over a run of `inner` bytes, and the
// addresses from its first byte to behind its last one (0, 0: no element).
struct View {
  uint64_t lo, hi;
  int64_t inner, size[3], stride[3];
  View(const void* p, int64_t run, const int64_t (&n)[3], const int64_t (&step)[3])
      : lo(reinterpret_cast<uintptr_t>(p)), inner(run), size{n[0], n[1], n[2]}, stride{step[0], step[1], step[2]} {
    wide end = static_cast<wide>(lo) + inner;
    for (int i = 0; i < 3; ++i) end += static_cast<wide>(size[i] - 1) * stride[i];
    hi = end > static_cast<wide>(UINT64_MAX) ? UINT64_MAX : static_cast<uint64_t>(end);
    if (inner <= 0 || size[0] <= 0 || size[1] <= 0 || size[2] <= 0) lo = hi = 0;
  }
};

// Whether the address ranges meet (also where the elements do not).
inline bool ranges_meet(const View& a, const View& b) { return a.lo < b.hi && b.lo < a.hi; }

// The dimensions along which a or b takes a step, largest stride first, with
// each one's size.  False where both take steps of different length in one.
struct Dims {
  int n = 0;
  int64_t a[3], b[3], stride[3];
};
inline bool merge(const View& a, const View& b, Dims& d) {
  for (int i = 0; i < 3; ++i) {
    if (a.size[i] <= 1 && b.size[i] <= 1) continue;
    if (a.size[i] > 1 && b.size[i] > 1 && a.stride[i] != b.stride[i]) return false;
    const int64_t s = a.size[i] > 1 ? a.stride[i] : b.stride[i];
    int k = d.n++;
    for (; k > 0 && d.stride[k - 1] < s; --k) {
      d.a[k] = d.a[k - 1];
      d.b[k] = d.b[k - 1];
      d.stride[k] = d.stride[k - 1];
    }
    d.a[k] = a.size[i];
    d.b[k] = b.size[i];
    d.stride[k] = s;
  }
  return true;
}
// Whether every dimension steps past all that the smaller ones span.
inline bool nested(const Dims& d, int64_t inner) {
  wide span = inner;
  for (int i = d.n - 1; i >= 0; --i) {
    if (d.stride[i] < span) return false;
    span += static_cast<wide>(std::max(d.a[i], d.b[i]) - 1) * d.stride[i];
  }
  return true;
}

// Whether no element of the view is reached twice.  (Views whose dimensions
// are interleaved without meeting, which no slicing or transposing makes, are
// taken for ones that do.)
inline bool nested(const View& v) {
  Dims d;
  return merge(v, v, d) && nested(d, v.inner);
}

// Whether two views share a byte.  Exact where they step alike, as slices of
// one buffer do: at each dimension only the two multiples of its stride around
// the distance leave less than a stride, which the smaller dimensions have to
// cover.  Elsewhere, whether their ranges meet.
inline bool share(const View& a, const View& b) {
  if (!ranges_meet(a, b)) return false;
  Dims dims;
  if (!merge(a, b, dims) || !nested(dims, std::max(a.inner, b.inner))) return true;
  const auto reach = [&](auto& self, wide d, int i) -> bool {  // d: from a's element to b's
    if (i == dims.n) return d < a.inner && -d < b.inner;
    wide k = d / dims.stride[i];
    if (d < 0 && k * dims.stride[i] != d) --k;  // round down
    for (int x = 0; x < 2; ++x, ++k)
      if (k < dims.a[i] && -k < dims.b[i] && self(self, d - k * dims.stride[i], i + 1)) return true;
    return false;
  };
  return reach(reach, static_cast<wide>(b.lo) - static_cast<wide>(a.lo), 0);
}

}  // namespace overlap
}  // namespace persona
