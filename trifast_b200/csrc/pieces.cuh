// Parts of 16-byte pieces: what lies at the edges of rows that do not begin at one.
#pragma once

#include <cstdint>

namespace trifast {

// Entries [lo, hi) of a piece, in halves, quarters and eighths where the rest is before them or behind them alone.
template <typename T>
__device__ __forceinline__ void store_part(T* to, const uint4& v, int lo, int hi) {
  constexpr int VEC = 16 / sizeof(T), h = VEC / 2, q = VEC / 4;
  static_assert(sizeof(T) == 2 || sizeof(T) == 4, "two or four bytes");
  auto entry = [&](int at) {
    const int word = VEC == 4 ? at : at >> 1;
    return word & 2 ? (word & 1 ? v.w : v.z) : (word & 1 ? v.y : v.x);
  };
  auto put = [&](int at) {
    if constexpr (VEC == 4)
      reinterpret_cast<uint32_t*>(to)[at] = entry(at);
    else
      reinterpret_cast<unsigned short*>(to)[at] = (unsigned short)(at & 1 ? entry(at) >> 16 : entry(at));
  };
  if (lo <= 0 && hi >= VEC) {
    *reinterpret_cast<uint4*>(to) = v;
  } else if (lo > 0 && hi < VEC) {
    for (int at = lo; at < hi; ++at) put(at);
  } else {
    const bool from = lo > 0;
    const int n = from ? VEC - lo : hi;
    if (n <= 0) return;
    if (n & h) *reinterpret_cast<uint2*>(to + (from ? h : 0)) = from ? make_uint2(v.z, v.w) : make_uint2(v.x, v.y);
    const bool upper = ((n & h) != 0) != from;   // the half that the rest lies in
    if (n & q) {
      const uint32_t a = upper ? v.z : v.x, b = upper ? v.w : v.y;
      *reinterpret_cast<uint32_t*>(to + (upper ? h : 0) + (from ? q : 0)) = from ? b : a;
    }
    if (VEC == 8 && (n & 1)) put(from ? lo : n - 1);
  }
}

// Classes of rows of `width` entries that begin at the same place of a piece of `vec`.
inline int row_classes(int64_t width, int vec) {
  int c = vec;
  while (c > 1 && width % 2 == 0) {
    width /= 2;
    c /= 2;
  }
  return c;
}

}  // namespace trifast
