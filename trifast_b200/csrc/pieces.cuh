// Parts of 16-byte pieces: what lies at the edges of rows that do not begin at one.
#pragma once

#include <cstdint>

namespace trifast {

// The last n entries of a piece (`from`) or the first n, n less than all, in halves, quarters and eighths.
template <typename T>
__device__ __forceinline__ void store_part(T* to, const uint4& v, bool from, int n) {
  constexpr int VEC = 16 / sizeof(T), h = VEC / 2, q = VEC / 4;
  if (n & h) *reinterpret_cast<uint2*>(to + (from ? h : 0)) = from ? make_uint2(v.z, v.w) : make_uint2(v.x, v.y);
  const bool upper = ((n & h) != 0) != from;   // the half that the rest lies in
  if (n & q) {
    const uint32_t lo = upper ? v.z : v.x, hi = upper ? v.w : v.y;
    *reinterpret_cast<uint32_t*>(to + (upper ? h : 0) + (from ? q : 0)) = from ? hi : lo;
  }
  if constexpr (VEC == 8) {
    if (n & 1) {
      const int at = from ? VEC - n : n - 1, word = at >> 1;
      const uint32_t w = word & 2 ? (word & 1 ? v.w : v.z) : (word & 1 ? v.y : v.x);
      reinterpret_cast<unsigned short*>(to)[at] = (unsigned short)(at & 1 ? w >> 16 : w);
    }
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
