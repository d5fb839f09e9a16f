// Which elements the strided row buffers of a call share. Host only, no CUDA, so that
// it is tested without a GPU.
#ifndef FMD_VIEWS_H
#define FMD_VIEWS_H

#include <cstdint>

namespace fmd {

// n_rows rows of n_heads heads of `dim` elements of 2 bytes from address `at`; strides in
// elements, >= 0.
struct HeadRows {
  uint64_t at;
  int64_t row, head;
  int64_t n_rows, n_heads, dim;

  __int128 span() const {  // elements from the first to behind the last
    return (__int128)(n_rows - 1) * row + (__int128)(n_heads - 1) * head + dim;
  }
  // Whether two of its heads share an element.
  bool overlaps() const {
    if ((n_rows > 1 && row < dim) || (n_heads > 1 && head < dim)) return true;
    if (n_rows <= 1 || n_heads <= 1) return false;
    if (row >= (__int128)(n_heads - 1) * head + dim || head >= (__int128)(n_rows - 1) * row + dim) return false;
    // neither axis lies within a step of the other: heads j apart against the rows nearest to that
    for (int64_t j = 1; j < n_heads; ++j) {
      const __int128 x = (__int128)j * head, k = x / row;
      if (k < n_rows && x - k * row < dim) return true;
      if (k + 1 < n_rows && (k + 1) * row - x < dim) return true;
    }
    return false;
  }
};

// Whether views a and b share an element. Exact where their rows have the same stride, as views
// of one buffer do; otherwise address ranges that meet count as shared.
inline bool meet(const HeadRows& a, const HeadRows& b) {
  const __int128 gap = ((__int128)b.at - (__int128)a.at) / 2;  // elements; views are 16-byte aligned
  if (gap >= a.span() || -gap >= b.span()) return false;
  const int64_t row = a.n_rows > 1 || b.n_rows > 1 ? a.row : 0;
  if ((a.n_rows > 1 || b.n_rows > 1) && a.row != b.row) return true;
  if (a.dim != b.dim) return true;
  // side by side in every row: of the heads of one fused row, for instance
  const __int128 ea = (__int128)(a.n_heads - 1) * a.head + a.dim, eb = (__int128)(b.n_heads - 1) * b.head + b.dim;
  if (row > 0 && ea <= row) {
    const __int128 d = gap >= 0 ? gap % row : (row - -gap % row) % row;
    if (d >= ea && d + eb <= row) return false;
  }
  auto near = [&](__int128 x) {  // whether heads x apart in some two rows overlap
    if (row == 0) return x < a.dim && -x < a.dim;
    const __int128 lo = -(b.n_rows - 1), hi = a.n_rows - 1;  // row of a less row of b
    __int128 k = x / row;
    for (int s = -1; s <= 1; ++s) {
      const __int128 kk = k + s < lo ? lo : k + s > hi ? hi : k + s, y = x - kk * row;
      if (y < a.dim && -y < a.dim) return true;
    }
    return false;
  };
  if (a.head == b.head) {
    for (int64_t j = -(a.n_heads - 1); j < b.n_heads; ++j)
      if (near(gap + (__int128)j * a.head)) return true;
    return false;
  }
  if (a.n_heads * b.n_heads > (1 << 20)) return true;
  for (int64_t i = 0; i < a.n_heads; ++i)
    for (int64_t j = 0; j < b.n_heads; ++j)
      if (near(gap + (__int128)j * b.head - (__int128)i * a.head)) return true;
  return false;
}

}  // namespace fmd

#endif  // FMD_VIEWS_H
