// row_address.hpp — which slot of a cache a row lies in: a slot column, or the page tables of ragged sequences (agpu_page_map); and whether what a call
// writes lies apart from what else it touches.  Plain C++, so that a host program can check it against tables and strides of any kind, broken ones too.
#pragma once
#include <algorithm>

#include "../../include/arrow_gpu.h"

#ifdef __HIPCC__
#define AGPU_ROW_FN __host__ __device__ __forceinline__
#else
#define AGPU_ROW_FN inline
#endif

// x / d by a product, x < 2^31: m = ⌈2^(31 + s) / d⌉ is off by less than d <= 2^s in 2^(31 + s), so the quotient by less than 1 / d
struct Divide {
  uint32_t d, m, s;
};
AGPU_ROW_FN uint32_t operator/(uint32_t x, Divide d) { return (uint32_t)((uint64_t)(x << 1) * d.m >> 32) >> d.s; }
inline Divide divide_by(uint32_t d) {
  uint32_t s = 0;
  while ((1ull << s) < d) s++;
  return {d, (uint32_t)(((1ull << (31 + s)) + d - 1) / d), s};
}

// whether n rows of m parts of `part` values each, rows and parts so far apart, lie beside each other: one of the two encloses the other
inline bool disjoint(uint64_t n, uint64_t row_stride, uint64_t m, uint64_t part_stride, uint64_t part) {
  const auto within = [&](uint64_t count, uint64_t step, uint64_t size, uint64_t outer) {  // (count − 1) · step + size <= outer, step >= size
    uint64_t span;
    if (count <= 1) return size <= outer;
    return step >= size && !__builtin_mul_overflow(count - 1, step, &span) && !__builtin_add_overflow(span, size, &span) && span <= outer;
  };
  if (n <= 1) return within(m, part_stride, part, ~0ull);
  if (m <= 1) return row_stride >= part;
  return within(m, part_stride, part, row_stride) || within(n, row_stride, part, part_stride);
}

// Memory that a call reads or writes, in bytes: n rows of m parts of `size` bytes.  Parts of one owner are not compared with each other
struct Places {
  uint64_t at, n, row_stride, m, part_stride, size;
  bool written;
  int32_t owner;
};
// bytes from the first to behind the last of n rows; 0: none.  false: past 2^63
inline bool extent(uint64_t n, uint64_t row_stride, uint64_t m, uint64_t part_stride, uint64_t size, uint64_t* out) {
  uint64_t a, b;
  if (n == 0 || m == 0 || size == 0) {
    *out = 0;
    return true;
  }
  return !__builtin_mul_overflow(n - 1, row_stride, &a) && !__builtin_mul_overflow(m - 1, part_stride, &b) && !__builtin_add_overflow(a, b, &a) &&
         !__builtin_add_overflow(a, size, out) && *out < (1ull << 63);
}
// Whether two places whose ends overlap share no byte because they lie interleaved.  Strides that are multiples of `step` leave addresses modulo `step`
// alone; the other axes make a stretch there, and the stretches of the two are apart — or each lies in one window of `step` bytes, and inside it the two are
// apart in the same way, by a stride of the axes that are left (heads of two states in turn, rows padded)
inline bool stretches_apart(const Places& a, const Places& b, uint64_t step, Places* x, Places* y) {
  const auto in_window = [&](const Places& p, Places* w) {
    *w = p;
    w->at = p.at % step;
    if (p.row_stride % step == 0) w->n = 1;
    if (p.part_stride % step == 0) w->m = 1;
    uint64_t r = 0;
    extent(w->n, w->row_stride, w->m, w->part_stride, w->size, &r);
    return r;
  };
  const uint64_t ra = in_window(a, x), rb = in_window(b, y), d = y->at >= x->at ? y->at - x->at : y->at + step - x->at;
  if (ra <= d && rb <= step - d) return true;
  const bool from_a = ra <= step && rb <= step - d, from_b = rb <= step && ra <= d;  // the window begins where a does, where b does
  x->at = from_a ? 0 : step - d, y->at = from_a ? d : 0;
  if (!from_a && !from_b) x->n = 0;  // no window
  return false;
}
inline bool interleaved(const Places& a, const Places& b) {
  for (const uint64_t outer : {a.row_stride, a.part_stride, b.row_stride, b.part_stride}) {
    Places x, y, u, v;
    if (outer == 0) continue;
    if (stretches_apart(a, b, outer, &x, &y)) return true;
    if (x.n == 0) continue;
    for (const uint64_t inner : {x.row_stride, x.part_stride, y.row_stride, y.part_stride})
      if (inner != 0 && inner < outer && stretches_apart(x, y, inner, &u, &v)) return true;
  }
  return false;
}
// The first two of `count` places (all within 2^63 bytes, none empty; at least one of the two written) that may share a byte.  false: none.  Sorts them
inline bool overlapping(Places* p, uint32_t count, uint32_t* first, uint32_t* second) {
  std::sort(p, p + count, [](const Places& a, const Places& b) { return a.at < b.at; });
  for (uint32_t i = 0; i < count; i++) {
    uint64_t end = 0;
    extent(p[i].n, p[i].row_stride, p[i].m, p[i].part_stride, p[i].size, &end);
    for (uint32_t j = i + 1; j < count && p[j].at - p[i].at < end; j++) {
      const Places &a = p[i], &b = p[j];
      if ((!a.written && !b.written) || a.owner == b.owner) continue;
      if (interleaved(a, b)) continue;
      *first = i, *second = j;
      return true;
    }
  }
  return false;
}

constexpr uint64_t ROW_NONE = ~0ull;     // the row is neither stored nor written
constexpr uint64_t ROW_BAD = ~0ull - 1;  // out of range

struct RowAddr {
  const uint32_t* slots;  // one slot a row, or NULL: the page map
  const uint32_t* tables;
  uint64_t table_stride;
  const uint32_t* offsets;
  const uint32_t* first;
  uint32_t n_seqs, max_pages, page_rows;
};

AGPU_ROW_FN uint64_t row_slot(const RowAddr& a, uint64_t i, uint64_t n_slots) {
  if (a.slots) {
    const uint32_t s = a.slots[i];
    return s == AGPU_NO_ROW ? ROW_NONE : s < n_slots ? s : ROW_BAD;
  }
  // the last sequence that starts at or before i (an empty one starts where the next does and is passed over)
  uint32_t lo = 0, hi = a.n_seqs;  // offsets[lo] <= i < offsets[hi], once the ends are checked
  if (i < a.offsets[0] || i >= a.offsets[hi]) return ROW_NONE;
  while (hi - lo > 1) {
    const uint32_t mid = lo + (hi - lo) / 2;
    if (a.offsets[mid] <= i) lo = mid;
    else hi = mid;
  }
  const uint64_t t = (a.first ? a.first[lo] : 0u) + (i - a.offsets[lo]);  // offsets[lo] <= i, also where they are out of order
  const uint64_t page = t / a.page_rows;
  if (page >= a.max_pages) return ROW_BAD;
  const uint32_t e = a.tables[lo * a.table_stride + page];
  if (e == AGPU_NO_ROW) return ROW_NONE;
  const uint64_t s = (uint64_t)e * a.page_rows + t % a.page_rows;
  return s < n_slots ? s : ROW_BAD;
}
