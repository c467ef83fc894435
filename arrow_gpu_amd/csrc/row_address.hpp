// row_address.hpp — which slot of a cache a row lies in: a slot column, or the page tables of ragged sequences (agpu_page_map).  Plain C++, so
// that a host program can check it against tables of any kind, broken ones too.
#pragma once
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
