// How a paged-attention launch splits its work over CTAs: host/device
// arithmetic only, so that the CPU tests run the same code.
//
// A work item is one query row and one group of up to 8 query heads that
// share a KV head. Its keys are cut into units of `unit` tokens (an item has
// at least one, so that a row without keys is still written). The units of
// all items in order -- row by row, within a row item by item -- are dealt
// out evenly: CTA c of G takes units [U c / G, U (c + 1) / G). A CTA's range
// is a run of pieces, one for each item it touches; an item whole inside one
// CTA is written at once, one that spans several CTAs is joined from their
// partial results.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define PS_HD __host__ __device__ __forceinline__
#else
#define PS_HD inline
#endif

// n / d for 0 <= n < 2^31 by one multiplication: with l = ceil(log2 d) and
// m = floor(2^(31+l) / d) + 1 < 2^32 + 1, n m / 2^(31+l) exceeds n / d by less
// than n / 2^(31+l) < 1 / d (d = 1: the number itself).
struct PsDiv {
  uint32_t mul;
  int shift;  // -1: d = 1
};
inline PsDiv ps_div_of(int d) {
  PsDiv r{0, -1};
  if (d == 1) return r;
  int l = 0;
  while ((1ll << l) < d) ++l;
  r.mul = (uint32_t)(((1ull << (31 + l)) / (unsigned)d) + 1);
  r.shift = l - 1;
  return r;
}
PS_HD int ps_div(int n, PsDiv d) {
  if (d.shift < 0) return n;
#ifdef __CUDA_ARCH__
  return (int)(__umulhi((uint32_t)n, d.mul) >> d.shift);
#else
  return (int)(((uint64_t)(uint32_t)n * d.mul) >> 32 >> d.shift);
#endif
}

// Keys of a row: [low, len).
struct PsRow {
  int low, len;
};

// len clamped to [0, capacity]; a window keeps the last `window` keys (0: all).
PS_HD PsRow ps_row(int len, long long capacity, int window) {
  PsRow r;
  r.len = len < 0 ? 0 : (long long)len > capacity ? (int)capacity : len;
  r.low = window > 0 && r.len > window ? r.len - window : 0;
  return r;
}

// Units of one item of a row.
PS_HD int ps_units(PsRow r, int unit) {
  const int n = r.len - r.low;
  return n <= unit ? 1 : (int)(((long long)n + unit - 1) / unit);
}

// floor(U c / G) without the wide product (32-bit divisions where U allows).
PS_HD long long ps_begin(long long U, int c, int G) {
  if (U <= 0x7fffffff) {
    const uint32_t q = (uint32_t)U / (uint32_t)G, r = (uint32_t)U - q * (uint32_t)G;  // r c < 2^20
    return (long long)q * c + r * (uint32_t)c / (uint32_t)G;
  }
  return U / G * c + U % G * c / G;
}

// The CTA whose range holds unit u (0 <= u < U, G <= U).
PS_HD int ps_owner(long long u, long long U, int G) {
  const long long c = ((u + 1) * G - 1) / U;
  return c < 0 ? 0 : c < G ? (int)c : G - 1;
}

// Walks the pieces of one CTA: the item, its units in this CTA, and how many
// units of the range are left from the piece's first one on.
struct PsCursor {
  int row, item;    // query row, item within the row
  int n;            // units of each of the row's items
  int unit, units;  // first unit of the piece within the item, unit count
  long long left;
};

// The piece that starts `in_row` units after the start of row `row` (n units
// an item), with `left` units of the range to go.
PS_HD PsCursor ps_first(int row, long long in_row, int n, int items, long long left) {
  PsCursor c;
  c.row = row;
  c.n = n;
  const long long item =
      in_row <= 0x7fffffff ? (long long)((uint32_t)in_row / (uint32_t)n) : in_row / n;
  c.item = item < items ? (int)item : items - 1;
  c.unit = item < items ? (int)(in_row - item * n) : n - 1;
  c.left = left;
  c.units = left < n - c.unit ? (int)left : n - c.unit;
  return c;
}

// Steps to the next piece; false at the range's end, and after the last of
// `rows` rows whatever the units say (lengths that another stream changes
// meanwhile give wrong results, but no index out of range). A row is done
// after `items` items; units_of(row) gives the next row's n.
template <typename F>
PS_HD bool ps_next(PsCursor& c, int items, int rows, F&& units_of) {
  c.left -= c.units;
  if (c.left <= 0) return false;
  c.unit = 0;
  if (++c.item == items) {
    c.item = 0;
    if (++c.row >= rows) return false;
    c.n = units_of(c.row);
  }
  c.units = c.left < c.n ? (int)c.left : c.n;
  return true;
}
