// How a paged-attention launch splits its work over CTAs: host/device
// arithmetic only, so that the CPU tests run the same code.
//
// A work item is one query row and one group of up to 8 or 16 query heads that
// share a KV head. Its keys are cut into units of `unit` tokens (an item has
// at least one, so that a row without keys is still written). The units of
// all items in order -- row by row, within a row item by item -- are dealt
// out evenly: CTA c of G takes units [U c / G, U (c + 1) / G). A CTA's range
// is a run of pieces, one for each item it touches; an item whole inside one
// CTA is written at once, one that spans several CTAs is joined from their
// partial results. Where the items are alike enough, the unit is made so long
// that every CTA has one piece (ps_factor). Elsewhere the start of an item
// counts as units of its own that hold no keys (ps_cost), so that a CTA with
// many short pieces gets fewer keys. The host chooses the smallest unit so that
// there are fewer than 2^31 (ps_small_unit): the arithmetic is in 32 bits.
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
PS_HD PsRow ps_row(int len, int capacity, int window) {
  PsRow r;
  r.len = len < 0 ? 0 : len > capacity ? capacity : len;
  r.low = window > 0 && r.len > window ? r.len - window : 0;
  return r;
}

// Units of one item of a row (unit < 2^31).
PS_HD int ps_units(PsRow r, int unit) {
  const uint32_t n = (uint32_t)(r.len - r.low);
  return n <= (uint32_t)unit ? 1 : (int)((n + (uint32_t)unit - 1) / (uint32_t)unit);
}

// What the start of an item counts as, in units: a CTA with one piece was done
// with its keys 2.6 us before one with two, 16 to 32 KB of keys take 1.1 to 1.5
// (ps_cost). 32 rows of 17 to 6000 keys of 64: 42.7 us with 0, 41.1, 40.9, 41.1
// with 1, 2, 3; 60 rows up to 1500: 29.7, 27.0, 27.4, 28.1; 64 e4m3 rows of 17 to
// 8200 keys of 128: 117.1, 109.0, 107.8, 108.5.
constexpr int kPsCost = 2;

// The smallest unit, `unit` times a power of two, with which `items` items of
// up to `capacity` keys have fewer than 2^31 units with their starts; 0: none.
inline int ps_small_unit(int unit, long long items, int capacity) {
  for (long long u = unit; u < 0x40000000; u *= 2) {
    const long long n = ((long long)capacity + u - 1) / u;
    if (items <= 0x7fffffffll / ((n < 1 ? 1 : n) + kPsCost)) return (int)u;
  }
  return 0;
}

// How many small units make the unit. Let U small units, at most n_max in an
// item, `items` items and `slots` CTAs. With f = ceil(n_max / (slots / items))
// no item has more than slots / items units, so each CTA gets one unit at
// most: no CTA works at two items and fewer items are joined, but the longest
// CTA has f small units instead of U / slots. A second piece in a CTA and a
// join cost as much as two or three small units, so f is taken while it is at
// most 2 above the even share; and items of up to 3 small units stay whole.
// (32 rows of 300 keys, 8 KV heads: 14.4 us without, 8.3 us; 8 rows of 2048:
// 16.5 us, 14.1 us.)
PS_HD int ps_factor(int U, int n_max, int items, int slots) {
  if (items > slots) return 1;
  if (n_max <= 3) return n_max;
  const int p = slots / items;
  const int f = (int)((uint32_t)(n_max + p - 1) / (uint32_t)p);
  return (f - 2) * slots <= U ? f : 1;  // (f - 2) slots < 2 n_max items + slots
}

// Units that the start of an item counts as: none where CTAs have a unit or
// two, or one piece each (`factor` above 1).
PS_HD int ps_cost(int U, int factor, int slots) {
  return factor == 1 && U / 2 >= slots ? kPsCost : 0;
}

// floor(U c / G), G <= 1024, 0 <= c <= G.
PS_HD int ps_begin(int U, int c, int G) {
  const uint32_t q = (uint32_t)U / (uint32_t)G, r = (uint32_t)U - q * (uint32_t)G;  // r c <= 2^20
  return (int)(q * (uint32_t)c + r * (uint32_t)c / (uint32_t)G);
}

// The CTA whose range holds unit u (0 <= u < U, G <= U).
PS_HD int ps_owner(int u, int U, int G) {
  const long long c = (((long long)u + 1) * G - 1) / U;
  return c < 0 ? 0 : c < G ? (int)c : G - 1;
}

// Walks the pieces of one CTA: the item, its units in this CTA, and how many
// units of the range are left from the piece's first one on. Counted with the
// items' starts, the first unit of the piece's item is unit (end of the range)
// - left - unit.
struct PsCursor {
  int row, item;    // query row, item within the row
  int n;            // units of each of the row's items
  int unit, units;  // first unit of the piece within the item, unit count
  int left;
  int cost;         // units of an item's start
};

// The piece that starts `in_row` units after the start of row `row` (n units
// an item and `cost` for its start), with `left` units of the range to go. Not
// above 0 units: the range holds no more than (a part of) a start.
PS_HD PsCursor ps_first(int row, int in_row, int n, int items, int left, int cost = 0) {
  PsCursor c;
  c.row = row;
  c.n = n;
  c.cost = cost;
  const int each = n + cost, item = (int)((uint32_t)in_row / (uint32_t)each);
  c.item = item < items ? item : items - 1;
  const int in_item = (item < items ? in_row - item * each : each - 1) - cost;
  c.unit = in_item < 0 ? 0 : in_item;
  c.left = in_item < 0 ? left + in_item : left;
  c.units = c.left < n - c.unit ? c.left : n - c.unit;
  return c;
}

// Steps to the next piece; false at the range's end, and after the last of
// `rows` rows whatever the units say (lengths that another stream changes
// meanwhile give wrong results, but no index out of range). A row is done
// after `items` items; units_of(row) gives the next row's n.
template <typename F>
PS_HD bool ps_next(PsCursor& c, int items, int rows, F&& units_of) {
  c.left -= c.units + c.cost;
  if (c.left <= 0) return false;
  c.unit = 0;
  if (++c.item == items) {
    c.item = 0;
    if (++c.row >= rows) return false;
    c.n = units_of(c.row);
  }
  c.units = c.left < c.n ? c.left : c.n;
  return true;
}
