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

// floor(U c / G) without the wide product.
PS_HD long long ps_begin(long long U, int c, int G) { return U / G * c + U % G * c / G; }

// The CTA whose range holds unit u (0 <= u < U, G <= U).
PS_HD int ps_owner(long long u, long long U, int G) { return (int)(((u + 1) * G - 1) / U); }

// One CTA's piece of an item.
struct PsPiece {
  int row, item;           // query row, item within the row
  int unit, units;         // first unit of the piece within the item, unit count
  int first_cta, last_cta; // CTAs that hold the item (equal: the item is whole)
};

// The piece that starts at unit u of a row whose units start at row_start
// (n units for each item) and ends by u_end.
PS_HD PsPiece ps_piece(long long u, long long u_end, int row, long long row_start, int n,
                       long long U, int G) {
  PsPiece p;
  const long long in_row = u - row_start;
  p.row = row;
  p.item = (int)(in_row / n);
  p.unit = (int)(in_row % n);
  const long long left = u_end - u;
  p.units = left < n - p.unit ? (int)left : n - p.unit;
  const long long a = row_start + (long long)p.item * n;
  p.first_cta = ps_owner(a, U, G);
  p.last_cta = ps_owner(a + n - 1, U, G);
  return p;
}
