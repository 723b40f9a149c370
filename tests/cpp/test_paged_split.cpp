// The split of paged attention's work over CTAs (paged_split.cuh), the code
// the kernel runs, checked on random batches: every key of every item lies in
// exactly one piece, the pieces of an item are held by consecutive CTAs, at
// most one item continues past a CTA's end and one into its start (the two
// partial results a CTA has room for), and the joining counter of an item
// that spans CTAs belongs to no other item.
#include <algorithm>
#include <cstdio>
#include <map>
#include <random>
#include <set>
#include <vector>

#include "../../molten_b200/csrc/paged_split.cuh"

static int failures = 0;
#define CHECK(c)                                             \
  do {                                                       \
    if (!(c)) {                                              \
      if (failures++ < 10) std::printf("FAIL line %d: %s\n", __LINE__, #c); \
    }                                                        \
  } while (0)

static void run(const std::vector<int>& lens, int capacity, int window, int items, int grid,
                int unit) {
  const int R = (int)lens.size();
  unit = ps_small_unit(unit, (long long)R * items, capacity);
  CHECK(unit > 0);
  long long sum = 0;
  int n_max = 0;
  for (int r = 0; r < R; ++r) {
    const int n = ps_units(ps_row(lens[r], capacity, window), unit);
    sum += (long long)n * items;
    n_max = std::max(n_max, n);
  }
  CHECK(sum <= 0x7fffffff);
  const int f = ps_factor((int)sum, n_max, R * items, grid);
  CHECK(f >= 1 && (f == 1 || f <= n_max));
  const bool one_each = f > 1 || ((long long)R * items <= grid && n_max <= 3);
  unit = (int)std::min<long long>((long long)unit * f, 0x7fffffff);
  int U = 0;
  for (int r = 0; r < R; ++r) U += ps_units(ps_row(lens[r], capacity, window), unit) * items;
  const int G = std::min(grid, U);
  auto units_of = [&](int r) {
    CHECK(r < R);
    return ps_units(ps_row(lens[r], capacity, window), unit);
  };
  std::map<std::pair<int, int>, std::vector<std::pair<int, PsCursor>>> of;  // item -> (cta, piece)
  int covered = 0;
  for (int c = 0; c < G; ++c) {
    const int u0 = ps_begin(U, c, G), u_end = ps_begin(U, c + 1, G);
    CHECK(u0 < u_end);
    CHECK(ps_owner(u0, U, G) == c && ps_owner(u_end - 1, U, G) == c);
    int row = 0;
    int start = 0;
    for (;;) {
      const int n = units_of(row) * items;
      if (u0 < start + n) break;
      start += n;
      ++row;
    }
    int continued = 0, joined_in = 0;
    PsCursor p = ps_first(row, u0 - start, units_of(row), items, u_end - u0);
    do {
      CHECK(p.units >= 1 && p.unit >= 0 && p.unit + p.units <= p.n && p.item < items);
      CHECK(p.n == units_of(p.row) && p.left == u_end - u0 - (covered - u0));
      const bool begins = p.unit == 0, ends = p.unit + p.units == p.n;
      // what the kernel asks of an item that is not whole in this CTA
      const int u = u_end - p.left;
      CHECK((ps_owner(u - p.unit, U, G) == c) == begins);
      CHECK((ps_owner(u - p.unit + p.n - 1, U, G) == c) == ends);
      if (!(begins && ends)) (begins ? continued : joined_in)++;
      of[{p.row, p.item}].push_back({c, p});
      covered += p.units;
    } while (ps_next(p, items, R, units_of));
    CHECK(covered == u_end);
    CHECK(continued <= 1 && joined_in <= 1);
    if (one_each) CHECK(u_end - u0 == 1);
  }
  CHECK(covered == U);
  CHECK((long long)of.size() == (long long)R * items);
  std::set<int> counters;
  for (auto& [key, pieces] : of) {
    int at = 0, cta = pieces[0].first;
    for (auto& [c, p] : pieces) {
      CHECK(p.unit == at && c == cta);
      at += p.units;
      ++cta;
    }
    CHECK(at == units_of(key.first));
    if (pieces.size() > 1) CHECK(counters.insert(pieces[0].first).second);
  }
}

// The same with `cost` units for the start of every item, which hold no keys: CTAs whose range is
// no more than a start have no piece.
static void run_with_starts(const std::vector<int>& lens, int capacity, int items, int grid,
                            int unit, int cost) {
  const int R = (int)lens.size();
  auto units_of = [&](int r) { return ps_units(ps_row(lens[r], capacity, 0), unit); };
  long long sum = 0, real = 0;
  for (int r = 0; r < R; ++r) {
    sum += ((long long)units_of(r) + cost) * items;
    real += (long long)units_of(r) * items;
  }
  CHECK(sum <= 0x7fffffff);
  const int U = (int)sum, G = std::min(grid, U);
  std::map<std::pair<int, int>, std::vector<std::pair<int, PsCursor>>> of;
  long long covered = 0;
  for (int c = 0; c < G; ++c) {
    const int u0 = ps_begin(U, c, G), u_end = ps_begin(U, c + 1, G);
    int row = 0, start = 0;
    for (;;) {
      const int n = (units_of(row) + cost) * items;
      if (u0 < start + n) break;
      start += n;
      ++row;
    }
    PsCursor p = ps_first(row, u0 - start, units_of(row), items, u_end - u0, cost);
    if (p.units <= 0) {
      CHECK(p.unit == 0 && u_end - u0 <= cost);
      continue;
    }
    int continued = 0, joined_in = 0, spent = 0;
    do {
      CHECK(p.units >= 1 && p.unit >= 0 && p.unit + p.units <= p.n && p.item < items);
      CHECK(p.n == units_of(p.row) && p.units <= p.left);
      const bool begins = p.unit == 0, ends = p.unit + p.units == p.n;
      const int first = u_end - p.left - p.unit;  // of the item, as the kernel finds it
      CHECK((ps_owner(first, U, G) == c) == begins);
      CHECK((ps_owner(first + p.n - 1, U, G) == c) == ends);
      if (!(begins && ends)) (begins ? continued : joined_in)++;
      of[{p.row, p.item}].push_back({c, p});
      covered += p.units;
      spent += p.units;
    } while (ps_next(p, items, R, units_of));
    CHECK(continued <= 1 && joined_in <= 1 && spent <= u_end - u0);
  }
  CHECK(covered == real && (long long)of.size() == (long long)R * items);
  std::set<int> counters;
  for (auto& [key, pieces] : of) {
    int at = 0, cta = pieces[0].first;
    for (auto& [c, p] : pieces) {
      CHECK(p.unit == at && c == cta);
      at += p.units;
      ++cta;
    }
    CHECK(at == units_of(key.first));
    if (pieces.size() > 1) CHECK(counters.insert(pieces[0].first).second);
  }
}

static void divisions(std::mt19937& g) {
  std::vector<int> ds{1, 2, 3, 5, 7, 16, 20, 24, 1000, 65535, 65536, 65537, 0x3fffffff, 0x40000000, 0x40000001, 0x7ffffffe, 0x7fffffff};
  for (int i = 0; i < 300; ++i) ds.push_back((int)(g() >> (1 + g() % 30)) | 1), ds.push_back((int)(g() >> (1 + g() % 30)) + 1);
  for (int d : ds) {
    if (d < 1) continue;
    const PsDiv v = ps_div_of(d);
    CHECK(d == 1 || (v.shift >= 0 && v.shift < 32));
    for (int i = 0; i < 2000; ++i) {
      const int k = (int)(g() >> 1) / d;  // multiples of d and their neighbours, and anything
      for (long long n : {(long long)k * d - 1, (long long)k * d, (long long)k * d + 1, (long long)(g() >> 1), 0x7fffffffll - i})
        if (n >= 0 && n <= 0x7fffffff) CHECK(ps_div((int)n, v) == n / d);
    }
  }
}

int main() {
  std::mt19937 g(7);
  auto pick = [&](int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(g); };
  divisions(g);
  run({0}, 16, 0, 1, 444, 64);
  run({1}, 16, 0, 8, 444, 64);
  run({131072}, 131072, 0, 8, 444, 64);
  run({0x7fffffff}, 0x7fff0000, 0, 1, 1024, 64);
  run(std::vector<int>(300, 0x7fffffff), 0x7fff0000, 0, 9, 1024, 64);
  CHECK(ps_small_unit(64, 1ll << 40, 1) == 0);
  run({-5, 70000, 0, 65}, 1 << 20, 0, 3, 296, 64);
  run(std::vector<int>(65, 64), 1 << 20, 0, 2, 7, 64);
  for (int i = 0; i < 400; ++i) {
    std::vector<int> lens(pick(1, 80));
    const int most = 1 << pick(0, 14);
    for (int& l : lens) l = pick(0, 4) == 0 ? 0 : pick(0, most);
    run(lens, pick(0, 1) ? 1 << 20 : most / 2 + 1, pick(0, 2) ? 0 : pick(1, most), pick(1, 40),
        pick(1, 600), 1 << pick(4, 8));
  }
  run_with_starts({0x7fffffff}, 0x7fff0000, 1, 1024, 64, kPsCost);
  run_with_starts({0}, 16, 1, 1, 64, 3);
  run_with_starts({5, 0, 0, 4000, 1}, 1 << 20, 8, 296, 128, kPsCost);
  CHECK(ps_cost(100, 1, 50) == kPsCost && ps_cost(99, 1, 50) == 0 && ps_cost(100, 2, 50) == 0);
  for (long long items : {1ll, 1000ll, 1000000ll}) {  // starts and units together stay in 31 bits
    const long long u = ps_small_unit(64, items, 0x7fff0000), n = (0x7fff0000 + u - 1) / u;
    CHECK(u > 0 && items * (n + kPsCost) <= 0x7fffffff);
  }
  for (int i = 0; i < 400; ++i) {
    std::vector<int> lens(pick(1, 60));
    const int most = 1 << pick(0, 14);
    for (int& l : lens) l = pick(0, 4) == 0 ? 0 : pick(0, most);
    run_with_starts(lens, 1 << 20, pick(1, 40), pick(1, 600), 1 << pick(4, 8), pick(0, 5));
  }
  std::printf("%s (%d failures)\n", failures ? "FAILED" : "ok", failures);
  return failures != 0;
}
