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

static void run(const std::vector<int>& lens, long long capacity, int window, int items, int grid,
                int unit) {
  const int R = (int)lens.size();
  long long U = 0;
  for (int r = 0; r < R; ++r) U += (long long)ps_units(ps_row(lens[r], capacity, window), unit) * items;
  const int G = (int)std::min<long long>(grid, U);
  std::map<std::pair<int, int>, std::vector<std::pair<int, PsPiece>>> of;  // item -> (cta, piece)
  long long covered = 0;
  for (int c = 0; c < G; ++c) {
    long long u = ps_begin(U, c, G);
    const long long u_end = ps_begin(U, c + 1, G);
    CHECK(u < u_end);
    CHECK(ps_owner(u, U, G) == c && ps_owner(u_end - 1, U, G) == c);
    int row = 0;
    long long start = 0;
    for (;;) {
      const long long n = (long long)ps_units(ps_row(lens[row], capacity, window), unit) * items;
      if (u < start + n) break;
      start += n;
      ++row;
    }
    int continued = 0, joined_in = 0;
    while (u < u_end) {
      const PsRow keys = ps_row(lens[row], capacity, window);
      const int n = ps_units(keys, unit);
      if (u >= start + (long long)n * items) {
        start += (long long)n * items;
        ++row;
        CHECK(row < R);
        continue;
      }
      const PsPiece p = ps_piece(u, u_end, row, start, n, U, G);
      CHECK(p.units >= 1 && p.unit >= 0 && p.unit + p.units <= n && p.item < items);
      CHECK(p.first_cta <= c && c <= p.last_cta);
      CHECK((p.unit == 0) == (c == p.first_cta));
      CHECK((p.unit + p.units == n) == (c == p.last_cta));
      if (p.first_cta != p.last_cta) (c == p.first_cta ? continued : joined_in)++;
      of[{row, p.item}].push_back({c, p});
      covered += p.units;
      u += p.units;
    }
    CHECK(continued <= 1 && joined_in <= 1);
  }
  CHECK(covered == U);
  CHECK((long long)of.size() == (long long)R * items);
  std::set<int> counters;
  for (auto& [key, pieces] : of) {
    int at = 0, cta = pieces[0].second.first_cta;
    for (auto& [c, p] : pieces) {
      CHECK(p.unit == at && c == cta);
      at += p.units;
      ++cta;
    }
    CHECK(at == ps_units(ps_row(lens[key.first], capacity, window), unit));
    CHECK(cta - 1 == pieces[0].second.last_cta);
    if (pieces.size() > 1) CHECK(counters.insert(pieces[0].second.first_cta).second);
  }
}

int main() {
  std::mt19937 g(7);
  auto pick = [&](int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(g); };
  run({0}, 16, 0, 1, 444, 64);
  run({1}, 16, 0, 8, 444, 64);
  run({131072}, 131072, 0, 8, 444, 64);
  run({0x7fffffff}, 0x7fff0000ll, 0, 1, 1024, 64);
  run({-5, 70000, 0, 65}, 1 << 20, 0, 3, 296, 64);
  run(std::vector<int>(65, 64), 1 << 20, 0, 2, 7, 64);
  for (int i = 0; i < 400; ++i) {
    std::vector<int> lens(pick(1, 80));
    const int most = 1 << pick(0, 14);
    for (int& l : lens) l = pick(0, 4) == 0 ? 0 : pick(0, most);
    run(lens, pick(0, 1) ? 1 << 20 : most / 2 + 1, pick(0, 2) ? 0 : pick(1, most), pick(1, 40),
        pick(1, 600), 1 << pick(4, 8));
  }
  std::printf("%s (%d failures)\n", failures ? "FAILED" : "ok", failures);
  return failures != 0;
}
