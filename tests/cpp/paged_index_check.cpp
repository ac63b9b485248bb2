// Host check of the paged cache's index guards and of the split of a ragged
// batch over CTAs (csrc/paged_index.h, csrc/paged_schedule.h): built by a
// plain C++ compiler, no GPU.  Prints PASS, or the first failure.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "paged_schedule.h"

namespace {

void require(bool ok, const char* what) {
  if (ok) return;
  std::printf("FAIL %s\n", what);
  std::exit(1);
}

void check_divisions() {
  std::mt19937 rng(7);
  for (uint32_t d : {1u, 2u, 3u, 5u, 7u, 16u, 24u, 100u, 255u, 4096u, 65537u, 0x7fffffffu}) {
    const opl::FastDiv f = opl::make_fast_div(d);
    for (uint32_t n : {0u, 1u, d - 1, d, d + 1, 2 * d - 1, 0x7ffffffeu, 0x7fffffffu})
      if (n < 0x80000000u) require(opl::fast_div(n, f) == n / d, "fast_div");
    for (int i = 0; i < 10000; ++i) {
      const uint32_t n = rng() & 0x7fffffffu;
      require(opl::fast_div(n, f) == n / d, "fast_div");
    }
  }
}

void check_guards() {
  int64_t page = 77;
  int inside = 77;
  require(opl::cache_slot(-1, 4, 16, &page, &inside) == -1, "negative slot is skipped");
  require(opl::cache_slot(INT64_MIN, 4, 16, &page, &inside) == -1, "lowest slot is skipped");
  require(opl::cache_slot(64, 4, 16, &page, &inside) == opl::kBadSlot, "slot past the cache");
  require(opl::cache_slot(INT64_MAX, 4, 16, &page, &inside) == opl::kBadSlot, "highest slot");
  require(page == 77 && inside == 77, "a refused slot sets nothing");
  require(opl::cache_slot(63, 4, 16, &page, &inside) == 0 && page == 3 && inside == 15, "last slot");
  require(opl::cache_slot((int64_t{1} << 40) + 5, int64_t{1} << 36, 24, &page, &inside) == 0 &&
              page == ((int64_t{1} << 40) + 5) / 24 && inside == ((int64_t{1} << 40) + 5) % 24,
          "slot past 32 bits");
  require(opl::cache_page(0, 3) && opl::cache_page(2, 3), "pages of the cache");
  require(!opl::cache_page(-1, 3) && !opl::cache_page(3, 3) && !opl::cache_page(INT32_MIN, 3) &&
              !opl::cache_page(INT32_MAX, 3),
          "pages outside the cache");
  require(opl::readable_length(-5, 2, 16) == 0, "negative length");
  require(opl::readable_length(33, 2, 16) == 32, "length past the table");
  require(opl::readable_length(31, 2, 16) == 31, "length");
  require(opl::readable_length(INT32_MAX, 1 << 20, 1 << 20) == INT32_MAX, "capacity past 32 bits");
}

// Every tile of every unit is taken once; whole units have no part; the parts
// of a cut unit are where the join looks for them.
void check_split(const std::vector<int>& lengths, int units, int tile, int grid, int least) {
  std::vector<int64_t> before(lengths.size() + 1, 0);
  for (size_t b = 0; b < lengths.size(); ++b)
    before[b + 1] = before[b] + opl::key_tiles(lengths[b], tile);
  const int64_t total = before.back() * units;
  const int ctas = opl::active_ctas(total, grid, least);
  require(ctas >= 1 && ctas <= grid, "active CTAs");
  std::vector<std::vector<char>> taken(lengths.size() * units);
  for (size_t b = 0; b < lengths.size(); ++b)
    for (int u = 0; u < units; ++u)
      taken[b * units + u].assign(opl::key_tiles(lengths[b], tile), 0);
  // Unit and first tile of each partial slot, as the CTAs fill them.
  std::vector<int64_t> slot_unit(2 * ctas, -1);
  std::vector<int> slot_begin(2 * ctas, -1), slot_end(2 * ctas, -1);
  require(opl::range_begin(total, ctas, 0) == 0 && opl::range_begin(total, ctas, ctas) == total,
          "ranges cover all tiles");
  for (int c = 0; c < ctas; ++c) {
    int64_t w = opl::range_begin(total, ctas, c);
    const int64_t limit = opl::range_begin(total, ctas, c + 1);
    require(w < limit, "no empty range");
    size_t b = 0;
    while (w < limit) {
      while (w >= before[b + 1] * units) ++b;
      require(opl::range_owner(total, ctas, w) == c, "owner");
      const int tiles = opl::key_tiles(lengths[b], tile);
      const opl::Segment s = opl::segment_at(w, limit, before[b], tiles, units);
      require(s.unit >= 0 && s.unit < units && s.begin < s.end && s.end <= tiles, "segment");
      auto& mine = taken[b * units + s.unit];
      for (int t = s.begin; t < s.end; ++t) {
        require(mine[t] == 0, "a tile taken twice");
        mine[t] = 1;
      }
      if (!s.whole()) {
        const int slot = 2 * c + s.slot();
        require(slot_unit[slot] == -1, "a partial slot used twice");
        slot_unit[slot] = static_cast<int64_t>(b) * units + s.unit;
        slot_begin[slot] = s.begin;
        slot_end[slot] = s.end;
      }
      w += s.end - s.begin;
    }
  }
  for (const auto& unit : taken)
    for (char t : unit) require(t == 1, "a tile left out");
  // The join of CTA c, as paged_join_kernel finds it.
  size_t joined = 0;
  for (int c = 0; c + 1 < ctas; ++c) {
    const int64_t limit = opl::range_begin(total, ctas, c + 1), at = limit - 1;
    size_t b = 0;
    while (at >= before[b + 1] * units) ++b;
    const int tiles = opl::key_tiles(lengths[b], tile);
    const opl::Segment last = opl::segment_at(at, limit, before[b], tiles, units);
    if (last.end == tiles) continue;
    const int64_t unit_begin = at - last.begin;
    if (unit_begin < opl::range_begin(total, ctas, c)) continue;
    const int end_cta = opl::range_owner(total, ctas, unit_begin + tiles - 1);
    const int64_t unit = static_cast<int64_t>(b) * units + last.unit;
    int next = 0;
    for (int p = 0; p <= end_cta - c; ++p, ++joined) {
      const int slot = p == 0 ? 2 * c + 1 : 2 * (c + p);
      require(slot_unit[slot] == unit && slot_begin[slot] == next, "a part out of place");
      next = slot_end[slot];
    }
    require(next == tiles, "a unit not joined to its end");
  }
  size_t parts = 0;
  for (int64_t u : slot_unit) parts += u != -1;
  require(parts == joined, "a part not joined");
}

}  // namespace

int main() {
  check_divisions();
  check_guards();
  std::mt19937 rng(11);
  check_split({0}, 1, 16, 296, 8);
  check_split({1}, 1, 16, 1, 8);
  check_split({131071}, 8, 16, 296, 8);
  check_split({0, 0, 0, 5}, 3, 8, 4, 1);
  for (int trial = 0; trial < 600; ++trial) {
    const int batch = 1 + rng() % 40, units = 1 + rng() % 12;
    const int most = 1 << (rng() % 12), grid = 1 + rng() % 300, least = 1 + rng() % 16;
    std::vector<int> lengths(batch);
    for (int& n : lengths) n = rng() % 5 == 0 ? 0 : static_cast<int>(rng() % (most + 1));
    check_split(lengths, units, rng() % 2 ? 8 : 16, grid, least);
  }
  std::printf("PASS\n");
  return 0;
}
