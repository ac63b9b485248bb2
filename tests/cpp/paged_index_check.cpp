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

// Every tile of every unit is taken once; a unit is written by the warp that
// takes it whole, by the CTA that joins all of its parts, or from the CTAs'
// partial slots, which lie where the join looks for them.
void check_split(const std::vector<int>& lengths, int units, int tile, int grid, int warps) {
  std::vector<int64_t> before(lengths.size() + 1, 0);
  for (size_t b = 0; b < lengths.size(); ++b)
    before[b + 1] = before[b] + opl::key_tiles(lengths[b], tile);
  const int64_t total = before.back() * units;
  const int ctas = opl::active_ctas(total, grid, warps);
  require(ctas >= 1 && ctas <= grid, "active CTAs");
  std::vector<char> written(lengths.size() * units, 0);
  std::vector<std::vector<char>> taken(lengths.size() * units);
  for (size_t b = 0; b < lengths.size(); ++b)
    for (int u = 0; u < units; ++u)
      taken[b * units + u].assign(opl::key_tiles(lengths[b], tile), 0);
  // Unit and tiles of each partial slot, as the CTAs fill them.
  std::vector<int64_t> slot_unit(2 * ctas, -1);
  std::vector<int> slot_begin(2 * ctas, -1), slot_end(2 * ctas, -1);
  const opl::Ranges ranges = opl::make_ranges(total, ctas * warps);
  const auto cta_start = [&](int64_t c) { return ranges.begin(c * warps); };
  require(cta_start(0) == 0 && cta_start(ctas) == total, "ranges cover all tiles");
  for (int c = 0; c < ctas; ++c) {
    const int64_t cta_begin = cta_start(c);
    require(cta_begin < cta_start(c + 1), "no empty CTA");
    std::vector<opl::PartRecord> storage(2 * warps, opl::PartRecord{});
    auto records = reinterpret_cast<opl::PartRecord(*)[2]>(storage.data());
    for (int x = 0; x < warps; ++x) {
      int64_t w = ranges.begin(static_cast<int64_t>(c) * warps + x);
      const int64_t limit = ranges.begin(static_cast<int64_t>(c) * warps + x + 1);
      const bool opens = w == cta_begin;
      size_t b = 0;
      while (w < limit) {
        while (w >= before[b + 1] * units) ++b;
        require(ranges.holder(w) == static_cast<int64_t>(c) * warps + x, "holder");
        const int tiles = opl::key_tiles(lengths[b], tile);
        const opl::TilePlace p = opl::place_of(w, before[b], tiles, units);
        require(p.unit >= 0 && p.unit < units && p.tile >= 0 && p.tile < tiles, "place");
        const int end = tiles - p.tile <= limit - w ? tiles : p.tile + static_cast<int>(limit - w);
        auto& mine = taken[b * units + p.unit];
        for (int t = p.tile; t < end; ++t) {
          require(mine[t] == 0, "a tile taken twice");
          mine[t] = 1;
        }
        w += end - p.tile;
        if (p.tile == 0 && end == tiles) {
          ++written[b * units + p.unit];
          continue;
        }
        const int kind = p.tile == 0 ? opl::kTail : opl::kHead;
        require(records[x][kind].empty(), "a warp has one head and one tail");
        records[x][kind] = {static_cast<int>(b), p.unit,    tiles, p.tile, end,
                            opens && kind == opl::kHead, w < limit};
        require(kind == opl::kHead || w == limit, "a tail ends its warp's range");
      }
    }
    uint32_t present = 0, starts = 0;
    for (int x = 0; x < 2 * warps; ++x) {
      present |= static_cast<uint32_t>(!storage[x].empty()) << x;
      starts |= static_cast<uint32_t>(opl::starts_unit(storage[x], x & 1)) << x;
    }
    uint32_t chained = 0;
    for (int x = 0; x < 2 * warps; ++x) {
      if ((starts >> x & 1u) == 0) continue;
      const uint32_t mine = opl::parts_of_unit(present, starts, x);
      require((mine & chained) == 0 && (mine >> x & 1u) != 0, "parts of a unit");
      chained |= mine;
      const opl::PartRecord& r = storage[x];
      int end = r.end;
      for (int y = x + 1; y < 2 * warps; ++y) {
        if ((mine >> y & 1u) == 0) continue;
        const opl::PartRecord& next = storage[y];
        require((mine >> (y ^ 1) & 1u) == 0, "one part of a warp");
        require(next.sequence == r.sequence && next.unit == r.unit && next.begin == end &&
                    next.opens == 0 && (y & 1) == opl::kHead,
                "a part out of place in the CTA");
        end = next.end;
      }
      const int64_t unit = static_cast<int64_t>(r.sequence) * units + r.unit;
      if (r.begin == 0 && end == r.tiles) {
        ++written[unit];
        continue;
      }
      const int slot = 2 * c + (r.begin == 0 ? 1 : 0);
      require(slot_unit[slot] == -1, "a partial slot used twice");
      slot_unit[slot] = unit;
      slot_begin[slot] = r.begin;
      slot_end[slot] = end;
    }
    require(present == chained, "a part of the CTA not joined");
  }
  for (const auto& unit : taken)
    for (char t : unit) require(t == 1, "a tile left out");
  // The join of CTA c, as paged_join_kernel finds it.
  size_t joined = 0;
  for (int c = 0; c + 1 < ctas; ++c) {
    const int64_t at = cta_start(c + 1) - 1;
    size_t b = 0;
    while (at >= before[b + 1] * units) ++b;
    const int tiles = opl::key_tiles(lengths[b], tile);
    const opl::TilePlace last = opl::place_of(at, before[b], tiles, units);
    if (last.tile + 1 == tiles) continue;
    const int64_t unit_begin = at - last.tile;
    if (unit_begin < cta_start(c)) continue;
    const int end_cta = static_cast<int>(ranges.holder(unit_begin + tiles - 1) / warps);
    const int64_t unit = static_cast<int64_t>(b) * units + last.unit;
    int next = 0;
    for (int p = 0; p <= end_cta - c; ++p, ++joined) {
      const int slot = p == 0 ? 2 * c + 1 : 2 * (c + p);
      require(slot_unit[slot] == unit && slot_begin[slot] == next, "a part out of place");
      next = slot_end[slot];
    }
    require(next == tiles, "a unit not joined to its end");
    ++written[unit];
  }
  size_t parts = 0;
  for (int64_t u : slot_unit) parts += u != -1;
  require(parts == joined, "a part not joined");
  for (char n : written) require(n == 1, "every unit is written once");
}

}  // namespace

int main() {
  check_divisions();
  check_guards();
  std::mt19937 rng(11);
  const opl::Ranges wide = opl::make_ranges((int64_t{1} << 40) + 77, 2368);
  for (int i = 0; i < 2368; ++i)
    require(wide.begin(i + 1) > wide.begin(i) && wide.holder(wide.begin(i)) == i &&
                wide.holder(wide.begin(i + 1) - 1) == i,
            "ranges past 32 bits");
  require(wide.begin(2368) == (int64_t{1} << 40) + 77, "ranges past 32 bits");
  const opl::TilePlace far = opl::place_of((int64_t{1} << 36) + 5, 3, 1 << 26, 4096);
  require(far.unit == ((int64_t{1} << 36) + 5 - 3 * 4096) >> 26 &&
              far.tile == (((int64_t{1} << 36) + 5 - 3 * 4096) & ((1 << 26) - 1)),
          "a place past 32 bits");
  check_split({0}, 1, 16, 296, 8);
  check_split({1}, 1, 16, 1, 8);
  check_split({131071}, 8, 16, 296, 8);
  check_split({0, 0, 0, 5}, 3, 8, 4, 4);
  for (int trial = 0; trial < 3000; ++trial) {
    const int batch = 1 + rng() % 40, units = 1 + rng() % 12, warps = 1 + rng() % 8;
    const int most = 1 << (rng() % 12), grid = 1 + rng() % 300;
    std::vector<int> lengths(batch);
    for (int& n : lengths) n = rng() % 5 == 0 ? 0 : static_cast<int>(rng() % (most + 1));
    check_split(lengths, units, rng() % 2 ? 8 : 16, grid, warps);
  }
  std::printf("PASS\n");
  return 0;
}
