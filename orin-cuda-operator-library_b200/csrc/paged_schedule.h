// How the keys of a ragged batch are cut over the warps and CTAs of one launch,
// in plain C++ so that it can be tested without a GPU.
//
// A unit is one sequence's keys for one group of query rows (a key-value head,
// or a part of its query heads).  Its keys are cut into tiles (an empty
// sequence counts one); the tiles of all units are laid end to end, sequence
// after sequence, and every warp takes an equal range of them, the warps of a
// CTA next to one another.  Lengths stay on the device, so every CTA computes
// the total and where its warps start.
//
// A warp writes the units that it covers whole to the output.  Of the at most
// two that its range cuts it leaves parts: its head (a unit that an earlier
// warp starts) and its tail (a unit that it starts and does not end).  The CTA
// joins the parts of a unit that follow one another, and a unit that reaches
// past the CTA is left as a part of the CTA: slot 0 if an earlier CTA starts
// it, else slot 1.  So the parts of a unit cut between CTAs are slot 1 of the
// CTA that starts it and slot 0 of the CTAs that follow, in key order.
#pragma once

#include <cstdint>

#include "paged_index.h"

namespace opl {

OPL_HD int key_tiles(int length, int tile) { return length <= tile ? 1 : (length - 1) / tile + 1; }

// CTAs that take part: no more than give every warp a tile.
OPL_HD int active_ctas(int64_t total, int ctas, int warps) {
  const int64_t useful = (total + warps - 1) / warps;
  return useful < ctas ? static_cast<int>(useful) : ctas;
}

// `total` tiles over `count` ranges that differ by at most one tile, the longer
// ones first.
struct Ranges {
  int64_t each;  // tiles of a shorter range
  int64_t more;  // ranges with one tile more

  OPL_HD int64_t begin(int64_t index) const {
    return each * index + (index < more ? index : more);
  }
  OPL_HD int64_t holder(int64_t tile) const {  // the range of a tile
    const int64_t longer = (each + 1) * more;
    return tile < longer ? quotient(tile, each + 1) : more + quotient(tile - longer, each);
  }
  // 64-bit divisions take hundreds of cycles.
  static OPL_HD int64_t quotient(int64_t a, int64_t b) {
    if (a >> 32 == 0 && b >> 32 == 0)
      return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
    return a / b;
  }
};

OPL_HD Ranges make_ranges(int64_t total, int count) {
  Ranges r;
  r.each = Ranges::quotient(total, count);
  r.more = total - r.each * count;
  return r;
}

// A tile of the batch: of unit `unit` (0 .. units - 1) of a sequence whose
// units have `tiles` tiles.
struct TilePlace {
  int unit, tile;
};

// Place of tile `w` in the sequence that holds it; `before` is the number of
// tiles of a single unit in the sequences before, whose units start at
// units * before.
OPL_HD TilePlace place_of(int64_t w, int64_t before, int tiles, int units) {
  const int64_t local = w - before * units;
  TilePlace p;
  p.unit = static_cast<int>(Ranges::quotient(local, tiles));
  p.tile = static_cast<int>(local - static_cast<int64_t>(p.unit) * tiles);
  return p;
}

// A part that a warp leaves, empty when begin == end.
struct PartRecord {
  int sequence, unit, tiles, begin, end;
  int opens;    // a head with which the CTA's range begins
  int aside;    // a head with more of the warp's range behind it

  OPL_HD bool empty() const { return begin == end; }
};

constexpr int kHead = 0, kTail = 1;

// The parts of a CTA in key order are its warps' heads and tails, warp after
// warp: bit 2 * warp + kind of these masks.  `present` are the parts that are
// not empty, `starts` the first of each unit (a tail, or the head with which
// the CTA's range begins).  The parts from a start up to the next one are one
// unit's.
OPL_HD bool starts_unit(const PartRecord& r, int kind) {
  return !r.empty() && (kind == kTail || r.opens != 0);
}

OPL_HD uint32_t parts_of_unit(uint32_t present, uint32_t starts, int start) {
  const uint32_t later = starts & ~((2u << start) - 1);
  const uint32_t end = later & (0u - later);  // lowest; none: 0
  return present & (end - 1) & ~((1u << start) - 1);
}

}  // namespace opl
