// How the keys of a ragged batch are cut over the CTAs of one launch, in plain
// C++ so that it can be tested without a GPU.
//
// A unit is one sequence's keys for one group of query rows (a key-value head,
// or a part of its query heads).  Its keys are cut into tiles (an empty
// sequence counts one); the tiles of all units are laid end to end, sequence
// after sequence, and CTA c takes [begin(c), begin(c + 1)) of them.  Lengths
// stay on the device, so every CTA computes the total and its own start.
//
// A CTA's range cuts at most two units: the one it starts inside of (partial
// slot 0) and the one it ends inside of (slot 1; when both are the same unit,
// slot 0).  So the parts of a cut unit are slot 1 of the CTA that starts it
// and slot 0 of the CTAs that follow, in key order.
#pragma once

#include <cstdint>

#include "paged_index.h"

namespace opl {

OPL_HD int key_tiles(int length, int tile) { return length <= tile ? 1 : (length - 1) / tile + 1; }

// CTAs that take part: each gets at least `least` tiles, but for the last
// ones of a small call.
OPL_HD int active_ctas(int64_t total, int ctas, int least) {
  const int64_t useful = (total + least - 1) / least;
  return useful < ctas ? static_cast<int>(useful) : ctas;
}

OPL_HD int64_t range_begin(int64_t total, int ctas, int cta) { return total * cta / ctas; }

// The CTA whose range holds tile w.
OPL_HD int range_owner(int64_t total, int ctas, int64_t w) {
  return static_cast<int>(((w + 1) * ctas + total - 1) / total) - 1;
}

// One run of tiles of one unit.  `before` is the number of tiles of a single
// unit in the sequences before `sequence`, whose units start at
// units * before.
struct Segment {
  int unit;   // of the sequence, 0 .. units - 1
  int tiles;  // of the unit
  int begin, end;

  OPL_HD bool whole() const { return begin == 0 && end == tiles; }
  OPL_HD int slot() const { return begin == 0 ? 1 : 0; }
};

OPL_HD Segment segment_at(int64_t w, int64_t limit, int64_t before, int tiles, int units) {
  Segment s;
  const int64_t local = w - before * units;
  s.tiles = tiles;
  s.unit = static_cast<int>(local / tiles);
  s.begin = static_cast<int>(local - static_cast<int64_t>(s.unit) * tiles);
  const int64_t left = limit - w;
  s.end = tiles - s.begin <= left ? tiles : static_cast<int>(s.begin + left);
  return s;
}

}  // namespace opl
