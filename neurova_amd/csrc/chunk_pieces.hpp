// Lengths of sequences, and of the pieces that a row block's keys are cut into, are counted in
// units of 64 << u keys: a tile, or two or four for tables of more than 2^26 or 2^27 tokens, so
// that no length is above kMostUnits.  (constexpr: for the host too.)
#pragma once

namespace lb {

constexpr int kTileShift = 6, kMostUnits = 1 << 20;  // log2 of a tile's keys

constexpr int units_of(int keys, int shift) { return (keys + (1 << shift) - 1) >> shift; }  // keys up to 2^28
constexpr int unit_shift(int max_tokens) {
  int shift = kTileShift;
  while (units_of(max_tokens, shift) > kMostUnits) ++shift;
  return shift;
}

// Pieces of at most `most` units in `units`, both from 1 to kMostUnits; `inverse` is 1 / most, off
// by at most one in its last place.  The fp32 quotient has a relative error of 2^-22 (1.5 in the last
// place of the inverse, half of one in the product).  (x + 1/2) / most is 1 / (2 most) away from
// a whole number, which is more as long as x + 1/2 is below 2^21.
constexpr int pieces_in(int units, int most, float inverse) { return (int)(((float)(units + most - 1) + 0.5f) * inverse); }

}  // namespace lb
