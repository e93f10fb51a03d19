// What a decode attention sees of a text, and its parts: shared by the plain
// cache and the one in 4 bits.
#pragma once
#include "decoder.hpp"

namespace ppocr {

// What of a text is seen, in tiles of KEYS tokens: those with sinks first,
// then those of the window, whose first starts at a multiple of KEYS (and of
// 16, so that a tile's halves lie in one page where pages are multiples of 16).
struct Seen {
  int length, low;     // tokens low .. length - 1 are in the window
  int sinks, first;    // tokens 0 .. sinks - 1 too; the window's first tile's start
  int sink_tiles, tiles;
};

__device__ __forceinline__ Seen seen_of(int length, int window, int sinks, int keys) {
  Seen s;
  s.length = max(length, 0);
  s.low = window > 0 && window < s.length ? s.length - window : 0;
  s.first = s.low / keys * keys;
  s.sinks = min(sinks, s.low);
  // A tile that holds sinks and the window's start is the window's.
  s.sink_tiles = min((s.sinks + keys - 1) / keys, s.first / keys);
  s.tiles = s.sink_tiles + (s.length - s.first + keys - 1) / keys;
  return s;
}

// Tiles of a part: as many in every text, so that workgroups have equal work
// where texts do not, unless a text is longer than was said.
__device__ __forceinline__ int tiles_a_part(int tiles, int each, int splits) {
  return max((tiles + splits - 1) / splits, each);
}

}  // namespace ppocr
