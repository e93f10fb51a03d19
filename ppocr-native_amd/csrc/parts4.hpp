// The parts that texts of a cache in 4 bits are split into: shared by their
// attention and its join.
#pragma once
#include "seen.hpp"
#include "writer.hpp"

namespace ppocr {

// Texts times their groups of heads up to which a call's parts go by what the
// lengths are. Each workgroup adds the lengths up, and with more of them there is
// enough to do without parts (100 texts to 4000, 8 key heads: 79 us so, 67 as the
// host chose; 300 to 2000: 156 and 85; but 128 to 4000 of 2 key heads: 30 and 46).
constexpr long kShared4 = 768;

// A text's tiles.
__device__ __forceinline__ Seen seen4(const Attend4Args &a, int b, int keys) {
  const int length = a.c.lengths[b];
  return seen_of(length > a.c.table_width * a.c.page_size ? 0 : length, a.window, a.sinks, keys);
}
// Tiles of a part, so that all texts have as many parts together as are wanted:
// by what the lengths are, which the host does not know. By a whole wave.
__device__ __forceinline__ int each4(const Attend4Args &a, int keys) {
  if (!a.pieces) return a.each;
  float sum = 0.0f;  // (a choice only, the same in every wave)
  for (int i = threadIdx.x % 64; i < a.batch; i += 64) sum += (float)seen4(a, i, keys).tiles;
#pragma unroll
  for (int o = 1; o < 64; o *= 2) sum += __shfl_xor(sum, o);
  return max(a.each, (int)fminf(ceilf(sum / (float)a.pieces), 0x1p30f));
}
// Text and part of the parts' number `id`, text after text; text -1: none.
struct Piece4 {
  int b, part;
};
__device__ __forceinline__ Piece4 piece4(const Attend4Args &a, int keys, int each, int id) {
  const int lane = threadIdx.x % 64;
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    int n = 0;
    if (b0 + lane < a.batch) {
      const int tiles = seen4(a, b0 + lane, keys).tiles, of = tiles_a_part(tiles, each, a.splits);
      n = max((tiles + of - 1) / of, 1);  // (an empty text's part writes its zeros)
    }
    int to = n;  // parts of the texts up to this one
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
      const int before = __shfl_up(to, o);
      to += lane >= o ? before : 0;
    }
    const uint64_t past = __ballot(to > id);
    if (past) {
      const int at = __builtin_ctzll(past);
      return {b0 + at, id - __builtin_amdgcn_readlane(to - n, at)};
    }
    id -= __builtin_amdgcn_readlane(to, 63);
  }
  return {-1, 0};
}

// A mean of values into an output of `type`. In f16 it is held at the largest, as
// what is read of the cache is: codes can stand for 60 more. (NaN stays NaN.)
__device__ __forceinline__ void put_at(void *p, long i, int type, float v) {
  if (type == PPOCR_F32)
    ((float *)p)[i] = v;
  else if (type == PPOCR_BF16)
    ((__bf16 *)p)[i] = (__bf16)v;
  else
    ((_Float16 *)p)[i] = (_Float16)(v > 65504.0f ? 65504.0f : v);
}

}  // namespace ppocr
