// Launch arguments and launchers of what a text decoder writes with: the
// rotation of positions with the append, the cache held in 4 bits, beam search.
// As in decoder.hpp: strides count values, shapes are checked by the C entries
// (writer.cpp), launchers never synchronise or allocate.
#pragma once
#include "decoder.hpp"

namespace ppocr {

// The rotation of rows by their positions, and the queries that go with it.
struct TurnArgs {
  const void *q;  // NULL: no queries
  void *q_out;
  long q_stride, q_out_stride;
  int heads;
  const float *freqs;    // rotary / 2, radians a position
  const int *positions;  // NULL: a token's place in its text
  int rotary, pairs;     // dims turned, in neighbouring pairs or halves apart
};

struct TurnedAppendArgs {
  AppendArgs a;
  TurnArgs t;
  int units;  // of two pieces of a head
  Divide by_unit, by_half;
};
hipError_t launch_kv_append_turned(const TurnedAppendArgs &a, int type, hipStream_t s);

// A cache in 4 bits: a page has a chunk of each key head, a chunk the planes
// K codes, scales, minima, V codes, scales, minima.
struct Kv4Args {
  char *data;
  long page_stride;  // bytes
  int chunk;         // bytes
  int at_ks, at_km, at_v, at_vs, at_vm;  // where a chunk's planes begin
  int pages, page_size, heads, dim, nc, group, groups;  // nc: 32s of a padded head
  Divide by_page;
  const int *table;
  long table_width;
  const int *lengths;
};

struct Append4Args {
  Kv4Args c;
  const void *k, *v;
  long k_stride, v_stride;
  const int *starts;
  long rows;
  int batch;
  TurnArgs t;
  int units;
  int teams;                // of threads, for the queries
  Divide by_unit, by_half;  // of a head; the turned pairs
};
hipError_t launch_kv4_append(const Append4Args &a, int type, hipStream_t s);

struct Read4Args {
  Kv4Args c;
  void *k, *v;
  long k_stride, v_stride;
  const int *starts;
  long rows;
  int batch;
};
hipError_t launch_kv4_read(const Read4Args &a, int type, hipStream_t s);

struct Attend4Args {
  Kv4Args c;
  const void *q;
  void *y;
  long q_stride, y_stride;
  int type, batch, heads;
  int splits, each;
  int window, sinks;
  float scale;  // not negative
  bool turn;    // the given one was negative
  float *part;  // splits > 1: batch x heads x splits rows of dim + 2 floats
  int pieces;   // parts of all texts that are wanted (but for batch of them at most), or 0: `each` says
};
PagedParts kv4_parts(int batch, int heads, int kv_heads, long longest);
// Columns of a product that a query head has (attend4.hpp), and 16s of keys a tile.
constexpr int copies4(int per) { return per <= 4 ? 4 : per <= 8 ? 2 : 1; }
constexpr int halves4(int copies) { return copies == 4 ? 4 : 2; }
template <bool TWO, int CP>
hipError_t launch_attention4(Attend4Args &a, hipStream_t s);
hipError_t launch_kv4_attention(Attend4Args a, hipStream_t s);

// Beam search: the choice over beams and vocabulary.
constexpr int kMostBeams = 128, kMostKeep = 128;
struct SelectArgs {
  const void *logits;
  long stride;
  const float *scores;
  const uint8_t *ended;  // NULL: none
  float *out_scores;
  int *parents, *tokens;
  uint8_t *out_ended;  // NULL: not wanted
  int end;             // -1: none
  int batch, beams, vocab, keep;
  int parts, chunk;  // of a row: chunk values a part
  uint64_t *keys;    // [row][part][keep]: a part's best, the best first, 0 past the last
  float *stats;      // [row][part]: largest, sum of exponentials
};
struct SelectParts {
  int parts, chunk;
};
SelectParts select_parts(long rows, int vocab);
hipError_t launch_beam_select(const SelectArgs &a, int type, hipStream_t s);

// Beam search: the reordering of caches and states. A plane is part of a cache
// whose tokens have `bytes` each a head.
struct Plane {
  char *base;
  long page_stride, token_stride, head_stride;  // bytes
  int heads, bytes;
};
struct BeamState {
  const char *from;
  char *to;
  long bytes, from_stride, to_stride;
};
constexpr int kMostPlanes = 56, kMostStates = 16;
struct ReorderArgs {
  Plane planes[kMostPlanes];
  BeamState states[kMostStates];
  int n_planes, n_states, splits, state_splits;  // splits: workgroups a plane (a state) and row
  int tables;                      // whether this launch has the tables
  int whole4;                      // tokens are copied by fours
  const int *parents, *table, *lengths, *spare;
  int *table_out, *spare_out;
  long table_width;
  int rows, beams, pages;
  Divide by_page, by_beams;
};
hipError_t launch_beam_reorder(const ReorderArgs &a, hipStream_t s);

}  // namespace ppocr
