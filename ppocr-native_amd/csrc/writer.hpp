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
  Divide by_unit;
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
  Divide by_unit;
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
};
PagedParts kv4_parts(int batch, int heads, int kv_heads, long longest);
hipError_t launch_kv4_attention_16(const Attend4Args &a, hipStream_t s);
hipError_t launch_kv4_attention_32(const Attend4Args &a, hipStream_t s);
hipError_t launch_kv4_join(const Attend4Args &a, hipStream_t s);

}  // namespace ppocr
