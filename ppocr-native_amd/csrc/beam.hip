// Beam search: the choice of the best continuations over beams and vocabulary
// (ppocr_hip_beam_select) and the reordering of caches and states after it
// (ppocr_hip_beam_reorder).
//
//   score(i, v) = scores_i + (x_iv - max_i) - log(sum over v of exp(x_iv - max_i))
//
// Within a beam the order of scores is that of the logits, so one pass over
// them gives each part of a row its largest value, its sum of exponentials and
// its `keep` best; a workgroup a text then has the beams' logarithms and
// chooses among the parts' best, in f64, so that scores of different beams that
// differ at all are told apart. Numbers to be ordered carry their position in
// their low bits, the lower one the larger: no two are equal, and the result
// does not depend on the order in which workgroups or lanes come to them.
#include <algorithm>

#include "writer.hpp"

namespace ppocr {
namespace {

// Floats and doubles as numbers that are ordered as they are.
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t u = __float_as_uint(v);
  return u ^ (u >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t u) {
  return __uint_as_float(u ^ (u >> 31 ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ uint64_t ordered(double v) {
  const uint64_t u = (uint64_t)__double_as_longlong(v);
  return u ^ (u >> 63 ? ~uint64_t(0) : uint64_t(1) << 63);
}
__device__ __forceinline__ double unordered(uint64_t u) {
  return __longlong_as_double((long long)(u ^ (u >> 63 ? uint64_t(1) << 63 : ~uint64_t(0))));
}

__device__ __forceinline__ uint64_t shuffled(uint64_t v, int o) {
  return (uint64_t)(uint32_t)__shfl_xor((int)(v >> 32), o) << 32 | (uint32_t)__shfl_xor((int)v, o);
}

__device__ __forceinline__ float exp_of(float v) { return __builtin_amdgcn_exp2f(v * 1.44269504088896340736f); }

// ---------------------------------------------------------------- a row's parts

constexpr int kThreads = 256, kList = 1024;
constexpr float kLowest = -3.402823466e38f;  // a bound that only -infinity, which is never chosen, is below

// Lanes of a group, of `used` threads that have values: as many as leave `groups`
// of them, up to a wave.
__host__ __device__ inline int lanes_of(int used, int groups) {
  int lanes = 64;
  while (lanes > 1 && used / lanes < groups) lanes /= 2;
  return lanes;
}

// How many of n numbers (at 16 bytes, three of -infinity or more behind them) come
// before number `at` of them, `mine`: larger ones, and equal ones before it.
__device__ __forceinline__ int rank_of(const float *numbers, int n, float mine, int at) {
  int rank = 0;
  for (int i = 0; i < n; i += 4) {
    const v4f of = *(const v4f *)(numbers + i);
#pragma unroll
    for (int j = 0; j < 4; j++) rank += of[j] > mine || (of[j] == mine && i + j < at);
  }
  return rank;
}

// The `keep` largest of a workgroup's numbers: those past a bound that at least
// `keep` are not below, which is the `keep`-th of twice as many groups' largest,
// gathered in LDS and ranked there. Of shuffled numbers that leaves a few times
// `keep`; where more than LDS holds (sorted ones, or equal ones), the bound is
// halved in on. What costs is arithmetic: eight instructions a value, four of them the
// exponential's, come to 250 of a wave's 580, and the bound, the list's pushes and
// its ranks to the others: 256 rows of 131072 in bf16, 30 % of them ended, take
// 18 us, 47 MB at 2.6 TB/s and 80 % of the vector units' time; four rows of 18385 in
// f32 take 4.8.
// R: rounds of 8 values a thread. FEW: rows of fewer than 8 values.
template <int T, int R, bool FEW>
__global__ __launch_bounds__(kThreads) void beam_parts(SelectArgs a) {
  typedef num_t<T> V;
  __shared__ __attribute__((aligned(16))) uint64_t list[kList + 4];
  __shared__ __attribute__((aligned(16))) float lds_group[kThreads + 4];
  __shared__ float lds_top[4], lds_sum[4], lds_bound;
  __shared__ int lds_n[4], lds_count;
  const int row = blockIdx.x / a.parts, part = blockIdx.x - row * a.parts;
  // Beams that have no score to go on from, or have ended, need no logits.
  const float score = a.scores[row];
  int over = 0;
  if (a.ended) over = a.ended[row];
  if (!(score > -INFINITY) || over) return;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int begin = part * a.chunk, end = min(begin + a.chunk, a.vocab);
  const V *p = (const V *)a.logits + row * a.stride;

  // Round r's piece: values at_of(r) .. at_of(r) + 7; the last one begins where the row still has eight, and its
  // first values are the piece's before it. (Nothing is read behind a branch, which would be waited for.)
  V raw[R][8];
  const int last = max(a.vocab - 8, 0);
  const auto at_of = [&](int r) { return min(begin + (r * kThreads + (int)threadIdx.x) * 8, last); };
#pragma unroll
  for (int r = 0; r < R; r++) {
    if constexpr (FEW) {
      for (int j = 0; j < 8; j++) raw[r][j] = p[min(at_of(r) + j, a.vocab - 1)];
    } else {
      __builtin_memcpy(raw[r], p + at_of(r), sizeof raw[r]);
    }
  }
  float x[R][8], top = -INFINITY;
#pragma unroll
  for (int r = 0; r < R; r++)
#pragma unroll
    for (int j = 0; j < 8; j++) x[r][j] = Num<T>::get(raw[r][j]);
  if (end - begin != R * kThreads * 8) {  // a row's last part
#pragma unroll
    for (int r = 0; r < R; r++) {
      const int first = begin + (r * kThreads + (int)threadIdx.x) * 8 - at_of(r), have = end - at_of(r);
#pragma unroll
      for (int j = 0; j < 8; j++) x[r][j] = j >= first && j < have ? x[r][j] : -INFINITY;
    }
  }
#pragma unroll
  for (int r = 0; r < R; r++)
#pragma unroll
    for (int j = 0; j < 8; j++) top = fmaxf(top, x[r][j]);
  const auto key_of = [&](int r, int j) {  // (-0 is 0)
    return (uint64_t)ordered(x[r][j] + 0.0f) << 32 | ~(uint32_t)(at_of(r) + j);
  };
  // The largest, and the bound: of groups of lanes the largest, of those the `keep`-th.
  const int used = (min(end - begin, kThreads * 8) + 7) / 8, lanes = lanes_of(used, 2 * a.keep);
  const int groups = (used + lanes - 1) / lanes;  // (those past it have nothing)
  float most = top;
  for (int o = 1; o < lanes; o *= 2) most = fmaxf(most, __shfl_xor(most, o));
  top = most;
  for (int o = lanes; o < 64; o *= 2) top = fmaxf(top, __shfl_xor(top, o));
  if (lane % lanes == 0) lds_group[threadIdx.x / lanes] = most;
  if (threadIdx.x < 4) lds_group[groups + threadIdx.x] = -INFINITY;
  if (lane == 0) lds_top[wave] = top;
  if (threadIdx.x == 0) lds_count = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 4; w++) top = fmaxf(top, lds_top[w]);
  float bound;
  if (groups <= 64) {  // each wave for itself
    const float mine = lds_group[min(lane, groups)];
    const uint64_t is = __ballot(lane < groups && rank_of(lds_group, groups, mine, lane) == a.keep - 1 && mine > -INFINITY);
    bound = is ? __shfl(mine, __builtin_ctzll(is)) : kLowest;
  } else {
    if (threadIdx.x == 0) lds_bound = kLowest;
    __syncthreads();
    if ((int)threadIdx.x < groups) {
      const float mine = lds_group[threadIdx.x];
      if (rank_of(lds_group, groups, mine, threadIdx.x) == a.keep - 1 && mine > -INFINITY) lds_bound = mine;
    }
    __syncthreads();
    bound = lds_bound;
  }
  // Which of a thread's values are past it, a bit each; their values are read once more, where there are any.
  const auto push = [&](uint64_t key) {
    const int at = atomicAdd(&lds_count, 1);
    if (at < kList) list[at] = key;
  };
  uint32_t past = 0;
#pragma unroll
  for (int r = 0; r < R; r++)
#pragma unroll
    for (int j = 0; j < 8; j++) past = past + past + (x[r][j] >= bound ? 1u : 0u);
  while (past) {
    const int bit = __builtin_ctz(past), k = 8 * R - 1 - bit;
    past &= past - 1;
    const int at = at_of(k / 8) + k % 8;
    push((uint64_t)ordered(Num<T>::get(p[at]) + 0.0f) << 32 | ~(uint32_t)at);
  }

  // The sum of exponentials.
  const float from = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f;
#pragma unroll
  for (int r = 0; r < R; r++)
#pragma unroll
    for (int j = 0; j < 8; j++) sum += exp_of(x[r][j] - from);
#pragma unroll
  for (int o = 1; o < 64; o *= 2) sum += __shfl_xor(sum, o);
  if (lane == 0) lds_sum[wave] = sum;
  __syncthreads();
  if (lds_count > kList) {  // (the same in all threads)
    // count(low) > kList, count(high) < keep; numbers differ, so some bound
    // between leaves between `keep` and kList of them.
    uint64_t low = (uint64_t)ordered(bound) << 32, high = ((uint64_t)ordered(top + 0.0f) + 1) << 32;
    while (high - low > 1) {
      const uint64_t mid = low + (high - low) / 2;
      int n = 0;
#pragma unroll
      for (int r = 0; r < R; r++)
#pragma unroll
        for (int j = 0; j < 8; j++) n += __popcll(__ballot(key_of(r, j) >= mid));
      __syncthreads();
      if (lane == 0) lds_n[wave] = n;
      __syncthreads();
      n = lds_n[0] + lds_n[1] + lds_n[2] + lds_n[3];
      if (n > kList) {
        low = mid;
      } else if (n < a.keep) {
        high = mid;
      } else {
        low = mid;
        break;
      }
    }
    if (threadIdx.x == 0) lds_count = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
      for (int j = 0; j < 8; j++)
        if (key_of(r, j) >= low) push(key_of(r, j));
    __syncthreads();
  }
  const int n = min(lds_count, kList);
  uint64_t *out = a.keys + (long)blockIdx.x * a.keep;
  if (threadIdx.x < 4) list[n + threadIdx.x] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const uint64_t mine = list[i];
    int rank = 0;
    for (int j = 0; j < n; j += 4) rank += (list[j] > mine) + (list[j + 1] > mine) + (list[j + 2] > mine) + (list[j + 3] > mine);
    if (rank < a.keep) out[rank] = mine;
  }
  for (int i = n + threadIdx.x; i < a.keep; i += kThreads) out[i] = 0;
  if (threadIdx.x == 0) {
    a.stats[2L * blockIdx.x] = top;
    a.stats[2L * blockIdx.x + 1] = (lds_sum[0] + lds_sum[1]) + (lds_sum[2] + lds_sum[3]);
  }
}

// ------------------------------------------------------- a text's choice

constexpr int kChoices = 2048;

// A candidate: its score, ordered, and what decides where scores are equal: the
// lower beam (8 bits), the larger logit (32), the lower token (24). 0, 0: none.
struct Choice {
  uint64_t score, at;
  __device__ __forceinline__ bool operator>(const Choice &o) const {
    return score > o.score || (score == o.score && at > o.at);
  }
};

// A workgroup a text, a candidate or more a thread; `lanes` of a group.
// A chain of waits: the parts' statistics, their logarithm, the candidates (asked
// for before it), the bound, the list. Bounds of 32-bit scores, ranks by waves, and
// results written side by side took it from 12.5 to 7.5 us for 32 texts of 8 beams
// with 1024 candidates each (4 beams and 144: 6.1).
__global__ __launch_bounds__(1024) void beam_choice(SelectArgs a, int lanes, Divide by_beams) {
  __shared__ Choice list[kChoices], chosen[kMostKeep];
  __shared__ double lds_base[kMostBeams], lds_top[kMostBeams], lds_log[kMostBeams];
  __shared__ __attribute__((aligned(16))) float lds_group[1024 + 4];
  __shared__ float lds_bound;
  __shared__ int lds_live[kMostBeams], lds_n[16], lds_count;  // live: 0 no candidates, 1 its tokens, 2 ended
  const int b = blockIdx.x, threads = blockDim.x, lane = threadIdx.x % 64, wave = threadIdx.x / 64, waves = threads / 64;
  const int each = a.parts * a.keep, all = a.beams * each, count = all + a.beams;  // (at most 2^25)
  const uint64_t *keys = a.keys + (long)b * all;
  // Neighbouring threads have candidates of different beams, so that a group has some of the best beam's.
  auto key_at = [&](int c) {
    const int i = by_beams(min(c, all - 1));
    return keys[(min(c, all - 1) - i * a.beams) * each + i];
  };
  constexpr int kAhead = 4;
  uint64_t ahead[kAhead];  // of beams without candidates: whatever lies there
#pragma unroll
  for (int k = 0; k < kAhead; k++) ahead[k] = key_at((int)threadIdx.x + k * threads);
  for (int i = wave; i < a.beams; i += waves) {
    const long row = (long)b * a.beams + i;
    const float base = a.scores[row];
    const v2f *stats = (const v2f *)a.stats + row * a.parts;
    const v2f first = stats[min(lane, a.parts - 1)];  // (asked for with the score)
    int live = !(base > -INFINITY) ? 0 : a.ended && a.ended[row] ? 2 : 1;
    float top = -INFINITY;
    double sum = 0;
    if (live == 1) {
      if (lane < a.parts) top = first[0];
      for (int k = lane + 64; k < a.parts; k += 64) top = fmaxf(top, stats[k][0]);
      for (int o = 1; o < min(a.parts, 64); o *= 2) top = fmaxf(top, __shfl_xor(top, o));
      top = __shfl(top, 0);
      auto add = [&](const v2f &of) {
        sum += of[0] == -INFINITY ? (double)of[1] : (double)of[1] * (double)exp_of(of[0] - top);
      };
      if (lane < a.parts) add(first);
      for (int k = lane + 64; k < a.parts; k += 64) add(stats[k]);
      for (int o = 1; o < min(a.parts, 64); o *= 2) sum += __longlong_as_double((long long)shuffled((uint64_t)__double_as_longlong(sum), o));
      // (Of lane 0. Not so for a row of -infinity, or with an infinity or a NaN.)
      if (!(sum > 0) || !(top < INFINITY)) live = 0;
    }
    if (lane == 0) {
      lds_base[i] = (double)base, lds_top[i] = (double)top, lds_log[i] = live == 1 ? log(sum) : 0;
      lds_live[i] = live;
    }
  }
  if (threadIdx.x == 0) lds_count = 0;
  __syncthreads();
  const auto place = [](int i, uint32_t logit, uint32_t token) {
    return (uint64_t)(255 - i) << 56 | (uint64_t)logit << 24 | (0xffffffu - token);
  };
  auto choice = [&](int c, uint64_t key) -> Choice {
    if (c >= all) {
      const int i = c - all;
      return lds_live[i] == 2 ? Choice{ordered(lds_base[i] + 0.0), place(i, 0, a.end)} : Choice{0, 0};
    }
    const int i = c - by_beams(c) * a.beams;
    if (lds_live[i] != 1) return Choice{0, 0};
    if (key == 0) return Choice{0, 0};
    const double x = (double)unordered((uint32_t)(key >> 32));
    const double score = lds_base[i] + ((x - lds_top[i]) - lds_log[i]);
    if (!(score > -INFINITY)) return Choice{0, 0};
    return Choice{ordered(score + 0.0), place(i, (uint32_t)(key >> 32), ~(uint32_t)key)};
  };
  // Each thread's candidates: the first from what was asked for ahead.
  auto each_choice = [&](auto &&take) {
#pragma unroll
    for (int k = 0; k < kAhead; k++) {
      const int c = (int)threadIdx.x + k * threads;
      if (c < count) take(choice(c, ahead[k]));
    }
    for (int c = (int)threadIdx.x + kAhead * threads; c < count; c += threads) take(choice(c, key_at(c)));
  };
  // The bound: the `keep`-th largest of groups' largest, of scores rounded to 32 bits (which keeps their order).
  float best = -INFINITY;
  each_choice([&](const Choice &k) {
    if (k.score) best = fmaxf(best, (float)unordered(k.score));
  });
  for (int o = 1; o < lanes; o *= 2) best = fmaxf(best, __shfl_xor(best, o));
  const int groups = threads / lanes;
  if (lane % lanes == 0) lds_group[threadIdx.x / lanes] = best;
  if (threadIdx.x < 4) lds_group[groups + threadIdx.x] = -INFINITY;
  if (threadIdx.x == 0) lds_bound = -INFINITY;  // (too few groups: all there are)
  __syncthreads();
  if ((int)threadIdx.x < groups) {
    const float mine = lds_group[threadIdx.x];
    if (rank_of(lds_group, groups, mine, threadIdx.x) == a.keep - 1) lds_bound = mine;
  }
  __syncthreads();
  const float from = lds_bound;
  auto gather = [&](auto past) {
    each_choice([&](const Choice &k) {
      if (k.score && past(k)) {
        const int at = atomicAdd(&lds_count, 1);
        if (at < kChoices) list[at] = k;
      }
    });
  };
  gather([&](const Choice &k) { return (float)unordered(k.score) >= from; });
  __syncthreads();
  if (lds_count > kChoices) {  // (the same in all threads)
    auto count_from = [&](const Choice &bound) {
      int n = 0;
      each_choice([&](const Choice &k) { n += !(bound > k); });
#pragma unroll
      for (int o = 1; o < 64; o *= 2) n += __shfl_xor(n, o);
      __syncthreads();
      if (lane == 0) lds_n[wave] = n;
      __syncthreads();
      n = 0;
      for (int w = 0; w < waves; w++) n += lds_n[w];
      return n;
    };
    // First by scores alone, then, where too many share one, by positions.
    uint64_t low = 1, high = ordered((double)INFINITY) + 1;
    Choice bound{0, 0};
    bool done = false;
    while (high - low > 1) {
      const uint64_t mid = low + (high - low) / 2;
      const int n = count_from(Choice{mid, 0});
      if (n > kChoices) {
        low = mid;
      } else if (n < a.keep) {
        high = mid;
      } else {
        bound = Choice{mid, 0}, done = true;
        break;
      }
    }
    if (!done) {
      const uint64_t score = low;
      uint64_t below = 0, above = ~uint64_t(0);
      while (above - below > 1) {
        const uint64_t mid = below + (above - below) / 2;
        const int n = count_from(Choice{score, mid});
        if (n > kChoices) {
          below = mid;
        } else if (n < a.keep) {
          above = mid;
        } else {
          below = mid;
          break;
        }
      }
      bound = Choice{score, below};
    }
    if (threadIdx.x == 0) lds_count = 0;
    __syncthreads();
    gather([&](const Choice &k) { return !(bound > k); });
    __syncthreads();
  }
  const int n = min(lds_count, kChoices);
  const long out = (long)b * a.keep;
  for (int i = wave; i < n; i += waves) {  // a wave ranks one of them against 64 at a time
    const Choice mine = list[i];
    int rank = 0;
    for (int j = lane; j < n + lane; j += 64) rank += __popcll(__ballot(j < n && list[min(j, n - 1)] > mine));
    if (lane == 0 && rank < a.keep) chosen[rank] = mine;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.keep; i += threads) {
    const uint64_t at = i < n ? chosen[i].at : 0;
    const int parent = 255 - (int)(at >> 56), token = (int)(0xffffffu - ((uint32_t)at & 0xffffffu));
    const long to = out + i;
    a.out_scores[to] = i < n ? (float)unordered(chosen[i].score) : -INFINITY;
    a.parents[to] = i < n ? parent : min(i, a.beams - 1);
    a.tokens[to] = i < n ? token : -1;
    if (a.out_ended) a.out_ended[to] = i < n && (token == a.end || lds_live[parent] == 2);
  }
}

template <int T>
hipError_t launch_parts_of(const SelectArgs &a, hipStream_t s) {
  const dim3 grid(unsigned((long)a.batch * a.beams * a.parts)), block(kThreads);
  if (a.vocab < 8) return launch_kernel(beam_parts<T, 1, true>, grid, block, 0, s, a);
  if (a.chunk == kThreads * 8) return launch_kernel(beam_parts<T, 1, false>, grid, block, 0, s, a);
  if (a.chunk == kThreads * 16) return launch_kernel(beam_parts<T, 2, false>, grid, block, 0, s, a);
  return launch_kernel(beam_parts<T, 4, false>, grid, block, 0, s, a);
}

// -------------------------------------------------------------- the reordering

__device__ __forceinline__ v4u piece_at(const char *p, long i) {
  v4u v;
  __builtin_memcpy(&v, p + 16 * i, 16);
  return v;
}
// (As a stream: the copies of 64 rows' pages, 143 MB, take 26 us so, and 29 without.)
__device__ __forceinline__ void put_piece(char *p, long i, v4u v) {
  typedef v4u __attribute__((aligned(1))) Loose;
  __builtin_nontemporal_store(v, (Loose *)(p + 16 * i));
}

// Copies `bytes` from one place to another, a thread's share: from piece of 16
// `first` on every `step`-th.
__device__ __forceinline__ void copy_pieces(char *to, const char *from, long bytes, long first, long step) {
  const long whole = bytes / 16;
  long i = first;
  for (; i + 3 * step < whole; i += 4 * step) {
    const v4u a = piece_at(from, i), b = piece_at(from, i + step), c = piece_at(from, i + 2 * step),
              d = piece_at(from, i + 3 * step);
    put_piece(to, i, a);
    put_piece(to, i + step, b);
    put_piece(to, i + 2 * step, c);
    put_piece(to, i + 3 * step, d);
  }
  for (; i < whole; i += step) put_piece(to, i, piece_at(from, i));
  for (long k = 16 * whole + first; k < bytes; k += step) to[k] = from[k];
}

// Row (a text's beam) blockIdx.y; workgroup 0 of it has its table, the next ones
// the states, the others a split of a plane's tokens each. Memory bound where a
// page's tokens lie together (64 rows, 12 layers, 143 MB: 26 us, 5.5 TB/s, where a
// copy has 5.2; head by head: 29), or by the launch (4 rows of one layer: 3.8 us).
// Caches in 4 bits have two or four pieces of 16 bytes a head of some planes, for
// 256 threads, and their heads go one after another: the same rows, 38 to 45 MB, take
// 18 to 20 us, two launches.
__global__ __launch_bounds__(256) void beam_reorder_rows(ReorderArgs a) {
  const int row = blockIdx.y, text = a.by_beams(row);
  const int parent = a.parents[row];
  const int from = parent < 0 || parent >= a.beams ? row : text * a.beams + parent;
  int job = blockIdx.x;
  const int of_states = a.n_states * a.state_splits;
  if (a.tables && job > 0 && job <= of_states) {
    const int state = (job - 1) / a.state_splits, split = job - 1 - state * a.state_splits;
    const BeamState &s = a.states[state];
    copy_pieces(s.to + row * s.to_stride, s.from + from * s.from_stride, s.bytes, split * 256 + threadIdx.x,
                a.state_splits * 256);
    return;
  }
  if (!a.table) return;
  const int length = max(a.lengths[from], 0), full = a.by_page(length), part = length - full * a.by_page.d;
  const int *mine = a.table + row * a.table_width, *other = a.table + from * a.table_width;
  // The page being written is copied where the row has another parent.
  const bool moved = from != row;
  int source = -1, into = -1;
  if (moved && part > 0 && full < a.table_width) source = other[full], into = a.spare[row];
  const bool there = source >= 0 && source < a.pages, copied = there && into >= 0 && into < a.pages;
  if (a.tables) {
    if (job == 0) {
      for (long i = threadIdx.x; i < a.table_width; i += 256)
        a.table_out[row * a.table_width + i] = !moved || i > full || (i == full && part == 0) ? mine[i]
                                               : i < full                                     ? other[i]
                                               : there                                        ? into
                                                                                              : source;
      if (threadIdx.x == 0) a.spare_out[row] = there ? mine[full] : a.spare[row];
      return;
    }
    job -= 1 + of_states;
  }
  if (!copied) return;
  const int plane = job / a.splits, split = job - plane * a.splits;
  const Plane &p = a.planes[plane];
  const char *src = p.base + source * p.page_stride;
  char *dst = p.base + into * p.page_stride;
  const int tokens = a.whole4 ? min((part + 3) / 4 * 4, a.by_page.d) : part;
  if (p.token_stride == p.bytes) {
    for (int h = 0; h < p.heads; h++)
      copy_pieces(dst + h * p.head_stride, src + h * p.head_stride, (long)tokens * p.bytes, split * 256 + threadIdx.x,
                  a.splits * 256);
  } else {
    // A row of a head a wave at a time (at most 2^31 - 4096).
    const int lane = threadIdx.x % 64;
    for (int i = split * 4 + threadIdx.x / 64; i < tokens * p.heads; i += a.splits * 4) {
      const int token = i / p.heads, h = i - token * p.heads;
      const long at = token * p.token_stride + h * p.head_stride;
      copy_pieces(dst + at, src + at, p.bytes, lane, 64);
    }
  }
}

}  // namespace

SelectParts select_parts(long rows, int vocab) {
  // Parts of 8192 values (32 a thread), or of 4096 or 2048 where that leaves the
  // card fewer than 2048 workgroups.
  int chunk = 8192;
  while (chunk > 2048 && rows * ((vocab + chunk - 1) / chunk) < 2048) chunk /= 2;
  return {(vocab + chunk - 1) / chunk, chunk};
}

hipError_t launch_beam_select(const SelectArgs &a, int type, hipStream_t s) {
  const hipError_t e = type == PPOCR_F32    ? launch_parts_of<PPOCR_F32>(a, s)
                       : type == PPOCR_BF16 ? launch_parts_of<PPOCR_BF16>(a, s)
                       : type == PPOCR_F16  ? launch_parts_of<PPOCR_F16>(a, s)
                                            : hipErrorInvalidValue;
  if (e != hipSuccess) return e;
  const long all = (long)a.beams * a.parts * a.keep;
  const int threads = int(std::min((all + 63) / 64 * 64, 1024L));
  // (The bound once was the least of all groups' largest: 132 us for 30 beams of 30, now 22.)
  const int lanes = lanes_of(threads, std::max(2 * a.keep, 16));
  return launch_kernel(beam_choice, dim3(a.batch), dim3(threads), 0, s, a, lanes, Divide(a.beams));
}

hipError_t launch_beam_reorder(const ReorderArgs &a, hipStream_t s) {
  const dim3 grid((a.tables ? 1 + a.n_states * a.state_splits : 0) + a.n_planes * a.splits, a.rows), block(256);
  return launch_kernel(beam_reorder_rows, grid, block, 0, s, a);
}

}  // namespace ppocr
