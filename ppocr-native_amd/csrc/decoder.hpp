// The decoder layers' number types, launch arguments and launchers.
//
// A tensor's rows are `*_stride` values apart; types are the codes of
// include/ppocr_hip.h. Launchers return a hipError_t from the launch; they
// never synchronise or allocate. Shapes are checked by the C entries
// (decoder.cpp).
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <atomic>

#include "ppocr_hip.h"

namespace ppocr {

// A launch whose own status is returned: the thread's last error may be that
// of another call.
template <class... P>
hipError_t launch_kernel(void (*kernel)(P...), dim3 grid, dim3 block, int lds, hipStream_t s, P... args) {
  void *at[] = {&args...};
  return hipLaunchKernel((const void *)kernel, grid, block, at, size_t(lds), s);
}

// Allows `bytes` of LDS to a kernel on the current device: once, for always the
// same number.
template <auto Kernel>
hipError_t allow_lds_of(int bytes) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return e;
  const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
  if (done.load(std::memory_order_acquire) & bit) return hipSuccess;
  e = hipFuncSetAttribute((const void *)Kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == hipSuccess) done.fetch_or(bit, std::memory_order_release);
  return e;
}

typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

// One number type: its values as floats and back (nearest, ties to even).
template <int T>
struct Num;
template <>
struct Num<PPOCR_F32> {
  typedef float type;
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
};
template <>
struct Num<PPOCR_BF16> {
  typedef __bf16 type;
  static __device__ __forceinline__ float get(__bf16 v) { return (float)v; }
  static __device__ __forceinline__ __bf16 put(float v) { return (__bf16)v; }
};
template <>
struct Num<PPOCR_F16> {
  typedef _Float16 type;
  static __device__ __forceinline__ float get(_Float16 v) { return (float)v; }
  static __device__ __forceinline__ _Float16 put(float v) { return (_Float16)v; }
};
template <int T>
using num_t = typename Num<T>::type;

// N values at p (any alignment of a value's own size), or the first `have`
// of them and zeros. Whole vectors are one load: global loads take any
// alignment here.
template <typename V, int N>
__device__ __forceinline__ void load_n(const V *p, long have, V (&v)[N]) {
  if (have >= N) {
    __builtin_memcpy(v, p, sizeof v);
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) {
      v[i] = V(0);
      if (i < have) v[i] = p[i];
    }
  }
}

template <typename V, int N>
__device__ __forceinline__ void store_n(V *p, long have, const V (&v)[N]) {
  if (have >= N) {
    __builtin_memcpy(p, v, sizeof v);
  } else {
#pragma unroll
    for (int i = 0; i < N; i++)
      if (i < have) p[i] = v[i];
  }
}

struct NormArgs {
  const void *x, *residual, *weight;
  void *sum, *y;
  float *scales;
  long x_stride, residual_stride, sum_stride, y_stride;
  long rows;
  int c, groups, group;  // group: values a scale covers (c: the whole row)
  float eps, inverse_c;
};
hipError_t launch_rms_norm(const NormArgs &a, int type, int y_type, hipStream_t s);

struct Q4Args {
  const void *x;
  const float *x_scales;
  const uint8_t *q;
  const void *scales;
  const uint8_t *zeros;
  const void *bias;
  void *y;
  long x_stride, y_stride;
  int m, n, k, group, groups;
  int x_group;  // 0: one scale a row of x (8-bit x)
  int scale_type, y_type;
};
// The 4-bit product's workgroups: up to kQ4Waves waves, each of which takes
// kQ4Stretch inputs at a time, and as few tiles of 16 outputs as all workgroups
// run at once with: 1, 2 or 4, and 8 of f32 rows (18385 outputs of 1024 inputs
// from 5 rows of f32: 288 workgroups 13.9 us, 144 of them 11.0). With more tiles
// than that they run one after another, by fours. Rows of 16 and 8 bits stop at
// four tiles: with eight, 4096 inputs to 40000 outputs took 28.7 us instead of 25
// for one row of bf16 (16 rows 33.3 and 33.7, 32 rows to 28672 outputs 34 and 41).
constexpr int kQ4Waves = 8, kQ4Stretch = 128;
inline int q4_waves(int k) {
  int waves = kQ4Waves;
  while (waves > 1 && waves / 2 * kQ4Stretch >= k) waves /= 2;
  return waves;
}
// Workgroups of kQ4Waves that the card holds at once, by their registers.
constexpr int q4_at_once(int x_type) { return x_type == PPOCR_F32 ? 256 : 512; }
inline int q4_tiles(int x_type, int m, int n, int k) {
  const long tiles = (n + 15L) / 16 * ((m + 15) / 16), at_once = q4_at_once(x_type) * (kQ4Waves / q4_waves(k));
  if (tiles <= at_once) return 1;
  if (tiles <= 2 * at_once) return 2;
  return x_type == PPOCR_F32 && tiles > 4 * at_once && tiles <= 8 * at_once ? 8 : 4;
}
hipError_t launch_q4_f32(const Q4Args &a, int, hipStream_t s);
hipError_t launch_q4_bf16(const Q4Args &a, int, hipStream_t s);
hipError_t launch_q4_f16(const Q4Args &a, int, hipStream_t s);
hipError_t launch_q4_i8(const Q4Args &a, int e4m3, hipStream_t s);

// Division of 0 .. 2^31 - 1 by d: n / d = n mul >> shift.
struct Divide {
  uint32_t mul;
  int shift, d;
  Divide(int by = 1) : d(by) {
    int l = 0;
    while ((int64_t(1) << l) < by) l++;
    shift = 31 + l;
    mul = uint32_t(((uint64_t(1) << shift) + by - 1) / by);
  }
  __device__ __forceinline__ int operator()(int n) const { return int((uint64_t)(uint32_t)n * mul >> shift); }
};

struct CacheArgs {
  void *k, *v;
  long page_stride, token_stride, head_stride;
  int pages, page_size, heads, dim;
  Divide by_page;
  const int *table;
  long table_width;
  const int *lengths;
};

struct AppendArgs {
  CacheArgs c;
  const void *k, *v;
  long k_stride, v_stride;
  const int *starts;  // NULL: one row a text
  long rows;
  int batch;
};
hipError_t launch_kv_append(const AppendArgs &a, int type, hipStream_t s);

struct PagedArgs {
  CacheArgs c;
  const void *q;
  void *y;
  long q_stride, y_stride;
  int batch, heads;
  int splits, each;  // parts of a text at most, and tiles of one at least
  int window, sinks;  // window 0: every key is seen
  float scale;        // of 2-logarithms, positive
  bool turn;          // the given scale was negative: q turns its sign
  float *part;  // splits > 1: batch x heads x splits rows of dim + 2 floats
};
// The parts a text's cache of up to `longest` seen tokens is split into.
struct PagedParts {
  int splits, each;
};
PagedParts paged_parts(int batch, int heads, int kv_heads, int type, long longest);
hipError_t launch_paged_attention(const PagedArgs &a, int type, hipStream_t s);

struct PromptArgs {
  const void *q, *k, *v;
  void *y;
  const int *starts_q, *starts_k;
  long q_stride, k_stride, v_stride, y_stride;
  int batch, rows_q, rows_k, heads, kv_heads, dim;
  int window, sinks;
  float scale;
  bool turn;
};
hipError_t launch_window_attention(const PromptArgs &a, int type, hipStream_t s);

}  // namespace ppocr
