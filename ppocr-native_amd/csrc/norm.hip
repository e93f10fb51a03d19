// Root-mean-square norm with the residual's addition, 16- or 32-bit or 8-bit
// output (ppocr_hip_rms_norm).
//
//   h = round(x + residual),  r = 1 / sqrt(mean(h^2) + eps),  y = h r w
//
// One pass over the data: L lanes hold a row in registers (CH runs of V
// consecutive values a lane, V * size = 16 bytes, run i at (i L + lane) V),
// so x and residual are read once and sum and y written once: memory bound
// (8192 rows of 8192 in bf16 with the residual: 99 us, 5.4 TB/s, in 16 bits; 98
// to 106 us, 4.5 TB/s and more, in 8).
// The 8-bit forms take the largest |y| of a group as integers of its bits, so
// that an infinity or NaN wins; a group of 32, 64 or 128 lies in neighbouring
// lanes of one run.
#include "decoder.hpp"

namespace ppocr {
namespace {

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xF, 0xF, false);
}

// The largest of each 4, 8, 16, 32 or 64 neighbouring lanes, in all of them.
__device__ __forceinline__ uint32_t lanes_max(uint32_t v, int lanes) {
  v = max(v, dpp<0xB1>(v));                    // lane ^ 1
  v = max(v, dpp<0x4E>(v));                    // lane ^ 2
  if (lanes >= 8) v = max(v, dpp<0x141>(v));   // lane i <-> 7 - i of 8
  if (lanes >= 16) v = max(v, dpp<0x140>(v));  // lane i <-> 15 - i of 16
  if (lanes >= 32) v = max(v, (uint32_t)__shfl_xor((int)v, 16));
  if (lanes >= 64) v = max(v, (uint32_t)__shfl_xor((int)v, 32));
  return v;
}

// The sum (or the largest) over the L lanes of a row; every lane gets it.
// A row of one wave needs no LDS.
template <int L>
__device__ __forceinline__ float row_sum(float v, float *lds) {
  v = wave_sum(v);
  if constexpr (L > 64) {
    if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int i = 0; i < L / 64; i++) v += lds[i];
  }
  return v;
}

template <int L>
__device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t *lds) {
  v = lanes_max(v, 64);
  if constexpr (L > 64) {
    if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int i = 0; i < L / 64; i++) v = max(v, lds[i]);
  }
  return v;
}

// 1 / sqrt(v), to a step of f32 (the instruction takes normal numbers).
__device__ __forceinline__ float inverse_root(float v) {
  return v > 1e-37f ? __builtin_amdgcn_rsqf(v) : 1.0f / sqrtf(v);
}

// A group's scale from the bits of its largest |y|, and what to multiply y
// with: 0 for a group whose scale would not be a normal number. Not finite:
// NaN.
__device__ __forceinline__ float scale8(uint32_t top, int i8, float &inverse) {
  if (top >= 0x7f800000u) {
    inverse = 0.0f;
    return __uint_as_float(0x7fc00000u);
  }
  const float s = __uint_as_float(top) * (i8 ? 1.0f / 127.0f : 1.0f / 448.0f);
  inverse = s >= 1.17549435e-38f ? __builtin_amdgcn_rcpf(s) : 0.0f;  // (a step of f32)
  return s >= 1.17549435e-38f ? s : 0.0f;
}

// N values to their codes, four a dword. `scale` NaN: the NaN code (E4M3) or 0.
template <int N>
__device__ __forceinline__ void codes8(const float (&y)[N], float inverse, float scale, int i8, uint32_t (&out)[N / 4]) {
  const bool bad = scale != scale;
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    uint32_t w;
    if (i8) {
      w = 0;
#pragma unroll
      for (int e = 0; e < 4; e++)
        w |= (uint32_t)((int)rintf(__builtin_amdgcn_fmed3f(y[i + e] * inverse, -127.0f, 127.0f)) & 255) << 8 * e;
      out[i / 4] = bad ? 0 : w;
    } else {
      float c[4];
#pragma unroll
      for (int e = 0; e < 4; e++) c[e] = __builtin_amdgcn_fmed3f(y[i + e] * inverse, -448.0f, 448.0f);
      w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false);
      w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], (int)w, true);
      out[i / 4] = bad ? 0x7f7f7f7fu : w;
    }
  }
}

template <int N>
__device__ __forceinline__ void store_codes(uint8_t *p, long have, const uint32_t (&w)[N / 4]) {
  if (have >= N) {
    __builtin_memcpy(p, w, N);
  } else {
#pragma unroll
    for (int i = 0; i < N; i++)
      if (i < have) p[i] = (uint8_t)(w[i / 4] >> 8 * (i % 4));
  }
}

// L lanes a row: 64 (four rows a workgroup) or the whole workgroup. A vector a
// lane (CH 1) wherever 1024 lanes hold a row: 8192 x 8192 of bf16 with the
// residual ran at 4.2 TB/s with four vectors a lane, 4.7 with two, 5.2 with
// one.
template <int T, bool Y8, int L, int CH>
__global__ __launch_bounds__(L == 64 ? 256 : L) void rms_norm_rows(NormArgs a, int i8) {
  typedef num_t<T> V;
  constexpr int N = 16 / sizeof(V);
  __shared__ float lds[32];
  __shared__ uint32_t lds_top[32];
  const int lane = threadIdx.x % L;
  const long row = (long)blockIdx.x * (L == 64 ? 4 : 1) + (L == 64 ? threadIdx.x / 64 : 0);
  if (row >= a.rows) return;  // whole waves; only where a row is one wave
  const V *x = (const V *)a.x + row * a.x_stride;
  const V *w = (const V *)a.weight;
  V hv[CH][N], wv[CH][N];
  float h[CH][N];
#pragma unroll
  for (int i = 0; i < CH; i++) load_n(x + (i * L + lane) * N, (long)a.c - (i * L + lane) * N, hv[i]);
  if (a.residual) {
    const V *r = (const V *)a.residual + row * a.residual_stride;
    V rv[CH][N];
#pragma unroll
    for (int i = 0; i < CH; i++) load_n(r + (i * L + lane) * N, (long)a.c - (i * L + lane) * N, rv[i]);
#pragma unroll
    for (int i = 0; i < CH; i++)
#pragma unroll
      for (int e = 0; e < N; e++) hv[i][e] = Num<T>::put(Num<T>::get(hv[i][e]) + Num<T>::get(rv[i][e]));
  }
#pragma unroll
  for (int i = 0; i < CH; i++) load_n(w + (i * L + lane) * N, (long)a.c - (i * L + lane) * N, wv[i]);
  if (a.sum) {
    V *s = (V *)a.sum + row * a.sum_stride;
#pragma unroll
    for (int i = 0; i < CH; i++) store_n(s + (i * L + lane) * N, (long)a.c - (i * L + lane) * N, hv[i]);
  }
  float q = 0.0f;
#pragma unroll
  for (int i = 0; i < CH; i++)
#pragma unroll
    for (int e = 0; e < N; e++) {
      h[i][e] = Num<T>::get(hv[i][e]);
      q = fmaf(h[i][e], h[i][e], q);
    }
  q = row_sum<L>(q, lds);
  const float r = inverse_root(fmaf(q, a.inverse_c, a.eps));
#pragma unroll
  for (int i = 0; i < CH; i++)
#pragma unroll
    for (int e = 0; e < N; e++) h[i][e] = h[i][e] * r * Num<T>::get(wv[i][e]);
  if constexpr (!Y8) {
    V *y = (V *)a.y + row * a.y_stride;
#pragma unroll
    for (int i = 0; i < CH; i++) {
      V o[N];
#pragma unroll
      for (int e = 0; e < N; e++) o[e] = Num<T>::put(h[i][e]);
      store_n(y + (i * L + lane) * N, (long)a.c - (i * L + lane) * N, o);
    }
  } else {
    uint8_t *y = (uint8_t *)a.y + row * a.y_stride;
    float *scales = a.scales + row * a.groups;
    uint32_t top[CH], all = 0;
#pragma unroll
    for (int i = 0; i < CH; i++) {
      top[i] = 0;
#pragma unroll
      for (int e = 0; e < N; e++)  // (past the row's end 0, or NaN where the whole row is)
        top[i] = max(top[i], __float_as_uint(h[i][e]) & 0x7fffffffu);
      all = max(all, top[i]);
    }
    const bool whole = a.groups == 1;
    if (whole) all = row_max<L>(all, lds_top);
#pragma unroll
    for (int i = 0; i < CH; i++) {
      const int at = (i * L + lane) * N;
      float inverse;
      const float s = scale8(whole ? all : lanes_max(top[i], a.group / N), i8, inverse);
      if (whole ? i == 0 && lane == 0 : at < a.c && at % a.group == 0) scales[whole ? 0 : at / a.group] = s;
      uint32_t o[N / 4];
      codes8(h[i], inverse, s, i8, o);
      store_codes<N>(y + at, (long)a.c - at, o);
    }
  }
}

// Rows too long for registers: 1024 lanes walk the row twice (8-bit rows with
// one scale: three times), reading h again from sum, or from x and residual.
template <int T, bool Y8>
__global__ __launch_bounds__(1024) void rms_norm_long(NormArgs a, int i8) {
  typedef num_t<T> V;
  constexpr int N = 16 / sizeof(V), L = 1024;
  __shared__ float lds[32];
  __shared__ uint32_t lds_top[32];
  const long row = blockIdx.x;
  const V *x = (const V *)a.x + row * a.x_stride;
  const V *res = a.residual ? (const V *)a.residual + row * a.residual_stride : nullptr;
  const V *w = (const V *)a.weight;
  V *sum = a.sum ? (V *)a.sum + row * a.sum_stride : nullptr;
  const int lane = threadIdx.x, runs = (a.c + L * N - 1) / (L * N);
  auto load_h = [&](int at, V(&v)[N], bool first) {
    if (!first && sum) {  // this lane's own stores
      load_n((const V *)sum + at, (long)a.c - at, v);
      return;
    }
    load_n(x + at, (long)a.c - at, v);
    if (res) {
      V rv[N];
      load_n(res + at, (long)a.c - at, rv);
#pragma unroll
      for (int e = 0; e < N; e++) v[e] = Num<T>::put(Num<T>::get(v[e]) + Num<T>::get(rv[e]));
    }
  };
  float q = 0.0f;
  for (int i = 0; i < runs; i++) {
    const int at = (i * L + lane) * N;
    V v[N];
    load_h(at, v, true);
    if (sum) store_n(sum + at, (long)a.c - at, v);
#pragma unroll
    for (int e = 0; e < N; e++) q = fmaf(Num<T>::get(v[e]), Num<T>::get(v[e]), q);
  }
  q = row_sum<L>(q, lds);
  const float r = inverse_root(fmaf(q, a.inverse_c, a.eps));
  auto load_y = [&](int at, float(&y)[N]) {
    V v[N], wv[N];
    load_h(at, v, false);
    load_n(w + at, (long)a.c - at, wv);
#pragma unroll
    for (int e = 0; e < N; e++) y[e] = Num<T>::get(v[e]) * r * Num<T>::get(wv[e]);
  };
  auto top_of = [&](int at, const float(&y)[N]) {
    uint32_t t = 0;
#pragma unroll
    for (int e = 0; e < N; e++)
      if (at + e < a.c) t = max(t, __float_as_uint(y[e]) & 0x7fffffffu);
    return t;
  };
  uint32_t all = 0;
  const bool whole = a.groups == 1;
  if constexpr (Y8) {
    if (whole) {
      for (int i = 0; i < runs; i++) {
        float y[N];
        load_y((i * L + lane) * N, y);
        all = max(all, top_of((i * L + lane) * N, y));
      }
      all = row_max<L>(all, lds_top);
    }
  }
  for (int i = 0; i < runs; i++) {
    const int at = (i * L + lane) * N;
    float y[N];
    load_y(at, y);
    if constexpr (!Y8) {
      V o[N];
#pragma unroll
      for (int e = 0; e < N; e++) o[e] = Num<T>::put(y[e]);
      store_n((V *)a.y + row * a.y_stride + at, (long)a.c - at, o);
    } else {
      float inverse;
      const float s = scale8(whole ? all : lanes_max(top_of(at, y), a.group / N), i8, inverse);
      float *scales = a.scales + row * a.groups;
      if (whole ? at == 0 : at < a.c && at % a.group == 0) scales[whole ? 0 : at / a.group] = s;
      uint32_t o[N / 4];
      codes8(y, inverse, s, i8, o);
      store_codes<N>((uint8_t *)a.y + row * a.y_stride + at, (long)a.c - at, o);
    }
  }
}

template <int T, bool Y8>
hipError_t launch_some(const NormArgs &a, int i8, hipStream_t s) {
  constexpr int N = 16 / sizeof(num_t<T>);
  const int vecs = (a.c + N - 1) / N;  // 16-byte vectors a row
#define NORM(L, CH)                                                                                         \
  return launch_kernel(rms_norm_rows<T, Y8, L, CH>, dim3(unsigned(L == 64 ? (a.rows + 3) / 4 : a.rows)), \
                       dim3(L == 64 ? 256 : L), 0, s, a, i8)
  if (vecs <= 64) NORM(64, 1);
  if (vecs <= 128) NORM(128, 1);
  if (vecs <= 256) NORM(256, 1);
  if (vecs <= 512) NORM(512, 1);
  if (vecs <= 1024) NORM(1024, 1);
  if (vecs <= 2048) NORM(1024, 2);
  if (vecs <= 4096) NORM(1024, 4);
#undef NORM
  return launch_kernel(rms_norm_long<T, Y8>, dim3(unsigned(a.rows)), dim3(1024), 0, s, a, i8);
}

// A launch has fewer than 2^32 threads: 2^21 rows at a time.
template <int T, bool Y8>
hipError_t launch(NormArgs a, int i8, hipStream_t s) {
  constexpr long most = 1L << 21;
  constexpr size_t size = sizeof(num_t<T>), y_size = Y8 ? 1 : size;
  auto on = [](auto *p, long rows, long stride, size_t each) { return p ? (char *)p + rows * stride * (long)each : nullptr; };
  for (long left = a.rows; left > 0; left -= most) {
    a.rows = left < most ? left : most;
    const hipError_t e = launch_some<T, Y8>(a, i8, s);
    if (e != hipSuccess || left <= most) return e;
    a.x = on(a.x, most, a.x_stride, size), a.residual = on(a.residual, most, a.residual_stride, size);
    a.sum = on(a.sum, most, a.sum_stride, size), a.y = on(a.y, most, a.y_stride, y_size);
    a.scales = (float *)on(a.scales, most, a.groups, 4);
  }
  return hipSuccess;
}

}  // namespace

hipError_t launch_rms_norm(const NormArgs &a, int type, int y_type, hipStream_t s) {
  const bool y8 = y_type == PPOCR_E4M3 || y_type == PPOCR_I8;
  const int i8 = y_type == PPOCR_I8;
  switch (type) {
    case PPOCR_F32: return y8 ? launch<PPOCR_F32, true>(a, i8, s) : launch<PPOCR_F32, false>(a, i8, s);
    case PPOCR_BF16: return y8 ? launch<PPOCR_BF16, true>(a, i8, s) : launch<PPOCR_BF16, false>(a, i8, s);
    case PPOCR_F16: return y8 ? launch<PPOCR_F16, true>(a, i8, s) : launch<PPOCR_F16, false>(a, i8, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace ppocr
