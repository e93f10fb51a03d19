// Attention over a cache in 4 bits, of bf16 and f16 queries; the join of a
// split cache's parts, and how many there are.
#include "attend4.hpp"

namespace ppocr {
namespace {

constexpr int kMostParts4 = 128;

// Joins a row's parts, a workgroup a head of a text: lane i of each wave has
// parts i and i + 64's factors, wave w adds parts w, w + 4, ... of them.
// J: 64s of dim, rounded up to a power of two.
template <int J>
__global__ __launch_bounds__(256) void kv4_attention_join(Attend4Args a) {
  __shared__ float lds_o[4][256], lds_f[kMostParts4];
  const int head = blockIdx.x, b = blockIdx.y, lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int length = a.c.lengths[b];
  const Seen s = seen_of(length > a.c.table_width * a.c.page_size ? 0 : length, a.window, a.sinks, kKeys4);
  const int each = tiles_a_part(s.tiles, a.each, a.splits);
  const int parts = max(1, (s.tiles + each - 1) / each), dim = a.c.dim, row = dim + 2, far = lane + 64;
  const float *p = a.part + ((long)b * a.heads + head) * a.splits * row;
  const float b0 = lane < parts ? p[(long)lane * row] : -INFINITY, l0 = lane < parts ? p[(long)lane * row + 1] : 0.0f;
  const float b1 = far < parts ? p[(long)far * row] : -INFINITY, l1 = far < parts ? p[(long)far * row + 1] : 0.0f;
  float base = fmaxf(b0, b1);
#pragma unroll
  for (int o = 32; o; o >>= 1) base = fmaxf(base, __shfl_xor(base, o));
  // A part's base is -infinity only where nothing of it is seen (or a seen page
  // does not exist: then its sum is NaN, and so is the whole).
  auto factor = [&](float bi, float li) {
    return bi == -INFINITY ? (li == 0.0f ? 0.0f : 1.0f) : __builtin_amdgcn_exp2f(bi - base);
  };
  const float f0 = factor(b0, l0), f1 = factor(b1, l1);
  float sum = f0 * l0 + f1 * l1;
#pragma unroll
  for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
  if (wave == 0) lds_f[lane] = f0, lds_f[far] = f1;
  __syncthreads();
  float o[J] = {};
#pragma unroll 8
  for (int i = wave; i < parts; i += 4) {
    const float f = lds_f[i];
#pragma unroll
    for (int j = 0; j < J; j++)  // (past dim: its last value, not kept)
      o[j] = fmaf(f, p[(long)i * row + 2 + min(lane + 64 * j, dim - 1)], o[j]);
  }
#pragma unroll
  for (int j = 0; j < J; j++) lds_o[wave][lane + 64 * j] = o[j];
  __syncthreads();
  const int d = threadIdx.x;
  if (d < dim) {
    const float v = (lds_o[0][d] + lds_o[1][d]) + (lds_o[2][d] + lds_o[3][d]);
    put_at(a.y, b * a.y_stride + (long)head * dim + d, a.type, sum == 0.0f ? 0.0f : v / sum);
  }
}

}  // namespace

PagedParts kv4_parts(int batch, int heads, int kv_heads, long longest) {
  // As the plain cache's parts of 32 keys a tile.
  return paged_parts(batch, heads, kv_heads, PPOCR_BF16, longest);
}

hipError_t launch_kv4_join(const Attend4Args &a, hipStream_t s) {
  const dim3 grid(a.heads, a.batch), block(256);
  if (a.c.dim <= 64) return launch_kernel(kv4_attention_join<1>, grid, block, 0, s, a);
  if (a.c.dim <= 128) return launch_kernel(kv4_attention_join<2>, grid, block, 0, s, a);
  return launch_kernel(kv4_attention_join<4>, grid, block, 0, s, a);
}

hipError_t launch_kv4_attention_16(const Attend4Args &a, hipStream_t s) { return launch_attention4<false>(a, s); }

}  // namespace ppocr
