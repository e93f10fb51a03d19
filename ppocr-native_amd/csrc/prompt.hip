// Causal attention of prompts with a sliding window and sinks
// (ppocr_hip_window_attention).
#include "attend.hpp"

namespace ppocr {
namespace {

// A block of queries: which text, and which of its rows. Blocks are counted
// through the texts; there are at most rows_q / SIZE + batch.
struct Block {
  int q0, nq;  // the text's first row of q and its queries
  int k0, nk;
  int first;  // the block's first query in its text
};

// Finds block `index`; false if there are fewer. Every wave of a workgroup
// walks the starts, 64 texts at a time. Starts past the rows there are, and
// such as decrease, leave texts of no rows.
template <int SIZE>
__device__ __forceinline__ bool find_block(const PromptArgs &a, int index, Block &out) {
  const int lane = threadIdx.x % 64;
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    const int b = b0 + lane;
    int q0 = 0, nq = 0;
    if (b < a.batch) {
      q0 = min(max(a.starts_q[b], 0), a.rows_q);
      nq = max(min(a.starts_q[b + 1], a.rows_q) - q0, 0);
    }
    const int blocks = (nq + SIZE - 1) / SIZE;
    int upto = blocks;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(upto, o);
      if (lane >= o) upto += v;
    }
    const unsigned long long past = __ballot(upto > index);
    if (past) {
      const int at = __ffsll(past) - 1;
      out.q0 = __shfl(q0, at);
      out.nq = __shfl(nq, at);
      out.first = (index - (__shfl(upto, at) - __shfl(blocks, at))) * SIZE;
      const int text = b0 + at;
      out.k0 = min(max(a.starts_k[text], 0), a.rows_k);
      out.nk = max(min(a.starts_k[text + 1], a.rows_k) - out.k0, 0);
      return true;
    }
    index -= __shfl(upto, 63);
  }
  return false;
}

// Any type and dim: four waves of 16 queries of one head each, keys and
// values straight from memory (the caches).
template <int T, int DP, bool EVEN>
__global__ __launch_bounds__(256) void window_attention_rows(PromptArgs a) {
  typedef Attend<T, DP, EVEN> A;
  typedef typename A::V V;
  constexpr int K = A::KEYS;
  Block bl;
  if (!find_block<64>(a, blockIdx.y, bl)) return;
  const int lane = threadIdx.x % 64, col = lane % 16, quarter = lane / 16;
  const int per = a.heads / a.kv_heads, kv = blockIdx.x % a.kv_heads, head = kv * per + blockIdx.x / a.kv_heads;
  const int first = bl.first + threadIdx.x / 64 * 16;
  if (first >= bl.nq) return;
  const int rows = min(16, bl.nq - first);
  const int p0 = bl.nk - bl.nq + first;  // the first query's place; the last's is p0 + rows - 1
  const int p = p0 + min(col, rows - 1);
  A at;
  at.start((const V *)a.q + (long)(bl.q0 + first + min(col, rows - 1)) * a.q_stride + (long)head * a.dim, a.dim,
           quarter);
  const V *k = (const V *)a.k + (long)bl.k0 * a.k_stride + (long)kv * a.dim;
  const V *v = (const V *)a.v + (long)bl.k0 * a.v_stride + (long)kv * a.dim;
  const int last = p0 + rows - 1;                            // of all rows' keys
  const int low = a.window ? max(p0 - a.window + 1, 0) : 0;  // the first row's window starts here
  const int sinks = min(a.sinks, low);                       // sinks before every window
  const int start = low / K * K, sink_tiles = min((sinks + K - 1) / K, start / K);
  const int tiles = sink_tiles + (last >= start ? (last - start) / K + 1 : 0);
  for (int t = 0; t < tiles; t++) {
    const int k0 = t < sink_tiles ? t * K : start + (t - sink_tiles) * K;
    const bool masked = k0 + K - 1 > p0 || (a.window && k0 <= last - a.window);
    auto seen = [&](int i) {
      const int j = k0 + i;
      return j <= p && (!a.window || j > p - a.window || j < a.sinks);
    };
    auto any = [&](int i) {  // whether some row sees it
      const int j = k0 + i;
      return j <= last && (j >= low || j < a.sinks);
    };
    at.template tile<true>(
        [&](int i) -> const V * { return masked && !any(i) ? nullptr : k + (long)(k0 + i) * a.k_stride; },
        [&](int i) -> const V * { return masked && !any(i) ? nullptr : v + (long)(k0 + i) * a.v_stride; }, seen,
        masked, a.dim, a.scale, lane);
  }
  const float l = at.total();
  const float f = l == 0.0f ? 0.0f : 1.0f / l;
  if (col >= rows) return;
  V *y = (V *)a.y + (long)(bl.q0 + first + col) * a.y_stride + (long)head * a.dim;
#pragma unroll
  for (int r = 0; r < 4; r++) {
    V out[A::E];
#pragma unroll
    for (int e = 0; e < A::E; e++) out[e] = Num<T>::put(l == 0.0f ? 0.0f : at.o[e][r] * f);
    const int d = A::E * (4 * quarter + r);
    store_n(y + d, (long)a.dim - d, out);
  }
}

template <int T, int DP>
void launch_rows(const PromptArgs &a, hipStream_t s) {
  const dim3 grid(a.heads, a.rows_q / 64 + a.batch);
  if (a.dim % 8 == 0)
    hipLaunchKernelGGL((window_attention_rows<T, DP, true>), grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((window_attention_rows<T, DP, false>), grid, dim3(256), 0, s, a);
}

template <int T>
hipError_t launch(const PromptArgs &a, hipStream_t s) {
  if (a.dim <= 64)
    launch_rows<T, 64>(a, s);
  else if (a.dim <= 128)
    launch_rows<T, 128>(a, s);
  else
    launch_rows<T, 256>(a, s);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_window_attention(const PromptArgs &a, int type, hipStream_t s) {
  switch (type) {
    case PPOCR_F32: return launch<PPOCR_F32>(a, s);
    case PPOCR_BF16: return launch<PPOCR_BF16>(a, s);
    case PPOCR_F16: return launch<PPOCR_F16>(a, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace ppocr
