// Attention over a cache in 4 bits, of f32 queries: their products in two parts.
#include "attend4.hpp"

namespace ppocr {
hipError_t launch_kv4_attention_32(const Attend4Args &a, hipStream_t s) { return launch_attention4<true>(a, s); }
}  // namespace ppocr
