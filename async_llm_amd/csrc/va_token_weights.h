// Accumulated attention weights beside a pool: [kv heads][slots], a sum for every token and kv head.
#pragma once
#include <hip/hip_runtime.h>

namespace va {

struct TokenWeights {
  float* sums;  // may be null: there are none
  long long slots;
};

// Copies a token's sums to another slot: those of heads first, first + step, ...
__device__ __forceinline__ void move_weights(const TokenWeights& w, int heads, long long src, long long dst, int first, int step) {
  if (!w.sums) return;
  for (int h = first; h < heads; h += step) w.sums[h * w.slots + dst] = w.sums[h * w.slots + src];
}

}  // namespace va
