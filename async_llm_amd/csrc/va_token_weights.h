// Accumulated attention weights beside a pool: [kv heads][slots], a sum for every token and kv head.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

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

// The sums of n tokens alone (va_move.hip).
int launch_move_weights(const TokenWeights& w, int heads, const int64_t* src, const int64_t* dst, long long n, hipStream_t stream);

}  // namespace va
