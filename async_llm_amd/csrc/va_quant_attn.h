// What the kernels of view attention over a quantised pool share.
#pragma once
#include <hip/hip_runtime.h>

#include "va_launch.h"
#include "va_quant.h"

namespace va {

struct QuantAttnArgs {
  AttnArgs a;  // k_pool, v_pool: codes
  const uint8_t* k_scales;
  const uint8_t* v_scales;
  PageMap pages;
};

// Element `at` of an activation array, by its run-time type: where a few hundred elements are read once a link, an
// instantiation for every type is not worth its code.
__device__ __forceinline__ float activation(const void* x, long long at, int dtype) {
  if (dtype == VA_BF16) return BF16::load(((const BF16::storage*)x)[at]);
  if (dtype == VA_F16) return F16::load(((const F16::storage*)x)[at]);
  return ((const float*)x)[at];
}
__device__ __forceinline__ void store_activation(void* x, long long at, float v, int dtype) {
  if (dtype == VA_BF16) {
    ((BF16::storage*)x)[at] = BF16::store(v);
  } else if (dtype == VA_F16) {
    ((F16::storage*)x)[at] = F16::store(v);
  } else {
    ((float*)x)[at] = v;
  }
}

// A row's result from its state: nothing visible gives 0 and -inf (a sum that is NaN stays NaN).
__device__ __forceinline__ float normalised(float acc, float sum) { return sum == 0.f ? 0.f : acc / sum; }
__device__ __forceinline__ float log_sum(float m, float sum, int base2) {
  const float lse2 = sum == 0.f ? -INFINITY : m + log2f(sum);
  return base2 ? lse2 : lse2 * kLn2;
}

// Pool row of token t of a sub-request for kv head hk.
__device__ __forceinline__ long long quant_token_row(const QuantAttnArgs& qa, int kv_begin, int t, bool slots, int hk) {
  if (slots) return quant_row(qa.pages, (uint32_t)qa.a.kv_indices[kv_begin + t], hk, qa.a.num_kv_heads);
  uint32_t page, place;
  qa.pages.split((uint32_t)t, page, place);
  return ((long long)qa.a.kv_indices[kv_begin + (int)page] * qa.a.num_kv_heads + hk) * qa.pages.size + place;
}

// The matrix-core kernels: 16-bit activations, head_dim 64, 128 or 256.  Tiles of whole pages (va_quant_stream.hip), or tokens
// looked up one by one (va_quant_scattered.hip: pages of fewer than 16 tokens or of a number that no power of two is).
// `pieces`: q rows start on 16-byte boundaries, out on 8-byte ones.  `only_if`: where it is given and holds 0 when the launch
// runs, all workgroups leave at once.  Such launches have kernels of their own: asked in the others, it takes 0.4 us of a
// step of 13.5.
int launch_quant_mfma(const QuantAttnArgs& qa, const int32_t* only_if, int dtype, int code_type, int n_items, int q_tile, hipStream_t stream);
int launch_quant_scattered(const QuantAttnArgs& qa, const int32_t* only_if, int dtype, int code_type, int n_items, int pieces, hipStream_t stream);

}  // namespace va
