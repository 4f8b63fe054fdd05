// 8-bit codes of a quantised key-value pool and how kernels address it.
//
// A row (one token of one kv head) is kD codes and a scale byte; element = code * 2^(scale - 127).  Powers of two keep
// every step but the one rounding to a code exact: the division by the scale, reading back (e4m3 has 4 significant bits,
// int8 8, bf16 8), and quantising again what was read back.  The price is up to one bit of an int8 code's range; an e4m3
// code loses nothing, its rounding is relative.
#pragma once
#include <hip/hip_runtime.h>

#include "va_device.h"
#include "va_mfma_common.h"

namespace va {

struct E4M3 {
  static constexpr int kId = VA_CODE_E4M3;
  // largest code 448 = 1.75 * 2^8: a row whose maximum has a mantissa up to 1.75 gets its exponent - 8, others one more
  static constexpr uint32_t kTopMantissa = 0x600000u;
  static constexpr int kTopExponent = 8;
  // 1.875 * 2^127 (code 240): what a larger number would round to, 2^128, is no fp32 number
  static constexpr uint32_t kLimit = 0x7f700000u;
  static constexpr uint32_t kNotZero = 0x7f7f7f7fu;  // bits of four codes of which one at least is set where not all are zero
  static __device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);  // round to nearest even; no value exceeds 448
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
  }
  static __device__ __forceinline__ void unpack4(uint32_t w, float* out) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    out[0] = lo[0], out[1] = lo[1], out[2] = hi[0], out[3] = hi[1];
  }
  // Eight codes as bf16, exactly, and times a power of two at no cost (four instructions, each at the full rate).
  static constexpr bool kScales = true;
  static __device__ __forceinline__ va_u32x4 bf16x8(va_u32x2 w, float scale = 1.f) {
    return va_u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[0], scale, false)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[0], scale, true)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[1], scale, false)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[1], scale, true))};
  }
};
struct INT8 {
  static constexpr int kId = VA_CODE_INT8;
  static constexpr uint32_t kTopMantissa = 0x7E0000u;  // largest code 127 = 1.984375 * 2^6
  static constexpr int kTopExponent = 6;
  static constexpr uint32_t kLimit = 0x7f7e0000u;  // 127 * 2^121, as above
  static constexpr uint32_t kNotZero = 0xffffffffu;
  static __device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
    const uint32_t x = (uint8_t)(int)rintf(a), y = (uint8_t)(int)rintf(b), z = (uint8_t)(int)rintf(c), w = (uint8_t)(int)rintf(d);
    return x | (y << 8) | (z << 16) | (w << 24);
  }
  static __device__ __forceinline__ void unpack4(uint32_t w, float* out) {
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = (float)(int8_t)(w >> (8 * i));
  }
  static constexpr bool kScales = false;
  static __device__ __forceinline__ va_u32x4 bf16x8(va_u32x2 w) {  // (bf16 has the eight bits of a code)
    float x[8];
    unpack4(w[0], x), unpack4(w[1], x + 4);
    return va_u32x4{Mma<BF16>::pack(x[0], x[1]), Mma<BF16>::pack(x[2], x[3]), Mma<BF16>::pack(x[4], x[5]), Mma<BF16>::pack(x[6], x[7])};
  }
};

// Scale byte of a row whose largest magnitude has the bits `top` (a NaN's are above an infinity's).
template <typename C>
__device__ __forceinline__ int scale_of(uint32_t top) {
  if (top >= 0x7f800000u) return 255;
  top = min(top, C::kLimit);
  const int e = (int)(top >> 23) - C::kTopExponent + ((top & 0x7fffffu) > C::kTopMantissa ? 1 : 0);
  return max(e, 1);  // at most 127 + 127 - 6 + 1
}
// An element in front of its division by the scale: numbers past the limit become the limit.
template <typename C>
__device__ __forceinline__ float limited(float x) {
  return __builtin_amdgcn_fmed3f(x, -__uint_as_float(C::kLimit), __uint_as_float(C::kLimit));
}
// 2^(127 - scale), the factor in front of the rounding; 0 for a row without finite values, whose codes become 0
// (a NaN or infinity times 0 is NaN: the caller clears those).
__device__ __forceinline__ float inverse_scale(int scale) { return __uint_as_float((uint32_t)(254 - min(scale, 254)) << 23); }
// 2^(scale - 127); infinite for 255, which makes NaN of the codes of zero that go with it
__device__ __forceinline__ float scale_value(uint32_t scale) { return __uint_as_float(scale << 23); }

// Pages of a pool: a shift where page_size is a power of two, 32-bit divisions otherwise.
struct PageMap {
  uint32_t size;
  int shift;  // -1: not a power of two
  __host__ __device__ __forceinline__ void split(uint32_t slot, uint32_t& page, uint32_t& place) const {
    page = shift >= 0 ? slot >> shift : slot / size;
    place = slot - page * size;
  }
};
inline PageMap page_map(int page_size) {
  return PageMap{(uint32_t)page_size, (page_size & (page_size - 1)) == 0 ? __builtin_ctz((unsigned)page_size) : -1};
}
// Index of the row (slot, head) of a layer: its scale byte lies there, its codes at kD times that.
__device__ __forceinline__ long long quant_row(const PageMap& p, uint32_t slot, int head, int num_kv_heads) {
  uint32_t page, place;
  p.split(slot, page, place);
  return ((long long)page * num_kv_heads + head) * p.size + place;
}

// Eight cosines and sines of pairs [i0, i0 + 8) at position p.
__device__ __forceinline__ void turns8(const RopeDev& rope, const Pos3& p, int i0, float* c, float* s) {
  if (rope.mode == VA_ROPE_TABLE) {
    long long a = p.t < 0 ? -p.t : p.t;
    if (a > rope.max_pos - 1) a = rope.max_pos - 1;
    const float* row = rope.cos_sin + a * (long long)rope.rotary_dim + i0;
    const float4 c0 = *(const float4*)row, c1 = *(const float4*)(row + 4);
    const float4 s0 = *(const float4*)(row + rope.half), s1 = *(const float4*)(row + rope.half + 4);
    c[0] = c0.x, c[1] = c0.y, c[2] = c0.z, c[3] = c0.w, c[4] = c1.x, c[5] = c1.y, c[6] = c1.z, c[7] = c1.w;
    s[0] = s0.x, s[1] = s0.y, s[2] = s0.z, s[3] = s0.w, s[4] = s1.x, s[5] = s1.y, s[6] = s1.z, s[7] = s1.w;
    if (p.t < 0) {
#pragma unroll
      for (int k = 0; k < 8; ++k) s[k] = -s[k];
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) rope_cos_sin(rope, p, i0 + k, c[k], s[k]);
  }
}

// Pairs (a, b) rotated in place in fp32, every product and sum rounded by itself (the definition's arithmetic).
__device__ __forceinline__ void turn8(const float* c, const float* s, float* a, float* b) {
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float x1 = a[k], x2 = b[k];
    a[k] = mul_rounded(c[k], x1) - mul_rounded(s[k], x2);
    b[k] = mul_rounded(c[k], x2) + mul_rounded(s[k], x1);
  }
}

// Host: refuses a pool that the kernels cannot address.
int check_quant_pool(const VaQuantPool* pool, const VaShape* shape);

}  // namespace va
