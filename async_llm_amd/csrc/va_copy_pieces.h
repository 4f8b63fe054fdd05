// Pieces of pool rows as copies move them.
#pragma once
#include <hip/hip_runtime.h>

#include "va_device.h"

namespace va {

template <typename S, int kVec>
struct alignas(kVec * sizeof(S) == 16 ? 16 : alignof(S)) Piece {
  S v[kVec];
};

// 16-byte pieces travel as non-temporal loads and stores: every row is read once and written once,
// nothing of it is worth a place in the caches (two 16 384-token blocks over four layers: 259 -> 247 us).
typedef uint32_t va_copy_u32x4 __attribute__((ext_vector_type(4)));

template <typename S, int kVec>
__device__ __forceinline__ Piece<S, kVec> load_piece(const S* p) {
  Piece<S, kVec> out;
  if constexpr (kVec * sizeof(S) == 16) {
    *reinterpret_cast<va_copy_u32x4*>(out.v) = __builtin_nontemporal_load(reinterpret_cast<const va_copy_u32x4*>(p));
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i) out.v[i] = p[i];
  }
  return out;
}

template <typename S, int kVec>
__device__ __forceinline__ void store_piece(S* p, const Piece<S, kVec>& x) {
  if constexpr (kVec * sizeof(S) == 16) {
    __builtin_nontemporal_store(*reinterpret_cast<const va_copy_u32x4*>(x.v), reinterpret_cast<va_copy_u32x4*>(p));
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i) p[i] = x.v[i];
  }
}

}  // namespace va
