// Attention weights by cached token: for every token and kv head the sum, over all rows and q heads that see the token, of
// exp(score - lse), added to the sums of former steps.
//
//   S^T[tokens, rows] = K . Q^T          matrix cores, keys as the A operand (a lane's elements of the result: tokens of one row)
//   sum[token] += exp2(S - lse2[row])    no running maximum: the log-sum is known, so rows may come in any order and be split
//
// Sums are 32-bit numbers that users compare and add up over many steps, so queries are not rounded to 16 bits: they come as sums
// of 16-bit numbers (bf16: three, which hold all 24 bits; float16: two of a row brought into its range by a power of two, 22
// bits) and each product is taken that often.  A first pass over the packed rows (weigh_rows_kernel) turns them, scales them by
// log2(e) / sqrt(D) and writes those parts as the matrix cores read them.
//
// Two ways, by span (va_weigh.h), in one launch where a step has both:
//   * strips (weigh_strip): the rows that see a token make one tile of 16, as in decode steps.  Bound by the keys: they travel to LDS
//     in whole lines, each wave's tile in a place of its own, while the tile before it is at the products.
//   * tile items (weigh_tiles): many rows see a token, as those of many new tokens.  Bound by the products: 64 tokens' keys stay
//     in a wave's registers while the rows' queries pass by through LDS, for all four waves at once.
// Where a chunk's rows are split among workgroups each writes partial sums, and weigh_join_kernel adds them in their order.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "va_device.h"
#include "va_internal.h"
#include "va_launch.h"
#include "va_mfma_common.h"
#include "va_quant.h"
#include "va_quant_mfma.h"
#include "va_weigh.h"

namespace va {

constexpr int kWeighThreads = 256, kWeighWaves = kWeighThreads / kWave;
constexpr int kWeighMaxDim = 256;

// What a (row, q head) brings besides its query: p = exp2(dot * scale + minus_lse), tokens [lo, hi) of the span.
struct WeighRow {
  float minus_lse, scale;
  int lo, hi;
};

struct WeighArgs {
  const void* q;
  long long q_row_stride;
  const void* k_pool;  // codes, of a quantised pool
  const uint8_t* k_scales;
  long long pool_row_stride;  // elements between token slots (16- and 32-bit pools)
  const int32_t* items;
  const int32_t* strips;
  const int32_t* joins;
  const int32_t* pages;
  const int32_t* sub_rows;
  const int32_t* lo;
  const int32_t* hi;
  int n_rows, n_tiles;
  int n_tile_items;   // the first items
  int n_first_tiles;  // tiles of 16 of their rows, the first ones
  const int64_t* sub_worker;
  const int64_t* sub_loc;
  long long sub_loc_axis_stride;
  const float* lse;
  int lse_base2;
  const float* weights_in;
  float* weights_out;
  long long num_slots;
  char* queries;  // [kv head][tile] parts as the products read them, or 32-bit rows
  WeighRow* rows;  // [kv head][tile][16]
  float* partials;  // [kv head][n_partials]
  long long n_partials;
  int num_q_heads, num_kv_heads, head_dim, dtype;
  int pieces;  // queries start on 16-byte boundaries
  PageMap page_map;
  RopeDev rope;
  float scale_log2;
};

__device__ __forceinline__ float weigh_activation(const void* x, long long at, int dtype) {
  if (dtype == VA_BF16) return BF16::load(((const BF16::storage*)x)[at]);
  if (dtype == VA_F16) return F16::load(((const F16::storage*)x)[at]);
  return ((const float*)x)[at];
}

// Pool slot of token t of a span.
__device__ __forceinline__ uint32_t weigh_slot(const WeighArgs& a, int page_begin, int t) {
  uint32_t page, place;
  a.page_map.split((uint32_t)t, page, place);
  return (uint32_t)a.pages[page_begin + (int)page] * a.page_map.size + place;
}

// ---------------------------------------------------------------------------
// queries
// ---------------------------------------------------------------------------
// What a row's query becomes.  Parts lie as [tile][part][step][lane] of 16 bytes, lane 16 * group + j (32 * group + j) for row j of
// a tile of 16 (32), so that a wave reads its operands of a step in one run; pieces of 8 (32-bit: 4) dims go to steps and
// contraction groups in the order in which lanes hold the keys: piece groups * step + group, or over codes, of which a lane reads 16 at
// once, 2 groups (step / 2) + 2 group + step % 2.  kTile*: for tile items, 32 rows a tile; the others are for strips.
enum RowKind { kPlain32, kParts32, kPartsBF16, kPartsF16, kCodesF16, kTileF16, kTileCodes };
__host__ __device__ constexpr int parts_of(int kind) { return kind >= kPartsF16 ? 2 : kind == kPartsBF16 ? 3 : 1; }
__host__ __device__ constexpr int rows_of(int kind) { return kind >= kTileF16 ? VA_WEIGH_TILE_ROWS : 16; }
__host__ __device__ constexpr int tile_bytes(int dim) { return 16 * dim * 6; }  // (room for any of them)

// Eight neighbouring elements of a row, piece `piece` of row j (32-bit: pieces 2 piece and 2 piece + 1); y is used up.
template <int kKind>
__device__ __forceinline__ void write_row_piece(char* tile_at, int dim, int j, int piece, float* y) {
  if constexpr (kKind == kPlain32) {
    float* to = (float*)tile_at + j * dim + 8 * piece;
#pragma unroll
    for (int e = 0; e < 8; ++e) to[e] = y[e];
  } else if constexpr (kKind == kParts32) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int p = 2 * piece + i;
      *(va_f32x4*)(tile_at + (p / 4) * 1024 + (16 * (p % 4) + j) * 16) = va_f32x4{y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]};
    }
  } else {
    constexpr bool kHalf = parts_of(kKind) == 2, kCodes = kKind == kTileCodes || kKind == kCodesF16;
    constexpr int kRows = rows_of(kKind), kGroups = 64 / kRows, kSteps = 8 * kGroups;  // contraction groups, dims of a step
    const int step = kCodes ? 2 * (piece / (2 * kGroups)) + piece % 2 : piece / kGroups, group = kCodes ? piece % (2 * kGroups) / 2 : piece % kGroups;
#pragma unroll
    for (int part = 0; part < parts_of(kKind); ++part) {
      va_u32x4 w;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (kHalf) {
          w[e] = Mma<F16>::pack(y[2 * e], y[2 * e + 1]);
          y[2 * e] -= F16::load(__builtin_bit_cast(__half, (uint16_t)w[e])), y[2 * e + 1] -= F16::load(__builtin_bit_cast(__half, (uint16_t)(w[e] >> 16)));
        } else {
          w[e] = Mma<BF16>::pack(y[2 * e], y[2 * e + 1]);
          y[2 * e] -= __uint_as_float(w[e] << 16), y[2 * e + 1] -= __uint_as_float(w[e] & 0xffff0000u);
        }
      }
      *(va_u32x4*)(tile_at + (part * (dim / kSteps) + step) * 1024 + (kRows * group + j) * 16) = w;
    }
  }
}

// The power of two that brings a row whose largest element is `most` to 2^10 .. 2^11, as its exponent.
__device__ __forceinline__ int row_exponent(float most) {
  return most > 0.f && most < INFINITY ? min(max(10 - ((int)(__float_as_uint(most) >> 23) - 127), -100), 100) : 0;
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

// The row's other half: a row that is padding, or whose log-sum is -inf, adds exp2(-inf) = 0 to every token.  The log-sum in powers of
// two is a 32-bit product, off by up to 1.3 * 2^-24 of it: an error that all of a row's weights share.
__device__ __forceinline__ WeighRow row_beside(const WeighArgs& a, int row, bool counts, float lse, float scale) {
  if (!counts) return WeighRow{-INFINITY, 0.f, 0, 0x7fffffff};
  return WeighRow{a.lse_base2 ? -lse : -lse * kLog2e, scale, a.lo[row], a.hi[row]};
}

__device__ __forceinline__ void weigh_activations8(const void* x, long long at, int dtype, int pieces, float* y) {
  if (pieces && dtype == VA_F32) {
    const float4 u = *(const float4*)((const float*)x + at), v = *(const float4*)((const float*)x + at + 4);
    y[0] = u.x, y[1] = u.y, y[2] = u.z, y[3] = u.w, y[4] = v.x, y[5] = v.y, y[6] = v.z, y[7] = v.w;
  } else if (pieces) {
    const va_u32x4 w = *(const va_u32x4*)((const uint16_t*)x + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint16_t u = (uint16_t)w[i], v = (uint16_t)(w[i] >> 16);
      y[2 * i] = dtype == VA_BF16 ? BF16::load(u) : __half2float(__builtin_bit_cast(__half, u));
      y[2 * i + 1] = dtype == VA_BF16 ? BF16::load(v) : __half2float(__builtin_bit_cast(__half, v));
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = weigh_activation(x, at + e, dtype);
  }
}

// A thread per 16 elements of a row: both halves of eight pairs, or two pieces past the rotary part.  head_dim 64, 128 or 256 and
// rotary_dim a multiple of 16.  A thread goes on to the rows of other kv heads while it holds the angles of this one.
// Few rows are a chain of trips (sub-row, its worker and position, query and angles: 3.5 us for one row, 8 to 9 for 64 over five blocks each),
// many are bound by what is written (4 chunks, 240 MB: 80 us).
template <int kKind>
__device__ __forceinline__ void weigh_row_units(const WeighArgs& a) {
  const int D = a.head_dim, units = D / 16, G = a.num_q_heads / a.num_kv_heads;
  const int task = blockIdx.x * kWeighThreads + threadIdx.x, pair = task / units, x = task - pair * units;
  if (pair >= a.n_tiles * 16) return;  // (whole rows leave)
  const int row = pair / G, sub = a.sub_rows[row];
  const int pairs = a.rope.half / 8, d0 = x < pairs ? 8 * x : 16 * x, d1 = x < pairs ? 8 * x + a.rope.half : 16 * x + 8;
  const long long worker = sub >= 0 ? a.sub_worker[sub] : 0;
  float c[8], s[8];
  if (sub >= 0 && x < pairs) turns8(a.rope, load_pos(a.sub_loc, a.sub_loc_axis_stride, sub), d0, c, s);
#pragma clang loop unroll(disable)
  for (int hk = blockIdx.y; hk < a.num_kv_heads; hk += gridDim.y) {
    const int hq = hk * G + pair - row * G;
    float y[2][8], scale = 1.f, lse = -INFINITY;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[0][e] = y[1][e] = 0.f;
    if (sub >= 0) {
      const long long at = worker * a.q_row_stride + (long long)hq * D;
      lse = a.lse[worker * a.num_q_heads + hq];
      weigh_activations8(a.q, at + d0, a.dtype, a.pieces, y[0]);
      weigh_activations8(a.q, at + d1, a.dtype, a.pieces, y[1]);
      if (x < pairs) turn8(c, s, y[0], y[1]);
    }
    const bool counts = lse != -INFINITY;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[0][e] = counts ? y[0][e] * a.scale_log2 : 0.f, y[1][e] = counts ? y[1][e] * a.scale_log2 : 0.f;
    if constexpr (parts_of(kKind) == 2) {
      float most = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) most = fmaxf(most, fmaxf(fabsf(y[0][e]), fabsf(y[1][e])));
      for (int off = 1; off < units; off <<= 1) most = fmaxf(most, __shfl_xor(most, off, kWave));
      const int e = row_exponent(most);
      scale = power_of_two(-e);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[0][i] *= power_of_two(e), y[1][i] *= power_of_two(e);
    }
    constexpr int kRows = rows_of(kKind);
    char* at = a.queries + ((long long)hk * a.n_tiles + pair / kRows * (kRows / 16)) * tile_bytes(D);
    write_row_piece<kKind>(at, D, pair % kRows, d0 / 8, y[0]);
    write_row_piece<kKind>(at, D, pair % kRows, d1 / 8, y[1]);
    if (x == 0) a.rows[(long long)hk * a.n_tiles * 16 + pair] = row_beside(a, row, counts, lse, scale);
  }
}
// kFirst: what the rows of tile items become, the others kKind.  (A wave's rows are of one kind: 16 of them are a wave or more.)
template <int kFirst, int kKind>
__global__ __launch_bounds__(kWeighThreads) void weigh_rows_kernel(WeighArgs a) {
  if constexpr (kFirst == kKind) {
    weigh_row_units<kKind>(a);
  } else {
    const int wave = blockIdx.x * kWeighWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    if ((long long)wave * kWave / (a.head_dim / 16) < (long long)a.n_first_tiles * 16) weigh_row_units<kFirst>(a); else weigh_row_units<kKind>(a);
  }
}

// Any head_dim up to kWeighMaxDim and any rotary_dim: a tile a workgroup, through LDS.
template <int kKind>
__device__ __forceinline__ void weigh_row_tile(const WeighArgs& a, float (&x)[16][kWeighMaxDim + 1]) {
  const int tile = blockIdx.x, hk = blockIdx.y, D = a.head_dim, G = a.num_q_heads / a.num_kv_heads;
  const int j = threadIdx.x / 16, c = threadIdx.x % 16;
  const int pair = tile * 16 + j, row = pair / G, hq = hk * G + pair - row * G;
  const int sub = a.sub_rows[row];
  const long long worker = sub < 0 ? 0 : a.sub_worker[sub];
  const float lse = sub < 0 ? -INFINITY : a.lse[worker * a.num_q_heads + hq];
  const bool counts = lse != -INFINITY;
  float most = 0.f;
  auto put = [&](int d, float v) __attribute__((always_inline)) {
    x[j][d] = v;
    most = fmaxf(most, fabsf(v));
  };
  if (counts) {
    const Pos3 pos = load_pos(a.sub_loc, a.sub_loc_axis_stride, sub);
    const long long at = worker * a.q_row_stride + (long long)hq * D;
    for (int i = c; i < a.rope.half; i += 16) {
      float cs, sn;
      rope_cos_sin(a.rope, pos, i, cs, sn);
      const float x1 = weigh_activation(a.q, at + i, a.dtype), x2 = weigh_activation(a.q, at + i + a.rope.half, a.dtype);
      put(i, (mul_rounded(cs, x1) - mul_rounded(sn, x2)) * a.scale_log2);
      put(i + a.rope.half, (mul_rounded(cs, x2) + mul_rounded(sn, x1)) * a.scale_log2);
    }
    for (int d = 2 * a.rope.half + c; d < D; d += 16) put(d, weigh_activation(a.q, at + d, a.dtype) * a.scale_log2);
  } else {
    for (int d = c; d < D; d += 16) x[j][d] = 0.f;
  }
  __syncthreads();
  float scale = 1.f, up = 1.f;
  if constexpr (parts_of(kKind) == 2) {
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) most = fmaxf(most, __shfl_xor(most, off, kWave));
    const int e = row_exponent(most);
    up = power_of_two(e), scale = power_of_two(-e);
  }
  constexpr int kRows = rows_of(kKind);
  char* at = a.queries + ((long long)hk * a.n_tiles + pair / kRows * (kRows / 16)) * tile_bytes(D);
  if constexpr (kKind == kPlain32) {
    for (int d = c; d < D; d += 16) ((float*)at)[j * D + d] = x[j][d];
  } else {
    for (int piece = c; piece < D / 8; piece += 16) {
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = x[j][8 * piece + e] * up;
      write_row_piece<kKind>(at, D, pair % kRows, piece, y);
    }
  }
  if (c == 0) a.rows[(long long)hk * a.n_tiles * 16 + pair] = row_beside(a, row, counts, lse, scale);
}
template <int kFirst, int kKind>
__global__ __launch_bounds__(kWeighThreads) void weigh_rows_any_kernel(WeighArgs a) {
  __shared__ float x[16][kWeighMaxDim + 1];
  if (kFirst != kKind && (int)blockIdx.x < a.n_first_tiles) weigh_row_tile<kFirst>(a, x); else weigh_row_tile<kKind>(a, x);
}

// ---------------------------------------------------------------------------
// matrix cores
// ---------------------------------------------------------------------------
// Sum over the 16 lanes of a row.
__device__ __forceinline__ float row_sum(float x) {
#define VA_DPP_ADD(ctrl) x += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), ctrl, 0xf, 0xf, false))
  VA_DPP_ADD(0xb1);   // quad_perm 1 0 3 2
  VA_DPP_ADD(0x4e);   // quad_perm 2 3 0 1
  VA_DPP_ADD(0x141);  // row_half_mirror
  VA_DPP_ADD(0x140);  // row_mirror
#undef VA_DPP_ADD
  return x;
}

// What the keys of a pool are in the products of the walks: 16-byte pieces of the parts' type.
template <typename E>
struct WalkKeys {  // bf16
  static constexpr int kBytes = 2, kRows = kPartsBF16;
  static constexpr bool kCodes = false;
  static __device__ __forceinline__ va_f32x4 run(va_u32x4 k, va_u32x4 q, va_f32x4 c) { return Mma<BF16>::run(k, q, c); }
};
template <>
struct WalkKeys<F16> {
  static constexpr int kBytes = 2, kRows = kPartsF16;
  static constexpr bool kCodes = false;
  static __device__ __forceinline__ va_f32x4 run(va_u32x4 k, va_u32x4 q, va_f32x4 c) { return Mma<F16>::run(k, q, c); }
};
template <>
struct WalkKeys<F32> {
  static constexpr int kBytes = 4, kRows = kParts32;
  static constexpr bool kCodes = false;
  static __device__ __forceinline__ va_f32x4 run(va_u32x4 k, va_u32x4 q, va_f32x4 c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k[e]), __uint_as_float(q[e]), c, 0, 0, 0);
    return c;
  }
};
// (codes are float16 numbers as they are; their row's scale comes to the scores)
template <>
struct WalkKeys<E4M3> : WalkKeys<F16> {
  static constexpr int kBytes = 1, kRows = kCodesF16;
  static constexpr bool kCodes = true;
  static __device__ __forceinline__ va_u32x4 keys(va_u32x2 codes) {
    va_u32x4 w;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      w[2 * e] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes[e], 1.f, false));
      w[2 * e + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes[e], 1.f, true));
    }
    return w;
  }
};
template <>
struct WalkKeys<INT8> : WalkKeys<F16> {
  static constexpr int kBytes = 1, kRows = kCodesF16;
  static constexpr bool kCodes = true;
  // A code plus 128 as the low byte of 1024's mantissa is 1152 plus the code.
  static __device__ __forceinline__ va_u32x4 keys(va_u32x2 codes) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    const f16x2 base = {(_Float16)1152.f, (_Float16)1152.f};
    va_u32x4 w;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t up = codes[e] ^ 0x80808080u;
      w[2 * e] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, up, 0x04010400u)) - base);
      w[2 * e + 1] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, up, 0x04030402u)) - base);
    }
    return w;
  }
};

// kv heads of a strip's workgroup.
__host__ __device__ inline int strip_heads(int num_kv_heads) { return num_kv_heads % 4 == 0 ? 4 : num_kv_heads % 2 == 0 ? 2 : 1; }

constexpr int groups_of(int row_bytes) { return row_bytes > 256 ? 1 : row_bytes > 128 ? 2 : 4; }

template <int kD, typename C>
struct WalkShape {
  using K = WalkKeys<C>;
  static constexpr int kRowBytes = kD * K::kBytes;
  static constexpr int kPieces = kRowBytes / 16;           // of a token's row
  static constexpr int kRaw = kPieces / 4;                 // pieces of a row that a lane takes
  static constexpr int kSteps = K::kCodes ? 2 * kRaw : kRaw;  // operand pieces of a lane, per part
  static constexpr int kParts = parts_of(K::kRows);
  // groups of 16 tokens of a wave's tile: 8 KB, up to 64 tokens, 16 at least
  static constexpr int kGroups = groups_of(kRowBytes);
  static constexpr int kTokens = 16 * kGroups;
  static constexpr int kGroupBytes = 16 * kRowBytes;
  static constexpr int kLoads = kGroupBytes / 1024;        // wave-level loads of a group
  // behind a tile's rows: the tokens' sums so far, a word for every scale, the tokens' slots
  static constexpr int kSumsAt = kGroups * kGroupBytes, kScalesAt = kSumsAt + 256, kSlotsAt = kScalesAt + (K::kCodes ? 256 : 0);
  static constexpr int kTileBytes = kSlotsAt + 256;
  // behind the tiles: where a wave turns a tile's sums from lanes to tokens, and holds those of several tiles with their places
  static constexpr int kTurnOffset = kWeighWaves * kTileBytes;
  static constexpr int kHold = kGroupBytes > 8 * 1024 ? 512 : 2048;
  static constexpr int kWaveBytes = 256 + kHold * 4 + kHold / 16 * 8;
  static constexpr int kLdsBytes = kTurnOffset + kWeighWaves * kWaveBytes;
  static_assert(2 * kLdsBytes <= 160 * 1024, "two workgroups share the LDS of a CU");
};
// Piece c of row r of a group lies at position c ^ walk_swz(r): the fragments of sixteen rows then lie in different banks.
template <int kPieces>
__device__ __forceinline__ int walk_swz(int r) {
  if constexpr (kPieces >= 16) return ((r & 7) << 1) | ((r >> 3) & 1);
  if constexpr (kPieces == 8) return (r & 6) | ((r >> 3) & 1);
  return (r >> 2) & 3;
}

// A workgroup walks a strip of items for up to four kv heads, whose rows of a token lie side by side, its waves on their own: each takes
// its head's tiles of an item's tokens (every second or fourth where there are fewer heads), brings them
// global -> LDS into a place of its own (keys, the sums so far and, over codes, scales) and asks for the next one, of the next item
// where this one ends, as soon as the keys are in registers.  There is no barrier, and nothing but the first tile of a strip
// is waited for idly.  8 requests of 131072 tokens and 4 heads of 256: 331 us, 6.6 TB/s; 16 heads of 64 5.5 TB/s, int8 codes 5.2.
// Sums are held in LDS and written many at a time: each store between the loads costs the memory about as much as 1 KB of
// keys (371 us with 512 held, 338 with 2048, rows' pass included).
template <int kD, typename C>
__device__ __forceinline__ void weigh_strip(const WeighArgs& a, unsigned block) {
  using Sh = WalkShape<kD, C>;
  using K = WalkKeys<C>;
  using Words = const __attribute__((address_space(4))) int32_t*;
  constexpr int kGroups = Sh::kGroups, kLoads = Sh::kLoads, kPieces = Sh::kPieces, kSteps = Sh::kSteps, kRaw = Sh::kRaw, kParts = Sh::kParts;
  constexpr int kTokens = Sh::kTokens;
  constexpr bool kSeveral = std::is_same_v<C, F32>;  // tokens may have several tiles of rows
  extern __shared__ va_u32x4 smem[];
  char* lds = (char*)smem;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int heads = strip_heads(a.num_kv_heads), turns = kWeighWaves / heads, place = wave / heads;  // tiles of a wave: place, + turns, ...
  const ItemHead where = item_and_head(block, a.num_kv_heads / heads);
  const int hk = where.head * heads + wave % heads, strip_begin = ((Words)a.strips)[where.item], strip_end = ((Words)a.strips)[where.item + 1];
  if (strip_begin == strip_end) return;
  const int lane = threadIdx.x % kWave, j = lane % 16, kg = lane / 16;
  char* tile = lds + wave * Sh::kTileBytes;
  const uint32_t dst = __builtin_amdgcn_readfirstlane(lds_address(tile));
  float* turn = (float*)(lds + Sh::kTurnOffset + wave * Sh::kWaveBytes);
  float* held_sums = turn + 64;
  uint2* held_groups = (uint2*)(held_sums + Sh::kHold);  // of 16 sums: where the first goes, how many there are
  const bool pages16 = a.page_map.shift >= 4;
  const long long row_bytes = K::kCodes ? kD : a.pool_row_stride * K::kBytes;
  const float* sums_in = a.weights_in + hk * a.num_slots;

  struct Piece {
    int pages, first, n_tok, tile_begin, tile_end, partial, tiles;  // tiles: this wave's, of tokens
  };
  auto piece_at = [&](int index) __attribute__((always_inline)) {
    const Words w = (Words)a.items + (long long)index * VA_WEIGH_ITEM_WORDS;
    Piece p{w[VA_WI_PAGES], w[VA_WI_FIRST], w[VA_WI_N_TOK], w[VA_WI_TILE_BEGIN], w[VA_WI_TILE_END], w[VA_WI_PARTIAL], 0};
    p.tiles = ((p.n_tok + kTokens - 1) / kTokens - place + turns - 1) / turns;
    return p;
  };

  // ---- keys ----
  // This lane's part of load u of a group: row and piece, which belongs at its LDS position.  Loads in groups of up to four share one
  // setting of M0, whose immediate offsets move the pool address as well (grouped_lane_offset; the base gives the bias back).
  constexpr int kBias = 1024 * (kLoads - 1);
  auto ld_row = [&](int u) __attribute__((always_inline)) { return u * (kWave / kPieces) + lane / kPieces; };
  auto ld_piece = [&](int u) __attribute__((always_inline)) { return (lane % kPieces) ^ walk_swz<kPieces>(ld_row(u)); };
  uint32_t ld_off[kLoads];
#pragma unroll
  for (int u = 0; u < kLoads; ++u) ld_off[u] = grouped_lane_offset((uint32_t)(ld_row(u) * row_bytes + 16 * ld_piece(u) + kBias), u);
  auto row_at = [&](uint32_t slot) __attribute__((always_inline)) {  // byte of a slot's row of this head
    if constexpr (K::kCodes) return quant_row(a.page_map, slot, hk, a.num_kv_heads) * kD;
    return (long long)slot * row_bytes + hk * (long long)Sh::kRowBytes;
  };
  auto request_group = [&](const char* from, const uint32_t* off, uint32_t dst) __attribute__((always_inline)) {
    if constexpr (kLoads >= 4) {
#pragma unroll
      for (int u = 0; u < kLoads; u += 4) load_group_to_lds<4, true>(from, off + u, dst + 1024 * u);
    } else if constexpr (kLoads == 2) {
      load_group_to_lds<2, true>(from, off, dst);
    } else {
      load_to_lds(from, off[0], dst);
    }
  };
  // The tile to ask for next: its pages are looked up (in scalar loads) when the one before it has been asked for, so that nothing
  // is waited for between a tile's landing and the next request.
  struct Next {
    int pages, first, last, t0, page[kGroups];
  };
  Next next{};
  bool more = false;  // there is one
  int find_index = strip_begin, find_n = 0;
  Piece find = piece_at(strip_begin);
  auto find_next = [&]() __attribute__((always_inline)) {
    more = false;
    while (find_n == find.tiles) {
      if (find_index + 1 >= strip_end) return;
      find = piece_at(++find_index);
      find_n = 0;
    }
    next.pages = find.pages, next.first = find.first, next.last = find.n_tok - 1;
    next.t0 = (find_n++ * turns + place) * kTokens;
    if (pages16 && next.first % 16 == 0) {
#pragma unroll
      for (int g = 0; g < kGroups; ++g)  // (a group past the end: the last one)
        next.page[g] = ((Words)a.pages)[next.pages + ((next.first + min(next.t0 + 16 * g, next.last / 16 * 16)) >> a.page_map.shift)];
    }
    more = true;
  };
  auto request_next = [&]() __attribute__((always_inline)) {
    if (!more) return;
    uint32_t of_lane = 0;  // slot of the token whose words this lane brings: token `lane` of the tile
    if (pages16 && next.first % 16 == 0) {  // 16 tokens of a group lie in one page
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        const int t = min(next.t0 + 16 * g, next.last / 16 * 16);
        const uint32_t slot = ((uint32_t)next.page[g] << a.page_map.shift) + ((uint32_t)(next.first + t) & (a.page_map.size - 1));
        const char* from = (const char*)a.k_pool + (row_at(slot) - kBias);
        const int most = next.last - t;  // rows behind the last one repeat it
        if (most >= 15) {
          request_group(from, ld_off, dst + g * Sh::kGroupBytes);
        } else {
          uint32_t off[kLoads];
#pragma unroll
          for (int u = 0; u < kLoads; ++u) off[u] = ld_off[u] - (uint32_t)(max(0, ld_row(u) - most) * row_bytes);
          request_group(from, off, dst + g * Sh::kGroupBytes);
        }
        of_lane = kg == g || g == 0 ? slot + min(j, most) : of_lane;
      }
    } else {  // tokens looked up one by one: each lane one, handed to those that load it
      of_lane = weigh_slot(a, next.pages, next.first + min(next.t0 + lane % kTokens, next.last));
#pragma unroll
      for (int g = 0; g < kGroups; ++g)
#pragma unroll
        for (int u = 0; u < kLoads; ++u) {
          const uint32_t slot = (uint32_t)__shfl((int)of_lane, 16 * g + ld_row(u), kWave);
          load_to_lds((const char*)a.k_pool + row_at(slot) + 16 * ld_piece(u), dst + g * Sh::kGroupBytes + 1024 * u);
        }
    }
    load_word_to_lds(sums_in + of_lane, dst + Sh::kSumsAt);
    if constexpr (K::kCodes) load_bytes_to_lds((unsigned long long)a.k_scales + row_at(of_lane) / kD, dst + Sh::kScalesAt);
    *(uint32_t*)(tile + Sh::kSlotsAt + 4 * lane) = of_lane;
    find_next();
  };
  find_next();

  // ---- queries ----
  va_u32x4 q[kParts][kSteps];
  WeighRow row;
  const char* queries = a.queries + (long long)hk * a.n_tiles * tile_bytes(kD) + 16 * lane;
  auto load_queries = [&](int tile) __attribute__((always_inline)) {
    row = a.rows[((long long)hk * a.n_tiles + tile) * 16 + j];
    const char* at = queries + (long long)tile * tile_bytes(kD);
#pragma unroll
    for (int p = 0; p < kParts; ++p)
#pragma unroll
      for (int s = 0; s < kSteps; ++s) q[p][s] = *(const va_u32x4*)(at + (p * kSteps + s) * 1024);
  };
  auto queries_here = [&]() __attribute__((always_inline)) {  // (waited for here, not in the loop)
#pragma unroll
    for (int p = 0; p < kParts; ++p)
#pragma unroll
      for (int s = 0; s < kSteps; ++s) asm volatile("" : "+v"(q[p][s]));
    asm volatile("" : "+v"(row.minus_lse), "+v"(row.scale), "+v"(row.lo), "+v"(row.hi));
  };

  // ---- the walk ----
  request_next();
  int index = strip_begin, n = 0, q_tile = -1;
  Piece at = piece_at(strip_begin);
  // Sums not yet written, all of one kind: of this workgroup's part of a span's rows or not, in groups of 16 that lie side by side
  // or, of scattered tokens, with a place for each in the upper half.
  int held = 0;
  bool held_partial = false, held_scattered = false;
  auto write_held = [&]() __attribute__((always_inline)) {
    float* to = held_partial ? a.partials + hk * a.n_partials : a.weights_out + hk * a.num_slots;
    if (held_scattered) {
      for (int i = lane; i < held; i += kWave) {
        const uint32_t at = ((const uint32_t*)held_sums)[Sh::kHold / 2 + i];
        if (at != ~0u) to[at] = held_sums[i];
      }
    } else {
      for (int i = lane; i < held; i += kWave) {
        const uint2 group = held_groups[i / 16];
        if (i % 16 < (int)group.y) to[group.x + i % 16] = held_sums[i];
      }
    }
    held = 0;
  };
  while (true) {
    while (n == at.tiles) {
      if (index + 1 >= strip_end) break;
      at = piece_at(++index);
      n = 0;
    }
    if (n == at.tiles) break;
    const bool single = !kSeveral || at.tile_end - at.tile_begin == 1;
    if (single && at.tile_begin != q_tile) {
      load_queries(at.tile_begin);
      queries_here();
      q_tile = at.tile_begin;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the tile has landed
    va_u32x4 keys[kGroups][kRaw];
    va_u32x4 scale[K::kCodes ? kGroups : 1];  // of a lane's four tokens
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
#pragma unroll
      for (int s = 0; s < kRaw; ++s)
        keys[g][s] = *(const va_u32x4*)(tile + g * Sh::kGroupBytes + j * Sh::kRowBytes + 16 * ((4 * s + kg) ^ walk_swz<kPieces>(j)));
      if constexpr (K::kCodes) scale[g] = *(const va_u32x4*)(tile + Sh::kScalesAt + 4 * (16 * g + 4 * kg));
    }
    const float before = *(const float*)(tile + Sh::kSumsAt + 4 * lane);
    const uint32_t slot = *(const uint32_t*)(tile + Sh::kSlotsAt + 4 * lane);
    const bool partial = at.partial >= 0, scattered = !partial && !(pages16 && at.first % 16 == 0);
    if (held + kTokens > (scattered ? Sh::kHold / 2 : Sh::kHold) || held_partial != partial || held_scattered != scattered) write_held();
    held_partial = partial, held_scattered = scattered;
    __builtin_amdgcn_sched_barrier(0);
    if (single) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      request_next();
    }
    __builtin_amdgcn_sched_barrier(0);

    const int t0 = (n * turns + place) * kTokens, t_tile = at.first + t0, t_end = min(t_tile + kTokens, at.first + at.n_tok);
    float sum[kGroups][4];
#pragma unroll
    for (int g = 0; g < kGroups; ++g)
#pragma unroll
      for (int r = 0; r < 4; ++r) sum[g][r] = 0.f;
    auto add_rows = [&]() __attribute__((always_inline)) {
      va_f32x4 dots[kGroups];
#pragma unroll
      for (int g = 0; g < kGroups; ++g) dots[g] = va_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
          va_u32x4 k;
          if constexpr (K::kCodes) {
            const va_u32x4 raw = keys[g][s / 2];
            k = K::keys(s % 2 ? va_u32x2{raw[2], raw[3]} : va_u32x2{raw[0], raw[1]});
          } else {
            k = keys[g][s];
          }
#pragma unroll
          for (int p = kParts - 1; p >= 0; --p) dots[g] = K::run(k, q[p][s], dots[g]);  // (small parts first)
        }
      if constexpr (K::kCodes) {
#pragma unroll
        for (int g = 0; g < kGroups; ++g)
#pragma unroll
          for (int r = 0; r < 4; ++r) dots[g][r] *= scale_value(scale[g][r]);
      }
      if (__any(row.lo > t_tile || row.hi < t_end)) {  // some row does not see some token
#pragma unroll
        for (int g = 0; g < kGroups; ++g)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int t = t_tile + 16 * g + 4 * kg + r;
            const float p = __builtin_amdgcn_exp2f(fmaf(dots[g][r], row.scale, row.minus_lse));
            sum[g][r] += t >= row.lo && t < row.hi ? p : 0.f;
          }
      } else {
#pragma unroll
        for (int g = 0; g < kGroups; ++g)
#pragma unroll
          for (int r = 0; r < 4; ++r) sum[g][r] += __builtin_amdgcn_exp2f(fmaf(dots[g][r], row.scale, row.minus_lse));
      }
    };
    if (single) {
      add_rows();
    } else if constexpr (kSeveral) {
      // Queries are loaded tile by tile; a wait for those would be one for the next keys as well, which are asked for behind them.
      for (int of = at.tile_begin; of < at.tile_end; ++of) {
        load_queries(of);
        add_rows();
      }
      q_tile = -1;
    }
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      float of_token = 0.f;  // lane j < 4 has token 4 kg + j (a choice among the elements of an array would be one among addresses)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float x = row_sum(sum[g][r]);
        of_token = j == r ? x : of_token;
      }
      if (j < 4) turn[16 * g + 4 * kg + j] = of_token;
    }
    if (lane < kTokens) {
      held_sums[held + lane] = partial ? turn[lane] : before + turn[lane];
      if (scattered) {
        ((uint32_t*)held_sums)[Sh::kHold / 2 + held + lane] = t0 + lane < at.n_tok ? slot : ~0u;
      } else if (j == 0) {
        held_groups[(held + lane) / 16] = make_uint2(partial ? (uint32_t)(at.partial + t0 + lane) : slot, (uint32_t)min(16, max(0, at.n_tok - t0 - lane)));
      }
    }
    held += kTokens;
    if (!single) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      request_next();
    }
    ++n;
  }
  write_held();
}

// A workgroup's sums to where they go.
__device__ __forceinline__ void finish_sums(const WeighArgs& a, int page_begin, int first, int n_tok, int partial, int hk, const float* sums) {
  for (int t = threadIdx.x; t < n_tok; t += kWeighThreads) {
    if (partial >= 0) {
      a.partials[hk * a.n_partials + partial + t] = sums[t];
    } else {
      const long long to = hk * a.num_slots + weigh_slot(a, page_begin, first + t);
      a.weights_out[to] = a.weights_in[to] + sums[t];
    }
  }
}

// What the keys of a pool are in the products of the tiles: float16 numbers, times 2^x for a token.  16-bit keys come within
// float16's range by a power of two: with their row's largest element at 2^14 .. 2^15 what is over 2^-31 of it stays exact, and an error
// of 2^-39 of it is the most.  Where one power serves 32 tokens a row may lie 2^8 lower: 2^-23 and 2^-31 of its largest.  Codes are float16
// numbers as they are and stay exact either way.  Two parts of a query instead of bf16's three: a third of the products less.
//   raw: 16 bytes of a row for every two operand pieces (codes) or one.  power: the token's x from those.  half: a piece of 8
//   dims as float16, times 2^(power - x).
template <typename C>
struct TileKeys;
template <>
struct TileKeys<F16> {
  static constexpr int kRows = kTileF16, kBytes = 2;
  static constexpr bool kPowers = false, kCodes = false;
  static __device__ __forceinline__ va_u32x4 half(va_u32x4 raw, int, int, int) { return raw; }
};
template <>
struct TileKeys<BF16> {
  static constexpr int kRows = kTileF16, kBytes = 2;
  static constexpr bool kPowers = true, kCodes = false;
  static __device__ __forceinline__ va_u32x4 half(va_u32x4 raw, int, int, int x) {
    const float up = power_of_two(-x);
    va_u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = Mma<F16>::pack(__uint_as_float(raw[e] << 16) * up, __uint_as_float(raw[e] & 0xffff0000u) * up);
    return w;
  }
};
template <>
struct TileKeys<E4M3> {
  static constexpr int kRows = kTileCodes, kBytes = 1;
  static constexpr bool kPowers = true, kCodes = true;
  static __device__ __forceinline__ va_u32x4 half(va_u32x4 raw, int b, int power, int x) {
    const float up = power_of_two(power - x);
    va_u32x4 w;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      w[2 * e] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(raw[2 * b + e], up, false));
      w[2 * e + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(raw[2 * b + e], up, true));
    }
    return w;
  }
};
template <>
struct TileKeys<INT8> {
  static constexpr int kRows = kTileCodes, kBytes = 1;
  static constexpr bool kPowers = true, kCodes = true;
  static __device__ __forceinline__ va_u32x4 half(va_u32x4 raw, int b, int power, int x) {
    const float up = power_of_two(power - x);
    va_u32x4 w;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float y[4];
      INT8::unpack4(raw[2 * b + e], y);
      w[2 * e] = Mma<F16>::pack(y[0] * up, y[1] * up), w[2 * e + 1] = Mma<F16>::pack(y[2] * up, y[3] * up);
    }
    return w;
  }
};

template <int kD>
struct TileShape {
  static constexpr int kSteps = kD / 16, kParts = 2;
  static constexpr int kBlocks = VA_WEIGH_TILE_TOKENS / (32 * kWeighWaves);  // of 32 tokens, a wave
  static constexpr int kQueryBytes = VA_WEIGH_TILE_ROWS * kD * 2 * kParts;
  static constexpr int kRowBytes = VA_WEIGH_TILE_ROWS * 16;                  // the rows' other halves, a copy a wave
  static constexpr int kBufferBytes = kQueryBytes + kWeighWaves * kRowBytes;
  static constexpr int kLoads = kQueryBytes / 1024 / kWeighWaves + 1;  // a wave's of a tile of rows
  static constexpr int kFactorsAt = 2 * kBufferBytes;                  // 2^x of the tokens
  static constexpr int kLdsBytes = kFactorsAt + VA_WEIGH_TILE_TOKENS * 4;
  static_assert(kQueryBytes % (1024 * kWeighWaves) == 0, "whole loads");
  static_assert(kFactorsAt >= VA_WEIGH_TILE_TOKENS * 4, "room for the sums");
};

// S^T[32 tokens, 32 rows] by v_mfma_f32_32x32x16: lane l has row l % 32 and tokens 8 (r / 4) + 4 (l / 32) + r % 4.
//
// 4 requests of 300 .. 1500 new tokens of 32 heads of 128 after a prompt of 8000: 730 us, or 985 TFLOP/s of the two parts' products, where
// a large product of bf16 matrices reaches 1264 on the same card.  The matrix cores are busy for 50 % of that time and the vector
// ALU, of which exp2 is two thirds, for 44 %; scores becoming sums while the next tile's products run took more registers
// than there are.  Tiles of 16 rows by 16x16x32 took 720 .. 760 us; with 32 rows a tile and half the barriers 8 readers of 65536 tokens
// take 49 us instead of 62.
template <int kD, typename C>
__device__ __forceinline__ void weigh_tiles(const WeighArgs& a, unsigned block) {
  using Sh = TileShape<kD>;
  using K = TileKeys<C>;
  using Words = const __attribute__((address_space(4))) int32_t*;
  constexpr int kBlocks = Sh::kBlocks, kSteps = Sh::kSteps, kParts = Sh::kParts, kLoads = Sh::kLoads;
  extern __shared__ va_u32x4 smem[];
  char* lds = (char*)smem;
  const ItemHead where = item_and_head(block, a.num_kv_heads);
  const Words item = (Words)a.items + (long long)where.item * VA_WEIGH_ITEM_WORDS;
  const int n_tok = item[VA_WI_N_TOK], hk = where.head;
  if (n_tok == 0) return;
  const int page_begin = item[VA_WI_PAGES], first = item[VA_WI_FIRST], partial = item[VA_WI_PARTIAL];
  const int tile_begin = item[VA_WI_TILE_BEGIN], n_tiles = item[VA_WI_TILE_END] - tile_begin;
  const int lane = threadIdx.x % kWave, j = lane % 32, kg = lane / 32;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const uint32_t lds_base = __builtin_amdgcn_readfirstlane(lds_address(lds));
  const char* queries = a.queries + ((long long)hk * a.n_tiles + 2 * tile_begin) * tile_bytes(kD) + wave * (kLoads - 1) * 1024 + 16 * lane;
  const WeighRow* rows = a.rows + ((long long)hk * a.n_tiles + 2 * tile_begin) * 16 + j;
  auto request = [&](int i) __attribute__((always_inline)) {
    const uint32_t dst = lds_base + (uint32_t)(i % 2) * Sh::kBufferBytes;
#pragma unroll
    for (int u = 0; u < kLoads - 1; ++u)
      load_to_lds(queries + (long long)i * (2 * tile_bytes(kD)) + 1024 * u, dst + (uint32_t)(wave * (kLoads - 1) + u) * 1024);
    if (lane < 32) load_to_lds(rows + (long long)i * VA_WEIGH_TILE_ROWS, dst + Sh::kQueryBytes + Sh::kRowBytes * wave);
  };

  // ---- keys: step s of a block holds dims 16 s + 8 kg .. of token j, or of codes 32 (s / 2) + 16 kg + 8 (s % 2) .. ----
  const int w0 = 32 * kBlocks * wave;  // first token of the wave, in the chunk
  va_u32x4 keys[kBlocks][kSteps];
  float factor[kBlocks];
  float* factors = (float*)(lds + Sh::kFactorsAt) + w0;
  bool even = true;  // one power of two serves each block
  {
    constexpr int kRaw = K::kCodes ? kSteps / 2 : kSteps;
    va_u32x4 raw[kBlocks][kRaw];
    int power[kBlocks], most[kBlocks];
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
      const uint32_t slot = weigh_slot(a, page_begin, first + min(w0 + 32 * b + j, n_tok - 1));
      power[b] = 0;
      if constexpr (K::kCodes) {
        const long long row = quant_row(a.page_map, slot, hk, a.num_kv_heads);
        power[b] = (int)a.k_scales[row] - 127;
#pragma unroll
        for (int s = 0; s < kRaw; ++s) raw[b][s] = *(const va_u32x4*)((const uint8_t*)a.k_pool + row * kD + 32 * s + 16 * kg);
      } else {
        const uint16_t* row = (const uint16_t*)a.k_pool + (long long)slot * a.pool_row_stride + (long long)hk * kD;
#pragma unroll
        for (int s = 0; s < kRaw; ++s) raw[b][s] = *(const va_u32x4*)(row + 16 * s + 8 * kg);
      }
    }
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
      factor[b] = 1.f;
      if constexpr (K::kPowers) {
        // A 16-bit row of 0, and one that is not finite, goes along with the others.  (Over codes a row of 0 has the least scale there
        // is, which counts: beside rows of another size its wave takes the branch with a power for each token.)
        bool counts = power[b] < 128;
        if constexpr (!K::kCodes) {
          uint32_t top = 0;  // magnitudes as whole numbers, which order them
#pragma unroll
          for (int s = 0; s < kRaw; ++s)
#pragma unroll
            for (int e = 0; e < 4; ++e) top = max(top, max(raw[b][s][e] & 0x7fffu, raw[b][s][e] >> 16 & 0x7fffu));
          top = max(top, (uint32_t)__shfl_xor((int)top, 32, kWave));
          counts = top != 0 && top < 0x7f80u;
          power[b] = max((int)(top >> 7) - 127 - 14, -126);
        }
        if (!counts) power[b] = -126;
        most[b] = power[b];
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) most[b] = max(most[b], __shfl_xor(most[b], off, kWave));
        even = even && !__any(counts && power[b] < most[b] - 8);
      }
    }
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
      int x = 0;
      if constexpr (K::kPowers) {
        x = even ? most[b] : power[b];
        factor[b] = power_of_two(x);
        if (!even) factors[32 * b + j] = factor[b];
      }
      bool finite = true;
      if constexpr (K::kCodes) finite = a.k_scales[quant_row(a.page_map, weigh_slot(a, page_begin, first + min(w0 + 32 * b + j, n_tok - 1)), hk, a.num_kv_heads)] != 255;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        keys[b][s] = K::half(raw[b][K::kCodes ? s / 2 : s], s % 2, power[b], x);
        if (K::kCodes && !finite) keys[b][s] = va_u32x4{0x7e007e00u, 0x7e007e00u, 0x7e007e00u, 0x7e007e00u};
        asm volatile("" : "+v"(keys[b][s]));  // (waited for here, not in the loop)
      }
    }
  }

  const int t_wave = first + w0, t_end = min(t_wave + 32 * kBlocks, first + n_tok);
  float sum[kBlocks][16];
#pragma unroll
  for (int b = 0; b < kBlocks; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) sum[b][r] = 0.f;
  request(0);
  for (int i = 0; i < n_tiles; ++i) {
    ring_barrier<0>();  // everyone's part of tile i has landed, and everyone is done with the buffer that tile i + 1 goes to
    if (i + 1 < n_tiles) request(i + 1);
    const char* buffer = lds + (i % 2) * Sh::kBufferBytes;
    const WeighRow row = *(const WeighRow*)(buffer + Sh::kQueryBytes + Sh::kRowBytes * wave + 16 * j);
    if (!__any(row.lo < t_end && row.hi > t_wave && row.scale != 0.f)) continue;
    __builtin_amdgcn_s_setprio(1);  // (before the sums of the SIMD's other wave: 4 prompts' 780 us would be 806)
    va_f32x16 dots[kBlocks];
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) dots[b][r] = 0.f;
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int p = kParts - 1; p >= 0; --p) {
        const va_u32x4 q = *(const va_u32x4*)(buffer + (p * kSteps + s) * 1024 + 16 * lane);
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) dots[b] = Mma<F16>::run32(keys[b][s], q, dots[b]);
      }
    __builtin_amdgcn_s_setprio(0);
    const bool all = !__any(row.lo > t_wave || row.hi < t_end);
    if (all && even) {
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        const float scale = row.scale * factor[b];
#pragma unroll
        for (int r = 0; r < 16; ++r) sum[b][r] += __builtin_amdgcn_exp2f(fmaf(dots[b][r], scale, row.minus_lse));
      }
    } else {  // some row does not see some token, or tokens have powers of their own
#pragma unroll
      for (int b = 0; b < kBlocks; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int at = 32 * b + 8 * (r / 4) + 4 * kg + r % 4, t = t_wave + at;
          float x = factor[b];
          if constexpr (K::kPowers)
            if (!even) x = factors[at];
          const float p = __builtin_amdgcn_exp2f(fmaf(dots[b][r] * x, row.scale, row.minus_lse));
          sum[b][r] += t >= row.lo && t < row.hi ? p : 0.f;
        }
    }
  }
  __syncthreads();
  float* sums = (float*)lds;
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      float x = row_sum(sum[b][r]);
      x += __shfl_xor(x, 16, kWave);
      if (j == r) sums[w0 + 32 * b + 8 * (r / 4) + 4 * kg + r % 4] = x;
    }
  }
  __syncthreads();
  finish_sums(a, page_begin, first, n_tok, partial, hk, sums);
}

template <int kD, typename C>
__global__ __launch_bounds__(kWeighThreads, 2) void weigh_strip_kernel(WeighArgs a) {
  weigh_strip<kD, C>(a, blockIdx.x);
}
template <int kD, typename C>
__global__ __launch_bounds__(kWeighThreads, 2) void weigh_tile_kernel(WeighArgs a) {
  weigh_tiles<kD, C>(a, blockIdx.x);
}
// Both, tile items first.
template <int kD, typename C>
__global__ __launch_bounds__(kWeighThreads, 2) void weigh_both_kernel(WeighArgs a, unsigned tile_blocks) {
  if (blockIdx.x < tile_blocks) weigh_tiles<kD, C>(a, blockIdx.x); else weigh_strip<kD, C>(a, blockIdx.x - tile_blocks);
}

// ---------------------------------------------------------------------------
// vector ALU: any type, alignment and head_dim up to kWeighMaxDim
// ---------------------------------------------------------------------------
constexpr int kWeighBatch = 4;  // rows of a wave at a time

template <typename C>
__global__ __launch_bounds__(kWeighThreads) void weigh_generic_kernel(WeighArgs a) {
  extern __shared__ float lds[];  // [64 tokens][D + 1], then [waves][64]
  const int hk = (int)(blockIdx.x % (unsigned)a.num_kv_heads);
  const int32_t* item = a.items + (long long)(blockIdx.x / (unsigned)a.num_kv_heads) * VA_WEIGH_ITEM_WORDS;
  const int n_tok = item[VA_WI_N_TOK], D = a.head_dim;
  if (n_tok == 0) return;
  const int page_begin = item[VA_WI_PAGES], first = item[VA_WI_FIRST], partial = item[VA_WI_PARTIAL];
  const int tile = blockIdx.x / (unsigned)a.num_kv_heads < (unsigned)a.n_tile_items ? VA_WEIGH_TILE_ROWS : 16;
  const int pair_begin = item[VA_WI_TILE_BEGIN] * tile, pair_end = item[VA_WI_TILE_END] * tile;
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  float* of_waves = lds + 64 * (D + 1);
  for (int t0 = 0; t0 < n_tok; t0 += 64) {
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * D; i += kWeighThreads) {
      const int t = i / D, d = i - t * D;
      const uint32_t slot = weigh_slot(a, page_begin, first + min(t0 + t, n_tok - 1));
      float x;
      if constexpr (std::is_same_v<C, E4M3> || std::is_same_v<C, INT8>) {
        const long long row = quant_row(a.page_map, slot, hk, a.num_kv_heads);
        float y[4];
        C::unpack4(((const uint8_t*)a.k_pool)[row * D + d], y);
        x = y[0] * scale_value(a.k_scales[row]);
      } else {
        x = C::load(((const typename C::storage*)a.k_pool)[(long long)slot * a.pool_row_stride + (long long)hk * D + d]);
      }
      lds[t * (D + 1) + d] = x;
    }
    __syncthreads();
    const int t_span = first + t0 + lane;
    float sum = 0.f;
    for (int pair = pair_begin + wave * kWeighBatch; pair < pair_end; pair += kWeighWaves * kWeighBatch) {
      const float* q = (const float*)(a.queries + ((long long)hk * a.n_tiles + pair / 16) * tile_bytes(D)) + pair % 16 * D;
      float dots[kWeighBatch];
#pragma unroll
      for (int u = 0; u < kWeighBatch; ++u) dots[u] = 0.f;
      for (int d = 0; d < D; ++d) {
        const float k = lds[lane * (D + 1) + d];
#pragma unroll
        for (int u = 0; u < kWeighBatch; ++u) dots[u] = fmaf(k, q[u * D + d], dots[u]);
      }
#pragma unroll
      for (int u = 0; u < kWeighBatch; ++u) {
        const WeighRow row = a.rows[(long long)hk * a.n_tiles * 16 + pair + u];
        const float p = __builtin_amdgcn_exp2f(dots[u] + row.minus_lse);
        sum += t_span >= row.lo && t_span < row.hi ? p : 0.f;
      }
    }
    of_waves[wave * 64 + lane] = sum;
    __syncthreads();
    if (wave == 0 && t0 + lane < n_tok) {
      sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWeighWaves; ++w) sum += of_waves[w * 64 + lane];
      if (partial >= 0) {
        a.partials[hk * a.n_partials + partial + t0 + lane] = sum;
      } else {
        const long long to = hk * a.num_slots + weigh_slot(a, page_begin, t_span);
        a.weights_out[to] = a.weights_in[to] + sum;
      }
    }
  }
}

__global__ __launch_bounds__(kWeighThreads) void weigh_join_kernel(WeighArgs a) {
  const int32_t* join = a.joins + (long long)blockIdx.x * VA_WEIGH_JOIN_WORDS;
  const int n_tok = join[VA_WJ_N_TOK], n_parts = join[VA_WJ_N_PARTS], hk = blockIdx.y;
  for (int t = threadIdx.x; t < n_tok; t += kWeighThreads) {
    const float* from = a.partials + hk * a.n_partials + join[VA_WJ_PARTIAL] + t;
    float sum = 0.f;
    for (int p = 0; p < n_parts; ++p) sum += from[(long long)p * n_tok];
    const long long to = hk * a.num_slots + weigh_slot(a, join[VA_WJ_PAGES], join[VA_WJ_FIRST] + t);
    a.weights_out[to] = a.weights_in[to] + sum;
  }
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
static int weigh_launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? VA_OK : va_fail(VA_ERR_HIP, "%s launch: %s", what, hipGetErrorString(e));
}

// Workgroups over rows from which on a thread goes over several kv heads: 1400 rows of 16 heads of 256 in 25.5 us instead of 29.8, and few
// rows stay spread over the chip (512 .. 8192 measure alike).
constexpr unsigned kRowBlocks = 2048;
template <int kFirst, int kKind>
static void launch_rows(const WeighArgs& a, bool fast, hipStream_t stream) {
  const unsigned hkv = (unsigned)a.num_kv_heads;
  if (fast) {
    const long long tasks = (long long)a.n_tiles * 16 * (a.head_dim / 16);
    const unsigned blocks = (unsigned)((tasks + kWeighThreads - 1) / kWeighThreads);
    hipLaunchKernelGGL((weigh_rows_kernel<kFirst, kKind>), dim3(blocks, std::min(hkv, (kRowBlocks + blocks - 1) / blocks)), dim3(kWeighThreads), 0, stream, a);
  } else {
    hipLaunchKernelGGL((weigh_rows_any_kernel<kFirst, kKind>), dim3((unsigned)a.n_tiles, hkv), dim3(kWeighThreads), 0, stream, a);
  }
}

template <int kD, typename C>
static int launch_matrix(const WeighArgs& a, int n_strips, bool fast, hipStream_t stream) {
  const unsigned tiles = (unsigned)a.n_tile_items * (unsigned)a.num_kv_heads, strips = (unsigned)n_strips * (unsigned)(a.num_kv_heads / strip_heads(a.num_kv_heads));
  const dim3 block(kWeighThreads);
  using Sh = WalkShape<kD, C>;
  if constexpr (std::is_same_v<C, F32>) {
    launch_rows<kParts32, kParts32>(a, fast, stream);
  } else {
    launch_rows<TileKeys<C>::kRows, WalkKeys<C>::kRows>(a, fast, stream);
    if (strips == 0) {
      static std::atomic<unsigned long long> tile_devices{0};
      const hipError_t e = allow_lds(reinterpret_cast<const void*>(&weigh_tile_kernel<kD, C>), TileShape<kD>::kLdsBytes, tile_devices);
      if (e != hipSuccess) return va_fail(VA_ERR_HIP, "raising the LDS limit: %s", hipGetErrorString(e));
      hipLaunchKernelGGL((weigh_tile_kernel<kD, C>), dim3(tiles), block, TileShape<kD>::kLdsBytes, stream, a);
      return weigh_launched("attention weights");
    }
    if (tiles > 0) {
      constexpr int bytes = Sh::kLdsBytes > TileShape<kD>::kLdsBytes ? Sh::kLdsBytes : TileShape<kD>::kLdsBytes;
      static std::atomic<unsigned long long> devices{0};
      const hipError_t e = allow_lds(reinterpret_cast<const void*>(&weigh_both_kernel<kD, C>), bytes, devices);
      if (e != hipSuccess) return va_fail(VA_ERR_HIP, "raising the LDS limit: %s", hipGetErrorString(e));
      hipLaunchKernelGGL((weigh_both_kernel<kD, C>), dim3(tiles + strips), block, bytes, stream, a, tiles);
      return weigh_launched("attention weights");
    }
  }
  static std::atomic<unsigned long long> devices{0};
  const hipError_t e = allow_lds(reinterpret_cast<const void*>(&weigh_strip_kernel<kD, C>), Sh::kLdsBytes, devices);
  if (e != hipSuccess) return va_fail(VA_ERR_HIP, "raising the LDS limit: %s", hipGetErrorString(e));
  hipLaunchKernelGGL((weigh_strip_kernel<kD, C>), dim3(strips), block, Sh::kLdsBytes, stream, a);
  return weigh_launched("attention weights");
}

template <typename C>
static int launch_weigh(const WeighArgs& a, int n_items, int n_strips, bool matrix, bool fast, hipStream_t stream) {
  if (matrix) {
    switch (a.head_dim) {
      case 64:
        return launch_matrix<64, C>(a, n_strips, fast, stream);
      case 128:
        return launch_matrix<128, C>(a, n_strips, fast, stream);
      default:
        return launch_matrix<256, C>(a, n_strips, fast, stream);
    }
  }
  const dim3 grid((unsigned)n_items * (unsigned)a.num_kv_heads), block(kWeighThreads);
  const int bytes = (64 * (a.head_dim + 1) + 64 * kWeighWaves) * 4;
  static std::atomic<unsigned long long> devices{0};
  const hipError_t e = allow_lds(reinterpret_cast<const void*>(&weigh_generic_kernel<C>), (64 * (kWeighMaxDim + 1) + 64 * kWeighWaves) * 4, devices);
  if (e != hipSuccess) return va_fail(VA_ERR_HIP, "raising the LDS limit: %s", hipGetErrorString(e));
  launch_rows<kPlain32, kPlain32>(a, false, stream);
  hipLaunchKernelGGL(weigh_generic_kernel<C>, grid, block, (unsigned)bytes, stream, a);
  return weigh_launched("attention weights");
}

static int weigh(WeighArgs& a, int code_type, int num_pages, const int32_t* plan_dev, const int32_t* h, void* workspace, int64_t workspace_bytes,
                 const VaShape* shape, const VaRope* rope, hipStream_t stream) {
  if (!h || h[VA_WH_MAGIC] != VA_WEIGH_MAGIC) return va_fail(VA_ERR_ARG, "not a plan of attention weights");
  if (h[VA_WH_HQ] != shape->num_q_heads || h[VA_WH_HKV] != shape->num_kv_heads || h[VA_WH_D] != shape->head_dim ||
      h[VA_WH_PAGE] != shape->page_size || h[VA_WH_DTYPE] != shape->dtype || h[VA_WH_CODES] != (code_type >= 0) || h[VA_WH_POOL_PAGES] != num_pages)
    return va_fail(VA_ERR_ARG, "the plan was made for another shape or pool");
  const int n_items = h[VA_WH_N_ITEMS];
  if (n_items == 0) return VA_OK;
  if (!a.q || !a.k_pool || !plan_dev || !a.sub_worker || !a.sub_loc || !a.lse || !a.weights_in || !a.weights_out) return va_fail(VA_ERR_ARG, "null pointer");
  if (shape->head_dim > kWeighMaxDim) return va_fail(VA_ERR_ARG, "head_dim %d is over %d", (int)shape->head_dim, kWeighMaxDim);
  int rc = make_rope(rope, shape->head_dim, &a.rope);
  if (rc) return rc;
  const int G = shape->num_q_heads / shape->num_kv_heads;
  const int64_t pairs = (int64_t)h[VA_WH_N_ROWS] * G, hkv = shape->num_kv_heads;
  const int64_t needed = hkv * (pairs * (6 * (int64_t)shape->head_dim + 16) + 4 * (int64_t)h[VA_WH_N_PARTIALS]);
  if (workspace_bytes < needed) return va_fail(VA_ERR_CAPACITY, "workspace of %lld bytes, %lld are needed", (long long)workspace_bytes, (long long)needed);
  if (!workspace || (uintptr_t)workspace % 16) return va_fail(VA_ERR_ARG, "the workspace must lie on a 16-byte boundary");
  if (hkv > 65535 || h[VA_WH_N_JOINS] < 0) return va_fail(VA_ERR_ARG, "too many heads for one launch");
  a.items = plan_dev + h[VA_WH_OFF_ITEMS];
  a.strips = plan_dev + h[VA_WH_OFF_STRIPS];
  a.joins = plan_dev + h[VA_WH_OFF_JOINS];
  a.pages = plan_dev + h[VA_WH_OFF_PAGES];
  a.sub_rows = plan_dev + h[VA_WH_OFF_ROWS];
  a.n_rows = h[VA_WH_N_ROWS];
  a.lo = a.sub_rows + a.n_rows;
  a.hi = a.lo + a.n_rows;
  a.n_tiles = (int)(pairs / 16);
  a.num_slots = (long long)h[VA_WH_POOL_PAGES] * shape->page_size;
  a.n_partials = h[VA_WH_N_PARTIALS];
  a.queries = (char*)workspace;
  a.rows = (WeighRow*)(a.queries + hkv * pairs * 6 * shape->head_dim);
  a.partials = (float*)(a.rows + hkv * pairs);
  a.num_q_heads = shape->num_q_heads, a.num_kv_heads = shape->num_kv_heads, a.head_dim = shape->head_dim, a.dtype = shape->dtype;
  a.page_map = page_map(shape->page_size);
  a.scale_log2 = kLog2e / sqrtf((float)shape->head_dim);
  const bool dims = shape->head_dim == 64 || shape->head_dim == 128 || shape->head_dim == 256;
  const int size = shape->dtype == VA_F32 ? 4 : 2;
  // (a walk addresses 16 rows of a page with 32-bit offsets)
  const bool matrix = dims && (code_type >= 0 || (a.pool_row_stride * size % 16 == 0 && (uintptr_t)a.k_pool % 16 == 0 && a.pool_row_stride < 1 << 24));
  const bool fast = a.rope.rotary_dim % 16 == 0 && (a.rope.mode != VA_ROPE_TABLE || (uintptr_t)a.rope.cos_sin % 16 == 0);
  a.pieces = a.q_row_stride * size % 16 == 0 && (uintptr_t)a.q % 16 == 0;
  a.n_tile_items = h[VA_WH_N_TILE_ITEMS];
  a.n_first_tiles = (int)((int64_t)h[VA_WH_N_TILE_ROWS] * G / 16);
  if (code_type == VA_CODE_E4M3) {
    rc = launch_weigh<E4M3>(a, n_items, h[VA_WH_N_STRIPS], matrix, fast, stream);
  } else if (code_type == VA_CODE_INT8) {
    rc = launch_weigh<INT8>(a, n_items, h[VA_WH_N_STRIPS], matrix, fast, stream);
  } else {
    switch (shape->dtype) {
      case VA_F32:
        rc = launch_weigh<F32>(a, n_items, h[VA_WH_N_STRIPS], matrix, fast, stream);
        break;
      case VA_F16:
        rc = launch_weigh<F16>(a, n_items, h[VA_WH_N_STRIPS], matrix, fast, stream);
        break;
      case VA_BF16:
        rc = launch_weigh<BF16>(a, n_items, h[VA_WH_N_STRIPS], matrix, fast, stream);
        break;
      default:
        rc = va_fail(VA_ERR_ARG, "unknown dtype %d", (int)shape->dtype);
    }
  }
  if (rc || h[VA_WH_N_JOINS] == 0) return rc;
  hipLaunchKernelGGL(weigh_join_kernel, dim3((unsigned)h[VA_WH_N_JOINS], (unsigned)hkv), dim3(kWeighThreads), 0, stream, a);
  return weigh_launched("joining attention weights");
}

}  // namespace va

extern "C" int va_weigh(const void* q_dev, int64_t q_row_stride, const void* k_pool_dev, int64_t pool_row_stride, int32_t num_pages,
                        const int32_t* plan_dev, const int32_t* plan_header_host, const int64_t* sub_worker_dev, const int64_t* sub_loc_dev,
                        int64_t sub_loc_axis_stride, const float* lse_dev, int32_t lse_base2, const float* weights_in_dev, float* weights_out_dev,
                        void* workspace_dev, int64_t workspace_bytes, const VaShape* shape, const VaRope* rope, void* stream) {
  if (!shape || shape->num_kv_heads <= 0 || shape->num_q_heads <= 0 || shape->num_q_heads % shape->num_kv_heads || shape->head_dim <= 0 || shape->page_size <= 0)
    return va_fail(VA_ERR_ARG, "bad shape");
  if (pool_row_stride < (int64_t)shape->num_kv_heads * shape->head_dim) return va_fail(VA_ERR_ARG, "pool rows overlap");
  va::WeighArgs a{};
  a.q = q_dev, a.q_row_stride = q_row_stride, a.k_pool = k_pool_dev, a.pool_row_stride = pool_row_stride, a.sub_worker = sub_worker_dev;
  a.sub_loc = sub_loc_dev, a.sub_loc_axis_stride = sub_loc_axis_stride, a.lse = lse_dev, a.lse_base2 = lse_base2;
  a.weights_in = weights_in_dev, a.weights_out = weights_out_dev;
  return va::weigh(a, -1, num_pages, plan_dev, plan_header_host, workspace_dev, workspace_bytes, shape, rope, (hipStream_t)stream);
}

extern "C" int va_weigh_q8(const void* q_dev, int64_t q_row_stride, const VaQuantPool* pool, const int32_t* plan_dev, const int32_t* plan_header_host,
                           const int64_t* sub_worker_dev, const int64_t* sub_loc_dev, int64_t sub_loc_axis_stride, const float* lse_dev,
                           int32_t lse_base2, const float* weights_in_dev, float* weights_out_dev, void* workspace_dev, int64_t workspace_bytes,
                           const VaShape* shape, const VaRope* rope, void* stream) {
  const int rc = va::check_quant_pool(pool, shape);
  if (rc) return rc;
  if (shape->num_q_heads <= 0 || shape->num_q_heads % shape->num_kv_heads) return va_fail(VA_ERR_ARG, "bad shape");
  va::WeighArgs a{};
  a.q = q_dev, a.q_row_stride = q_row_stride, a.k_pool = pool->k_codes_dev, a.k_scales = pool->k_scales_dev, a.sub_worker = sub_worker_dev;
  a.sub_loc = sub_loc_dev, a.sub_loc_axis_stride = sub_loc_axis_stride, a.lse = lse_dev, a.lse_base2 = lse_base2;
  a.weights_in = weights_in_dev, a.weights_out = weights_out_dev;
  return va::weigh(a, pool->code_type, pool->num_pages, plan_dev, plan_header_host, workspace_dev, workspace_bytes, shape, rope, (hipStream_t)stream);
}
