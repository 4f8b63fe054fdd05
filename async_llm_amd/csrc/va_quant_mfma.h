// Matrix-core pieces of view attention over a quantised pool, shared by the kernels for whole and for scattered tiles.
#pragma once
#include <hip/hip_runtime.h>

#include "va_mfma_common.h"
#include "va_quant.h"
#include "va_quant_attn.h"

namespace va {

constexpr int kQuantThreads = 256;
constexpr int kQuantWaves = 4;
constexpr int kQuantTokens = 32;  // tokens per tile
// How far (log2) a score may lie above the running reference before sums are rescaled to it.  Weights up to 2^8 lose nothing: they
// are split into two bf16 numbers and summed in fp32, whose errors are relative (what they cost is range: sums overflow for
// values over 2^119 instead of 2^127 divided by their number).  Maxima of 16 rows rise in most tiles
// of a walk, and each time all of O^T is multiplied (64 of 400 vector instructions a tile at 256 dims).
constexpr float kQuantLeap = 8.f;

__device__ __forceinline__ va_u32x2 lds_read_tr8(uint32_t lds_byte_address) {
  typedef int v2i __attribute__((ext_vector_type(2)));
  // Within 16 lanes, lane s supplies the address of eight bytes; lane i receives byte i of every 16: byte i % 8 of what
  // lanes i / 8, i / 8 + 2, ... pointed at.
  const v2i r = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) v2i*)(uintptr_t)lds_byte_address);
  return __builtin_bit_cast(va_u32x2, r);
}

// x as the sum of two bf16 numbers, pairs packed.
__device__ __forceinline__ void split_pair(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = Mma<BF16>::pack(a, b);
  lo = Mma<BF16>::pack(a - __uint_as_float(hi << 16), b - __uint_as_float(hi & 0xffff0000u));
}

__device__ __forceinline__ float quant_group_max(float x) {  // over lanes l, l ^ 16, l ^ 32, l ^ 48
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// Eight activations from `at` on as fp32; `pieces`: rows lie on 16-byte boundaries.
__device__ __forceinline__ void activations8(const void* x, long long at, int dtype, bool pieces, float* y) {
  if (pieces) {
    const va_u32x4 w = *(const va_u32x4*)((const uint16_t*)x + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint16_t a = (uint16_t)w[i], b = (uint16_t)(w[i] >> 16);
      y[2 * i] = dtype == VA_BF16 ? BF16::load(a) : __half2float(__builtin_bit_cast(__half, a));
      y[2 * i + 1] = dtype == VA_BF16 ? BF16::load(b) : __half2float(__builtin_bit_cast(__half, b));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = activation(x, at + i, dtype);
  }
}

// Piece c of token t of a tile lies at position c ^ ring_swz(t).  Sixteen tokens' pieces c (a fragment of K), and the piece
// that a transposing read takes of tokens 4 k .. + 3 and 16 + 4 k .. + 3 (V), then lie in different banks.
template <int kD>
__device__ __forceinline__ int ring_swz(int t) {
  if constexpr (kD == 256) return (t & 15) ^ (((t >> 4) & 1) << 2);
  if constexpr (kD == 128) return ((t >> 1) & 7) ^ (((t >> 4) & 1) << 1);
  return ((t >> 2) & 3) ^ ((t >> 4) & 1);
}

// A byte per lane, each a word in LDS: lane l's lands at lds_base + 4 l.
__device__ __forceinline__ void load_bytes_to_lds(unsigned long long at, uint32_t lds_base) {
  uint32_t saved;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_ubyte %1, off\n\ts_mov_b32 m0, %0"
               : "=&s"(saved)
               : "v"(at), "s"(lds_base)
               : "memory");
}

// Wait until at most n of the wave's vector memory operations are outstanding.
template <int n>
__device__ __forceinline__ void wave_wait_loads() {
  static_assert(n < kAnyInFlight, "the counter holds no more");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(n) : "memory");
}

// The query rows of a tile for a link, rotated in fp32, scaled (scores are powers of two from here on) and split into two
// bf16 numbers: this thread's two pieces of eight
// dims of a row, high parts and low parts.  (16 rows of kD / 16 units: at 64 and 128 dims some threads have none.)
struct QueryPieces {
  va_u32x4 part[2][2];  // [high, low][piece]
  int row, d[2];        // row -1: no unit
};
// Where a thread's query row lies and what it is turned by: asked for ahead of its use.
struct QuerySource {
  int row, unit, g;  // row of the tile (-1: no unit), unit of the row, q head of the kv head
  long long at;      // query row, or -1
  Pos3 pos;
};
template <int kD>
__device__ __forceinline__ QuerySource query_source(const AttnArgs& a, int n_q, int lflags, int qref) {
  static_assert(16 * (kD / 16) <= kQuantThreads, "a unit a thread");
  const int G = a.num_q_heads / a.num_kv_heads, r = threadIdx.x / (kD / 16), iq = r / G;
  QuerySource s{r < 16 ? r : -1, (int)(threadIdx.x % (kD / 16)), r - iq * G, -1, Pos3{0, 0, 0}};
  if (r < 16 && iq < n_q) {
    const bool indirect = lflags & VA_LINK_INDIRECT;
    const int subrow = indirect ? a.qrefs[qref + iq] : qref + iq;
    s.at = indirect ? (long long)a.qref_rows[qref + iq] : a.sub_worker[subrow];
    if (a.rope.rotary_dim) s.pos = load_pos(a.sub_loc, a.sub_loc_axis_stride, subrow);
  }
  return s;
}
template <int kD>
__device__ __forceinline__ QueryPieces turned_query(const AttnArgs& a, const QuerySource& from, int hk, int dtype, bool pieces) {
  const int G = a.num_q_heads / a.num_kv_heads, x = from.unit, pairs = a.rope.rotary_dim / 16;
  QueryPieces q;
  q.row = from.row;
  q.d[0] = x < pairs ? 8 * x : 16 * x;
  q.d[1] = x < pairs ? 8 * x + a.rope.half : 16 * x + 8;
  float y[2][8];
#pragma unroll
  for (int e = 0; e < 8; ++e) y[0][e] = y[1][e] = 0.f;
  if (from.at >= 0) {
    const long long at = from.at * a.q_row_stride + (long long)(hk * G + from.g) * kD;
    float c[8], s[8];
    if (x < pairs) turns8(a.rope, from.pos, q.d[0], c, s);
    activations8(a.q, at + q.d[0], dtype, pieces, y[0]);
    activations8(a.q, at + q.d[1], dtype, pieces, y[1]);
    if (x < pairs) turn8(c, s, y[0], y[1]);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[0][e] *= a.scale_log2, y[1][e] *= a.scale_log2;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      uint32_t hi, lo;
      split_pair(y[i][2 * e], y[i][2 * e + 1], hi, lo);
      q.part[0][i][e] = hi, q.part[1][i][e] = lo;
    }
  return q;
}
// High or low parts in LDS (kD * 32 bytes): piece c of row r at position c ^ (r & 7).
template <int kD>
__device__ __forceinline__ void stage_query(const QueryPieces& q, int part, char* query) {
  if (q.row < 0) return;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    *(va_u32x4*)(query + q.row * (2 * kD) + 16 * ((q.d[i] / 8) ^ (q.row & 7))) = part == 0 ? q.part[0][i] : q.part[1][i];
}
// B operands of K.Q^T: step 2 s + b holds dims [64 s + 16 kg + 8 b, + 8) of row j.
template <int kD>
__device__ __forceinline__ va_u32x4 staged_query(const char* query, int step) {
  const int j = threadIdx.x % 16, kg = (threadIdx.x % kWave) / 16;
  return *(const va_u32x4*)(query + j * (2 * kD) + 16 * ((8 * (step / 2) + 2 * kg + step % 2) ^ (j & 7)));
}

// Four neighbouring results at `at`.
__device__ __forceinline__ void store_results4(void* out, long long at, const float* y, int dtype, bool pieces) {
  if (pieces) {
    const bool bf = dtype == VA_BF16;
    *(uint2*)((uint16_t*)out + at) = make_uint2(bf ? Mma<BF16>::pack(y[0], y[1]) : Mma<F16>::pack(y[0], y[1]),
                                                bf ? Mma<BF16>::pack(y[2], y[3]) : Mma<F16>::pack(y[2], y[3]));
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) store_activation(out, at + k, y[k], dtype);
  }
}

// The state of a tile at the end: four waves', folded through LDS, then the result or the partial state.  o[t][r] is dim
// 16 t + 4 kg + r of row j, l_run a sum spread over the four contraction groups.
template <int kD>
struct QuantFold {
  static constexpr int kRowBytes = kD * 4 + 16;  // (padded, so that the sixteen rows of a write spread over the banks)
  static constexpr int kBytes = 16 * (kRowBytes + 8);
};
template <int kD>
__device__ __forceinline__ void fold_and_finish(const AttnArgs& a, const va_f32x4 (&o)[kD / 16], float m_run, float l_run, char* lds,
                                                int n_q, int part_base, int qref0, int flags0, int hk, int dtype, bool pieces) {
  using F = QuantFold<kD>;
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave, j = lane % 16, kg = lane / 16;
  const int G = a.num_q_heads / a.num_kv_heads;
  l_run += __shfl_xor(l_run, 16, kWave);
  l_run += __shfl_xor(l_run, 32, kWave);
  {
    char* state = lds + wave * F::kBytes;
#pragma unroll
    for (int t = 0; t < kD / 16; ++t) *(va_f32x4*)(state + j * F::kRowBytes + 16 * kg + 64 * t) = o[t];
    if (kg == 0) *(float2*)(state + 16 * F::kRowBytes + 8 * j) = make_float2(m_run, l_run);
  }
  __syncthreads();
  const int r = tid / 16, seg = tid % 16, iq = r / G;
  if (iq >= n_q) return;
  float weight[kQuantWaves], m = kNegBig, l = 0.f;
  float2 ml[kQuantWaves];
#pragma unroll
  for (int w = 0; w < kQuantWaves; ++w) {
    ml[w] = *(const float2*)(lds + w * F::kBytes + 16 * F::kRowBytes + 8 * r);
    m = fmaxf(m, ml[w].x);
  }
#pragma unroll
  for (int w = 0; w < kQuantWaves; ++w) {
    weight[w] = __builtin_amdgcn_exp2f(ml[w].x - m);
    l += ml[w].y * weight[w];
  }
  const int hq = hk * G + r - iq * G;
  va_f32x4 sum[kD / 64];
#pragma unroll
  for (int x = 0; x < kD / 64; ++x) {
    sum[x] = va_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kQuantWaves; ++w)
      sum[x] += *(const va_f32x4*)(lds + w * F::kBytes + r * F::kRowBytes + 16 * (seg + 16 * x)) * weight[w];
  }
  if (part_base < 0) {
    const long long out_row = (flags0 & VA_LINK_INDIRECT) ? (long long)a.qref_rows[qref0 + iq] : a.sub_worker[qref0 + iq];
    const long long at = (out_row * a.num_q_heads + hq) * (long long)kD;
#pragma unroll
    for (int x = 0; x < kD / 64; ++x) {
      const int d = 4 * (seg + 16 * x);
      float y[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) y[k] = normalised(sum[x][k], l);
      store_results4(a.out, at + d, y, dtype, pieces);
    }
    if (seg == 0 && a.lse) a.lse[out_row * a.num_q_heads + hq] = log_sum(m, l, a.lse_base2);
  } else {
    const long long slot = (long long)(part_base + iq) * a.num_q_heads + hq;
    float* prow = a.part_acc + slot * kD;
#pragma unroll
    for (int x = 0; x < kD / 64; ++x) *(va_f32x4*)(prow + 4 * (seg + 16 * x)) = sum[x];
    if (seg == 0) {
      a.part_ml[slot * 2 + 0] = m;
      a.part_ml[slot * 2 + 1] = l;
    }
  }
}

}  // namespace va
