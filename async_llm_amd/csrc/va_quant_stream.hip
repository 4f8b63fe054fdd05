// Matrix-core view attention over a quantised pool: query tiles of up to 16 MFMA rows (decode tiles of 16 / G requests that
// read the same tokens, and prefill tiles of 16 / G new tokens), row = tile row R / G, head R % G.
//
//   S^T[32 tokens, 16 rows] = K . Q^T      v_mfma_f32_16x16x32_bf16; the codes of K as the A operand, converted to bf16
//                                          (exact) in the registers they were loaded to
//   p = exp2(S * 2^e_k * scale - max),     w = p * 2^e_v
//   O^T[D, 16 rows] += V^T . W^T           the same product; V^T from transposing LDS reads of the codes
//
// Operands that are not codes are split into two bf16 numbers, x = hi + lo with an error of 2^-17 of x, and each product is
// taken twice: rounded to one bf16 a query or a weight would put an error of the size of the result's own rounding on it (a
// float16 result would lose three bits).  The range of bf16 is why no scale has to be normalised: w is whatever p * 2^e_v is.
// The matrix pipe has the time, the kernel is bound by HBM.
//
// Four independent waves a workgroup, each takes every fourth 32-token tile of the walk with loads of its own: no barrier in
// the tile loop.  K goes from memory straight to the registers that feed the products: lane (j, kg) of a 16-token half
// takes bytes [64 s + 16 kg, + 16) of token j, which are the contraction elements of steps 2 s and 2 s + 1 when the query is
// laid out by the same order.  V passes through LDS (eight tokens of a dim in one ds_read_b64_tr_b8).  Both are requested a
// tile ahead, V while the tile before is taken apart, K behind its last product; page entries two tiles ahead.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "va_internal.h"
#include "va_launch.h"
#include "va_mfma_common.h"
#include "va_quant.h"
#include "va_quant_attn.h"

namespace va {

constexpr int kQuantThreads = 256;
constexpr int kQuantWaves = 4;
constexpr int kQuantTokens = 32;  // tokens per tile

template <int kD>
struct QuantShape {
  static constexpr int kPieces = kD / 64;    // 16-byte pieces of a token's row that a lane takes
  static constexpr int kSteps = kD / 32;     // contraction steps of K.Q^T
  static constexpr int kDimTiles = kD / 16;  // 16-dim tiles of the output
  static constexpr int kTileBytes = kQuantTokens * kD;         // V of a tile
  static constexpr int kWaveBytes = kTileBytes + 2 * kQuantTokens * 4;  // and its scales, K then V
  static constexpr int kQueryBytes = 2 * 16 * kD * 2;          // hi and lo rows
  static constexpr int kLoopBytes = kQuantWaves * kWaveBytes + kQueryBytes;
  // The waves' states at the end: accumulators (rows padded by 16 bytes), maxima and sums.
  static constexpr int kFoldRowBytes = kD * 4 + 16;
  static constexpr int kFoldBytes = 16 * (kFoldRowBytes + 8);
  static constexpr int kLdsBytes = kLoopBytes > kQuantWaves * kFoldBytes ? kLoopBytes : kQuantWaves * kFoldBytes;
};

// Piece c of token t of a V tile lies at position c ^ quant_swz(t): the sixteen tokens that a write covers spread over the
// banks, and so do the eight that a transposing read takes of one piece.
template <int kD>
__device__ __forceinline__ int quant_swz(int t) {
  if constexpr (kD == 256) return (t & 3) | (((t >> 4) & 1) << 2) | (((t >> 2) & 1) << 3);
  if constexpr (kD == 128) return ((t >> 1) & 3) | (((t >> 4) & 1) << 2);
  return ((t >> 2) & 3) ^ ((t >> 4) & 1);
}

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

template <int kD, typename C>
__global__ __launch_bounds__(kQuantThreads, kD == 256 ? 1 : 2) void attn_quant_stream_kernel(QuantAttnArgs qa, int dtype, int pieces) {
  const AttnArgs& a = qa.a;
  using Sh = QuantShape<kD>;
  constexpr int kPieces = Sh::kPieces, kSteps = Sh::kSteps, kDimTiles = Sh::kDimTiles;

  extern __shared__ va_u32x4 smem[];
  char* lds = (char*)smem;

  const ItemHead where = item_and_head(blockIdx.x, a.num_kv_heads);
  using Words = const __attribute__((address_space(4))) int32_t*;
  const Words item = (Words)a.items + (long long)where.item * VA_ITEM_WORDS;
  const int n_q = item[VA_I_N_Q], n_links = item[VA_I_N_LINKS], part_base = item[VA_I_PART_BASE];
  if (n_q == 0) return;  // padding item: keeps the launch order aligned with the die round-robin
  const int hk = where.head, G = a.num_q_heads / a.num_kv_heads;
  const int tid = threadIdx.x, lane = tid % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int j = lane % 16, kg = lane / 16;  // MFMA row (token of a half tile, query row), contraction group
  const int row_iq = j / G;
  const uint8_t* kp = (const uint8_t*)a.k_pool;
  const uint8_t* vp = (const uint8_t*)a.v_pool;

  char* mine = lds + wave * Sh::kWaveBytes;
  float* scales = (float*)(mine + Sh::kTileBytes);  // [2][32]: K, V
  char* query = lds + kQuantWaves * Sh::kWaveBytes;
  // where this lane's pieces of V go, and where it reads them transposed
  int v_write[2][kPieces];
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int s = 0; s < kPieces; ++s) v_write[u][s] = (16 * u + j) * kD + 16 * ((4 * s + kg) ^ quant_swz<kD>(16 * u + j));
  const int v_token = (j / 2 < 4 ? 0 : 12) + 4 * kg + j / 2;  // tokens 4 kg .. + 3, then 16 + 4 kg .. + 3
  const uint32_t v_read = lds_address(mine) + v_token * kD + 8 * (j % 2);
  const int v_swz = quant_swz<kD>(v_token);

  float m_run = kNegBig, l_run = 0.f;  // running maximum (log2 units) and sum, of this wave's tokens
  va_f32x4 o[kDimTiles];
#pragma unroll
  for (int t = 0; t < kDimTiles; ++t) o[t] = va_f32x4{0.f, 0.f, 0.f, 0.f};

  for (int li = 0; li < n_links; ++li) {
    const Words link = li == 0 ? item + VA_I_LINK0 : (Words)a.links + (long long)(item[VA_I_LINK_BEGIN] + li) * VA_LINK_WORDS;
    const int lflags = link[VA_L_FLAGS], kv_begin = link[VA_L_KV_BEGIN], tok_begin = link[VA_L_TOK_BEGIN];
    const int tok_end = link[VA_L_TOK_END], causal_base = link[VA_L_CAUSAL_BASE], qref = link[VA_L_QREF];
    const bool slots = lflags & VA_LINK_SLOTS;
    const int t_stop = min(tok_end, causal_base + n_q);      // tokens any row of the tile sees
    const int t_row = min(tok_end, causal_base + row_iq + 1);  // tokens this lane's row sees
    const int t_last = t_stop - 1;
    const int n_all = t_stop > tok_begin ? (t_stop - tok_begin + kQuantTokens - 1) / kQuantTokens : 0;
    const int n_tiles = n_all > wave ? (n_all - wave + kQuantWaves - 1) / kQuantWaves : 0;  // this wave's
    auto first_token = [&](int i) __attribute__((always_inline)) { return tok_begin + (i * kQuantWaves + wave) * kQuantTokens; };

    // Tokens of a half tile, past the visible range the last visible one (masked): its entry of the index, then its row.
    auto token_of = [&](int i, int u) __attribute__((always_inline)) { return min(first_token(i) + 16 * u + j, t_last); };
    int entry[2];
    auto read_entries = [&](int i) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint32_t t = (uint32_t)token_of(i, u);
        uint32_t page = t, place;
        if (!slots) qa.pages.split(t, page, place);
        entry[u] = a.kv_indices[kv_begin + (int)page];
      }
    };
    long long row[2];
    auto rows_of = [&](int i) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        uint32_t page = (uint32_t)entry[u], place;
        if (slots) {
          qa.pages.split((uint32_t)entry[u], page, place);
        } else {
          uint32_t ahead;
          qa.pages.split((uint32_t)token_of(i, u), ahead, place);
        }
        row[u] = ((long long)page * a.num_kv_heads + hk) * qa.pages.size + place;
      }
    };
    va_u32x4 kraw[2][kPieces], vraw[2][kPieces];
    uint32_t scale_byte;
    auto load_v = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int s = 0; s < kPieces; ++s) vraw[u][s] = *(const va_u32x4*)(vp + row[u] * kD + 64 * s + 16 * kg);
      // lanes 0 .. 31 the scales of the 32 keys, the others those of the values
      scale_byte = (lane < 32 ? qa.k_scales : qa.v_scales)[row[kg & 1]];
    };
    auto load_k = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int s = 0; s < kPieces; ++s) kraw[u][s] = *(const va_u32x4*)(kp + row[u] * kD + 64 * s + 16 * kg);
    };
    if (n_tiles > 0) {
      read_entries(0);
      rows_of(0);
      read_entries(1);
      load_v();
      load_k();
      rows_of(1);
    }

    // ---- the query rows, rotated in fp32 and split, in LDS: piece c of row r at position c ^ (r & 7) ----
    if (li > 0) __syncthreads();  // every wave has read the previous link's
    for (int idx = tid; idx < 16 * (kD / 16); idx += kQuantThreads) {
      const int r = idx / (kD / 16), x = idx - r * (kD / 16), iq = r / G, g = r - iq * G;
      const int pairs = a.rope.rotary_dim / 16;
      const int d0 = x < pairs ? 8 * x : 16 * x, d1 = x < pairs ? 8 * x + a.rope.half : 16 * x + 8;
      float y0[8], y1[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y0[e] = y1[e] = 0.f;
      if (iq < n_q) {
        const bool indirect = lflags & VA_LINK_INDIRECT;
        const int subrow = indirect ? a.qrefs[qref + iq] : qref + iq;
        const long long src = indirect ? (long long)a.qref_rows[qref + iq] : a.sub_worker[subrow];
        const long long at = src * a.q_row_stride + (long long)(hk * G + g) * kD;
        activations8(a.q, at + d0, dtype, pieces, y0);
        activations8(a.q, at + d1, dtype, pieces, y1);
        if (x < pairs) {
          float c[8], s[8];
          turns8(a.rope, load_pos(a.sub_loc, a.sub_loc_axis_stride, subrow), d0, c, s);
          turn8(c, s, y0, y1);
        }
      }
      va_u32x4 h0, l0, h1, l1;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t hi, lo;
        split_pair(y0[2 * e], y0[2 * e + 1], hi, lo);
        h0[e] = hi, l0[e] = lo;
        split_pair(y1[2 * e], y1[2 * e + 1], hi, lo);
        h1[e] = hi, l1[e] = lo;
      }
      char* q_row = query + r * (2 * kD);
      const int c0 = 16 * ((d0 / 8) ^ (r & 7)), c1 = 16 * ((d1 / 8) ^ (r & 7));
      *(va_u32x4*)(q_row + c0) = h0;
      *(va_u32x4*)(q_row + c1) = h1;
      *(va_u32x4*)(q_row + 32 * kD + c0) = l0;
      *(va_u32x4*)(q_row + 32 * kD + c1) = l1;
    }
    __syncthreads();
    // B operands: step 2 s + b holds dims [64 s + 16 kg + 8 b, + 8) of row j
    va_u32x4 q_hi[kSteps], q_lo[kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const char* at = query + j * (2 * kD) + 16 * ((8 * (s / 2) + 2 * kg + s % 2) ^ (j & 7));
      q_hi[s] = *(const va_u32x4*)at;
      q_lo[s] = *(const va_u32x4*)(at + 32 * kD);
    }

    // ---- the tile loop ----
    for (int i = 0; i < n_tiles; ++i) {
      // V and the scales to LDS, and the next ones on their way
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int s = 0; s < kPieces; ++s) *(va_u32x4*)(mine + v_write[u][s]) = vraw[u][s];
      scales[lane] = scale_value(scale_byte);
      asm volatile("" ::: "memory");
      if (i + 1 < n_tiles) {
        load_v();
        read_entries(i + 2);
      }

      va_f32x4 hi[2], lo[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) hi[u] = lo[u] = va_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const va_u32x4 raw = kraw[u][s / 2];
          const va_u32x4 k8 = C::bf16x8(s % 2 ? va_u32x2{raw[2], raw[3]} : va_u32x2{raw[0], raw[1]});
          hi[u] = Mma<BF16>::run(k8, q_hi[s], hi[u]);
          lo[u] = Mma<BF16>::run(k8, q_lo[s], lo[u]);
        }
      }
      if (i + 1 < n_tiles) load_k();

      // online softmax; this lane holds tokens 16 u + 4 kg + r of row j
      const int t0 = first_token(i);
      float sc[2][4], vs[2][4], most = -INFINITY;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const va_f32x4 ks = *(const va_f32x4*)(scales + 16 * u + 4 * kg), v4 = *(const va_f32x4*)(scales + 32 + 16 * u + 4 * kg);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const bool seen = t0 + 16 * u + 4 * kg + r < t_row;
          sc[u][r] = seen ? (hi[u][r] + lo[u][r]) * (ks[r] * a.scale_log2) : -INFINITY;
          vs[u][r] = seen ? v4[r] : 0.f;
          most = fmaxf(most, sc[u][r]);
        }
      }
      if (__any(most > m_run)) {
        const float m_new = fmaxf(m_run, quant_group_max(most));
        const float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
        m_run = m_new;
        l_run *= alpha;
#pragma unroll
        for (int t = 0; t < kDimTiles; ++t) o[t] *= alpha;
      }
      va_u32x4 w_hi, w_lo;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float w[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float p = __builtin_amdgcn_exp2f(sc[u][r] - m_run);
          l_run += p;
          w[r] = p * vs[u][r];
        }
        uint32_t h, l;
        split_pair(w[0], w[1], h, l);
        w_hi[2 * u] = h, w_lo[2 * u] = l;
        split_pair(w[2], w[3], h, l);
        w_hi[2 * u + 1] = h, w_lo[2 * u + 1] = l;
      }

      // O^T += V^T . W^T, the lane's contraction elements being tokens 4 kg .. + 3 and 16 + 4 kg .. + 3
#pragma unroll
      for (int t = 0; t < kDimTiles; ++t) {
        const va_u32x4 v8 = C::bf16x8(lds_read_tr8(v_read + 16 * (t ^ v_swz)));
        o[t] = Mma<BF16>::run(v8, w_hi, o[t]);
        o[t] = Mma<BF16>::run(v8, w_lo, o[t]);
      }
      asm volatile("" ::: "memory");
      if (i + 1 < n_tiles) rows_of(i + 2);
    }
  }

  // ---- the four waves' states are folded through LDS: o[t][r] is dim 16 t + 4 kg + r of row j ----
  l_run += __shfl_xor(l_run, 16, kWave);
  l_run += __shfl_xor(l_run, 32, kWave);
  __syncthreads();  // every wave is done with its tiles and the query
  {
    char* state = lds + wave * Sh::kFoldBytes;
#pragma unroll
    for (int t = 0; t < kDimTiles; ++t) *(va_f32x4*)(state + j * Sh::kFoldRowBytes + 16 * kg + 64 * t) = o[t];
    if (kg == 0) *(float2*)(state + 16 * Sh::kFoldRowBytes + 8 * j) = make_float2(m_run, l_run);
  }
  __syncthreads();
  const int r = tid / 16, seg = tid % 16, iq = r / G;
  if (iq >= n_q) return;
  float weight[kQuantWaves], m = kNegBig, l = 0.f;
  float2 ml[kQuantWaves];
#pragma unroll
  for (int w = 0; w < kQuantWaves; ++w) {
    ml[w] = *(const float2*)(lds + w * Sh::kFoldBytes + 16 * Sh::kFoldRowBytes + 8 * r);
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
      sum[x] += *(const va_f32x4*)(lds + w * Sh::kFoldBytes + r * Sh::kFoldRowBytes + 16 * (seg + 16 * x)) * weight[w];
  }
  if (part_base < 0) {
    const Words link0 = item + VA_I_LINK0;
    const int qref0 = link0[VA_L_QREF];
    const long long out_row = (link0[VA_L_FLAGS] & VA_LINK_INDIRECT) ? (long long)a.qref_rows[qref0 + iq] : a.sub_worker[qref0 + iq];
    const long long at = (out_row * a.num_q_heads + hq) * (long long)kD;
#pragma unroll
    for (int x = 0; x < kD / 64; ++x) {
      const int d = 4 * (seg + 16 * x);
      float y[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) y[k] = normalised(sum[x][k], l);
      if (pieces) {
        const bool bf = dtype == VA_BF16;
        const uint2 w = make_uint2(bf ? Mma<BF16>::pack(y[0], y[1]) : Mma<F16>::pack(y[0], y[1]),
                                   bf ? Mma<BF16>::pack(y[2], y[3]) : Mma<F16>::pack(y[2], y[3]));
        *(uint2*)((uint16_t*)a.out + at + d) = w;
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) store_activation(a.out, at + d + k, y[k], dtype);
      }
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

template <int kD, typename C>
static int launch_quant_stream_one(const QuantAttnArgs& qa, int dtype, int n_items, int pieces, hipStream_t stream) {
  const dim3 grid((unsigned)n_items * (unsigned)qa.a.num_kv_heads), block(kQuantThreads);
  constexpr int bytes = QuantShape<kD>::kLdsBytes;
  static std::atomic<unsigned long long> devices{0};
  hipError_t e = allow_lds(reinterpret_cast<const void*>(&attn_quant_stream_kernel<kD, C>), bytes, devices);
  if (e != hipSuccess) return va_fail(VA_ERR_HIP, "raising the LDS limit: %s", hipGetErrorString(e));
  hipLaunchKernelGGL((attn_quant_stream_kernel<kD, C>), grid, block, bytes, stream, qa, dtype, pieces);
  e = hipGetLastError();
  return e == hipSuccess ? VA_OK : va_fail(VA_ERR_HIP, "quantised attention launch: %s", hipGetErrorString(e));
}

template <typename C>
static int launch_quant_stream_coded(const QuantAttnArgs& qa, int dtype, int n_items, int pieces, hipStream_t stream) {
  switch (qa.a.head_dim) {
    case 64:
      return launch_quant_stream_one<64, C>(qa, dtype, n_items, pieces, stream);
    case 128:
      return launch_quant_stream_one<128, C>(qa, dtype, n_items, pieces, stream);
    default:
      return launch_quant_stream_one<256, C>(qa, dtype, n_items, pieces, stream);
  }
}

int launch_quant_stream(const QuantAttnArgs& qa, int dtype, int code_type, int n_items, int q_tile, hipStream_t stream) {
  const AttnArgs& a = qa.a;
  const int g = a.num_q_heads / a.num_kv_heads;
  if (!va_mfma_supported(dtype, a.head_dim, g))
    return va_fail(VA_ERR_ARG, "matrix-core path does not support this dtype/head_dim/group size");
  if (q_tile * g > 16) return va_fail(VA_ERR_ARG, "plan tile of %d rows x %d heads exceeds 16 MFMA rows", q_tile, g);
  if (a.rope.rotary_dim % 16) return va_fail(VA_ERR_ARG, "matrix-core path needs rotary_dim to be a multiple of 16");
  if (a.rope.mode == VA_ROPE_TABLE && a.rope.rotary_dim > 0 && (uintptr_t)a.rope.cos_sin % 16)
    return va_fail(VA_ERR_ARG, "matrix-core path needs a 16-byte aligned cos|sin table");
  if ((uintptr_t)a.part_acc % 16) return va_fail(VA_ERR_ARG, "matrix-core path needs a 16-byte aligned workspace");
  // queries and results in 16-byte (8-byte) accesses where their addresses allow it
  const int pieces = a.q_row_stride % 8 == 0 && (uintptr_t)a.q % 16 == 0 && (uintptr_t)a.out % 8 == 0;
  return code_type == VA_CODE_E4M3 ? launch_quant_stream_coded<E4M3>(qa, dtype, n_items, pieces, stream)
                                   : launch_quant_stream_coded<INT8>(qa, dtype, n_items, pieces, stream);
}

}  // namespace va
