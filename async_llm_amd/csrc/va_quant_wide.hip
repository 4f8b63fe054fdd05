// Matrix-core view attention over a quantised pool for many new tokens: query tiles of 128 (head_dim 256) or 256 MFMA rows.
//
// Bound by the instructions around the matrix products, not by memory: a tile of tokens is read once for all rows of a
// workgroup.  So where the streaming kernel (va_quant_stream.hip) spends two products on an operand, this one spends one, in
// float16, whose eleven bits put less error on a result than its rounding to bf16 does:
//
//   S^T[32 tokens, 16 rows] = K . Q^T      v_mfma_f32_16x16x32_f16; codes are exact in float16.  Queries are turned and scaled
//                                          in fp32 and multiplied by a power of two that puts the largest of the wave's
//                                          rows under 2^14: elements 2^28 times smaller keep all their bits.
//   p = exp2(S * 2^e_k - max + 13)         the maximum is raised when a tile exceeds it by a factor of two
//   w = p * 2^(e_v - E)                    E: the largest e_v so far, one less at most: w <= 2^15, and a weight keeps its bits
//                                          down to 2^-27 of the row's largest
//   O^T[D, 16 rows] += V^T . W^T           (in units of 2^E)
//
// Eight waves, two per SIMD, so that one's exponentials run beside the other's products; each owns one (head_dim 256) or two
// blocks of sixteen rows, row = tile row R / G, head R % G.  All walk the same 32-token tiles, which travel to a ring of four
// buffers in LDS as codes (every wave brings an eighth of a tile), one barrier a tile; each wave converts the codes for its
// own products, once for both of its blocks.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "va_internal.h"
#include "va_launch.h"
#include "va_mfma_common.h"
#include "va_quant.h"
#include "va_quant_attn.h"
#include "va_quant_mfma.h"

namespace va {

constexpr int kWideQThreads = 512;
constexpr int kWideQWaves = 8;
constexpr int kWideQBuffers = 4;
constexpr float kWideQOffset = 13.f;  // log2 of the weight of a row's largest score
constexpr float kWideQRaise = 1.f;    // how far (log2) a tile may exceed the maximum

template <int kD>
struct WideQ {
  static constexpr int kBlocks = kD == 256 ? 1 : 2;
  static constexpr int kRows = 16 * kBlocks;  // of a wave
  static constexpr int kPieces = kD / 64;
  static constexpr int kSteps = kD / 32;
  static constexpr int kDimTiles = kD / 16;
  static constexpr int kHalfBytes = 16 * kD;
  static constexpr int kTileBytes = 4 * kHalfBytes;     // K, then V
  static constexpr int kTileLoads = kTileBytes / 1024;  // wave-level loads: 4, 8 or 16
  static constexpr int kWaveLoads = kTileLoads >= kWideQWaves ? kTileLoads / kWideQWaves : 1;  // of the waves that load
  static constexpr int kBufferBytes = kTileBytes + 64 * 4;  // and a word per scale
  static constexpr int kQueryOffset = kWideQBuffers * kBufferBytes;
  static constexpr int kQueryBytes = kRows * kD * 2;  // of a wave
  static constexpr int kUnits = kRows * (kD / 16) / kWave;  // query units (two pieces of eight dims) a lane turns
  static constexpr int kLdsBytes = kQueryOffset + kWideQWaves * kQueryBytes;
  static_assert(kLdsBytes <= 160 * 1024, "the LDS of a CU");
};

__device__ __forceinline__ void wait_tiles(int loads_of_two_tiles) {  // (the same for a whole wave)
  switch (loads_of_two_tiles) {
    case 0: break;
    case 2: wave_wait_loads<2>(); break;
    case 4: wave_wait_loads<4>(); break;
    default: wave_wait_loads<6>(); break;
  }
}

template <int kD, typename C>
__global__ __launch_bounds__(kWideQThreads, 1) void attn_quant_wide_kernel(QuantAttnArgs qa, int dtype, int pieces) {
  const AttnArgs& a = qa.a;
  using W = WideQ<kD>;
  using Words = const __attribute__((address_space(4))) int32_t*;
  constexpr int kBlocks = W::kBlocks, kPieces = W::kPieces, kSteps = W::kSteps, kDimTiles = W::kDimTiles;

  extern __shared__ va_u32x4 smem[];
  char* lds = (char*)smem;

  // Workgroup -> (slot, kv head): the slots of a die run in groups of up to 32 under one kv head at a time, so that its L2
  // holds one head's stream.
  int slot, hk;
  {
    const unsigned die = blockIdx.x & 7u, turn = blockIdx.x >> 3, per_die = gridDim.x / (8u * a.num_kv_heads);
    unsigned g = 32;
    while (per_die % g) g >>= 1;
    const unsigned block = turn / (g * a.num_kv_heads), within = turn % (g * a.num_kv_heads);
    slot = (int)((block * g + within % g) * 8u + die);
    hk = (int)(within / g);
  }
  const int item_begin = ((Words)a.wide_slots)[slot], item_end = ((Words)a.wide_slots)[slot + 1];
  const int G = a.num_q_heads / a.num_kv_heads;
  const int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int j = lane % 16, kg = lane / 16;
  const int row0 = wave * W::kRows;
  int row_iq[kBlocks];
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) row_iq[b] = (row0 + 16 * b + j) / G;
  const uint8_t* kp = (const uint8_t*)a.k_pool;
  const uint8_t* vp = (const uint8_t*)a.v_pool;
  const int P = a.page_size, p_shift = qa.pages.shift;
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_address(lds));
  char* query = lds + W::kQueryOffset + wave * W::kQueryBytes;

  // This wave's loads of a tile: load n of the tile fills its bytes [1024 n, + 1024).
  constexpr int kRowPieces = kD / 16;
  const int first_load = wave * W::kWaveLoads;
  const bool loads = first_load < W::kTileLoads, loads_scales = wave == kWideQWaves - 1;
  const int two_tiles = 2 * ((loads ? W::kWaveLoads : 0) + (loads_scales ? 1 : 0));
  int ld_half[W::kWaveLoads], ld_row[W::kWaveLoads];
  uint32_t ld_off[W::kWaveLoads];
#pragma unroll
  for (int n = 0; n < W::kWaveLoads; ++n) {
    const int load = first_load + n, in_half = load % (W::kHalfBytes / 1024);
    ld_half[n] = load / (W::kHalfBytes / 1024);  // K first, K second, V first, V second
    ld_row[n] = in_half * (64 / kRowPieces) + lane / kRowPieces;
    ld_off[n] = (uint32_t)(ld_row[n] * kD + 16 * ((lane % kRowPieces) ^ ring_swz<kD>(16 * (ld_half[n] & 1) + ld_row[n])));
  }
  int k_at[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) k_at[h] = 16 * (kg ^ ring_swz<kD>(16 * h + j));
  const int v_token = (j / 2 < 4 ? 0 : 12) + 4 * kg + j / 2;
  const int v_at = 2 * W::kHalfBytes + v_token * kD + 8 * (j % 2), v_swz = 16 * ring_swz<kD>(v_token);

  for (int it = item_begin; it < item_end; ++it) {
    const Words item = (Words)a.items + (long long)it * VA_ITEM_WORDS;
    const int n_q = item[VA_I_N_Q], n_links = item[VA_I_N_LINKS], part_base = item[VA_I_PART_BASE];
    if (n_q == 0) continue;
    float m_run[kBlocks], l_run[kBlocks];
    va_f32x4 o[kBlocks][kDimTiles];
    int e_ref = 0;  // scale byte of the units of o
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
      m_run[b] = kNegBig;
      l_run[b] = 0.f;
#pragma unroll
      for (int t = 0; t < kDimTiles; ++t) o[b][t] = va_f32x4{0.f, 0.f, 0.f, 0.f};
    }

    for (int li = 0; li < n_links; ++li) {
      const Words link = li == 0 ? item + VA_I_LINK0 : (Words)a.links + (long long)(item[VA_I_LINK_BEGIN] + li) * VA_LINK_WORDS;
      const int lflags = link[VA_L_FLAGS], kv_begin = link[VA_L_KV_BEGIN], tok_begin = link[VA_L_TOK_BEGIN];
      const int tok_end = link[VA_L_TOK_END], causal_base = link[VA_L_CAUSAL_BASE], qref = link[VA_L_QREF];
      const bool slots = lflags & VA_LINK_SLOTS, whole = !slots && tok_begin % 16 == 0;
      const int t_stop = min(tok_end, causal_base + n_q), t_last = t_stop - 1;
      const int n_tiles = t_stop > tok_begin ? (t_stop - tok_begin + kQuantTokens - 1) / kQuantTokens : 0;
      int t_row[kBlocks];
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) t_row[b] = min(tok_end, causal_base + row_iq[b] + 1);
      // tokens that all rows of the wave see, and that any of them does
      const int t_all = min(tok_end, causal_base + row0 / G + 1);
      const int t_any = row0 / G < n_q ? min(t_stop, causal_base + min(n_q - 1, (row0 + W::kRows - 1) / G) + 1) : 0;

      auto row_of = [&](int t) __attribute__((always_inline)) {  // of token t, looked up by a lane
        const int at = min(t, t_last), entry = a.kv_indices[kv_begin + (slots ? at : at >> p_shift)];
        const int page = slots ? entry >> p_shift : entry, place = (slots ? entry : at) & (P - 1);
        return ((long long)page * a.num_kv_heads + hk) * P + place;
      };
      // first row of a half of tile i, and its last visible row
      auto half_row = [&](int i, int h) __attribute__((always_inline)) {
        const int t = min(tok_begin + i * kQuantTokens + 16 * h, t_last);
        return ((long long)((Words)a.kv_indices)[kv_begin + (t >> p_shift)] * a.num_kv_heads + hk) * P + (t & (P - 1));
      };
      auto request = [&](int i) __attribute__((always_inline)) {
        const uint32_t dst = lds0 + (uint32_t)(i % kWideQBuffers) * W::kBufferBytes;
        const int t0 = tok_begin + i * kQuantTokens;
        if (loads) {
#pragma unroll
          for (int n = 0; n < W::kWaveLoads; ++n) {
            const int h = ld_half[n] & 1;
            const uint8_t* pool = ld_half[n] < 2 ? kp : vp;
            const uint32_t at = dst + (uint32_t)(first_load + n) * 1024;
            if (whole) {
              const int most = max(0, t_last - (t0 + 16 * h));
              load_to_lds(pool + half_row(i, h) * kD, ld_off[n] - (uint32_t)(max(0, ld_row[n] - most) * kD), at);
            } else {
              load_to_lds(pool + row_of(t0 + 16 * h + ld_row[n]) * kD + (ld_off[n] - ld_row[n] * kD), at);
            }
          }
        }
        if (loads_scales) {
          const uint8_t* of = lane < 32 ? qa.k_scales : qa.v_scales;
          long long row;
          if (whole) {
            const long long r0 = half_row(i, 0), r1 = half_row(i, 1);
            row = (kg & 1 ? r1 : r0) + min(j, max(0, t_last - (t0 + 16 * (kg & 1))));
          } else {
            row = row_of(t0 + lane % 32);
          }
          load_bytes_to_lds((unsigned long long)of + row, dst + W::kTileBytes);
        }
      };

      // every wave has read the tiles and scales of the link before
      ring_barrier<kAnyInFlight>();
#pragma unroll
      for (int i = 0; i < kWideQBuffers - 1; ++i)
        if (i < n_tiles) request(i);

      // ---- the wave's query rows: turned, scaled, and as float16 in LDS and then in registers ----
      float q_inv;  // what a product with them is multiplied by
      {
        float y[W::kUnits][2][8];
        uint32_t top = 0;
#pragma unroll
        for (int n = 0; n < W::kUnits; ++n) {
          const int idx = n * kWave + lane, r = idx / kRowPieces, x = idx % kRowPieces, iq = (row0 + r) / G, g = row0 + r - iq * G;
          const int pairs = a.rope.rotary_dim / 16;
          const int d0 = x < pairs ? 8 * x : 16 * x, d1 = x < pairs ? 8 * x + a.rope.half : 16 * x + 8;
#pragma unroll
          for (int e = 0; e < 8; ++e) y[n][0][e] = y[n][1][e] = 0.f;
          if (iq < n_q) {
            const bool indirect = lflags & VA_LINK_INDIRECT;
            const int subrow = indirect ? a.qrefs[qref + iq] : qref + iq;
            const long long src = indirect ? (long long)a.qref_rows[qref + iq] : a.sub_worker[subrow];
            const long long at = src * a.q_row_stride + (long long)(hk * G + g) * kD;
            activations8(a.q, at + d0, dtype, pieces, y[n][0]);
            activations8(a.q, at + d1, dtype, pieces, y[n][1]);
            if (x < pairs) {
              float c[8], s[8];
              turns8(a.rope, load_pos(a.sub_loc, a.sub_loc_axis_stride, subrow), d0, c, s);
              turn8(c, s, y[n][0], y[n][1]);
            }
          }
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              y[n][i][e] *= a.scale_log2;
              const uint32_t bits = __float_as_uint(y[n][i][e]) & 0x7fffffffu;
              if (bits < 0x7f800000u) top = max(top, bits);  // (a row that is not finite stays so by itself)
            }
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, off, kWave));
        const int up = min(126, max(-126, 127 + 13 - (int)(top >> 23)));  // the largest: from 2^13 on, under 2^14
        const float scale = __uint_as_float((uint32_t)(127 + up) << 23);
        q_inv = __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
        for (int n = 0; n < W::kUnits; ++n) {
          const int idx = n * kWave + lane, r = idx / kRowPieces, x = idx % kRowPieces;
          const int pairs = a.rope.rotary_dim / 16;
          const int d0 = x < pairs ? 8 * x : 16 * x, d1 = x < pairs ? 8 * x + a.rope.half : 16 * x + 8;
          va_u32x4 w[2];
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) w[i][e] = Mma<F16>::pack(y[n][i][2 * e] * scale, y[n][i][2 * e + 1] * scale);
          *(va_u32x4*)(query + r * (2 * kD) + 16 * ((d0 / 8) ^ (r & 7))) = w[0];
          *(va_u32x4*)(query + r * (2 * kD) + 16 * ((d1 / 8) ^ (r & 7))) = w[1];
        }
      }
      // (the wave's own rows: its LDS operations stay in order)
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      va_u32x4 q[kBlocks][kSteps];
#pragma unroll
      for (int b = 0; b < kBlocks; ++b)
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
          q[b][s] = staged_query<kD>(query + b * 16 * 2 * kD, s);
          asm volatile("" : "+v"(q[b][s]));
        }

      // ---- the tile loop ----
      for (int i = 0; i < n_tiles; ++i) {
        // this wave's part of the tile has landed once at most those of the two tiles behind it are outstanding
        if (i + 2 < n_tiles) {
          wait_tiles(two_tiles);
        } else {
          wave_wait_loads<0>();
        }
        ring_barrier<kAnyInFlight>();  // everyone's part has, and everyone has read the tile before
        if (i + kWideQBuffers - 1 < n_tiles) request(i + kWideQBuffers - 1);
        const int t0 = tok_begin + i * kQuantTokens;
        if (t0 >= t_any) continue;
        const uint32_t buffer = (uint32_t)(i % kWideQBuffers) * W::kBufferBytes;
        const char* tile = lds + buffer;

        va_f32x4 acc[kBlocks][2];
#pragma unroll
        for (int b = 0; b < kBlocks; ++b)
#pragma unroll
          for (int h = 0; h < 2; ++h) acc[b][h] = va_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < kPieces; ++s) {
          va_u32x4 raw[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) raw[h] = *(const va_u32x4*)(tile + h * W::kHalfBytes + j * kD + (k_at[h] ^ (64 * s)));
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const va_u32x4 k8 = C::f16x8(u ? va_u32x2{raw[h][2], raw[h][3]} : va_u32x2{raw[h][0], raw[h][1]});
#pragma unroll
              for (int b = 0; b < kBlocks; ++b) acc[b][h] = Mma<F16>::run(k8, q[b][2 * s + u], acc[b][h]);
            }
        }
        // scales of this lane's tokens 16 h + 4 kg + r
        float ks[2][4], vs[2][4];
        {
          uint32_t most = 0;
          va_u32x4 vb[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const va_u32x4 kb = *(const va_u32x4*)(tile + W::kTileBytes + 64 * h + 16 * kg);
            vb[h] = *(const va_u32x4*)(tile + W::kTileBytes + 128 + 64 * h + 16 * kg);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              ks[h][r] = scale_value(kb[r]) * q_inv;
              most = max(most, vb[h][r] == 255u ? 0u : vb[h][r]);
            }
          }
          if (__any((int)most > e_ref + 1)) {  // larger values than so far: o changes its units
#pragma unroll
            for (int off = 16; off < kWave; off <<= 1) most = max(most, (uint32_t)__shfl_xor((int)most, off, kWave));
            const int next = __builtin_amdgcn_readfirstlane((int)most);
            const float down = __uint_as_float((uint32_t)max(0, 127 + e_ref - next) << 23);
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
#pragma unroll
              for (int t = 0; t < kDimTiles; ++t) o[b][t] *= down;
            e_ref = next;
          }
          const float unit = __uint_as_float((uint32_t)(254 - e_ref) << 23);  // 2^(127 - e_ref)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 4; ++r) vs[h][r] = scale_value(vb[h][r]) * unit;
        }

        va_u32x4 w[kBlocks];
        const bool masked = t0 + kQuantTokens > t_all;
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
          float sc[2][4], most = -INFINITY;
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 4; ++r) sc[h][r] = acc[b][h][r] * ks[h][r];
          if (masked) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (t0 + 16 * h + 4 * kg + r >= t_row[b]) sc[h][r] = -INFINITY;
          }
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 4; ++r) most = fmaxf(most, sc[h][r]);
          if (__any(most > m_run[b] + kWideQRaise)) {
            const float m_new = fmaxf(m_run[b], quant_group_max(most));
            const float alpha = __builtin_amdgcn_exp2f(m_run[b] - m_new);
            m_run[b] = m_new;
            l_run[b] *= alpha;
#pragma unroll
            for (int t = 0; t < kDimTiles; ++t) o[b][t] *= alpha;
          }
          const float base = kWideQOffset - m_run[b];
          float p[2][4];
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              p[h][r] = __builtin_amdgcn_exp2f(sc[h][r] + base);
              l_run[b] += p[h][r];
              p[h][r] *= vs[h][r];
            }
          if (masked) {  // (a token that the row does not see may have any scale)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (t0 + 16 * h + 4 * kg + r >= t_row[b]) p[h][r] = 0.f;
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            w[b][2 * h] = Mma<F16>::pack(p[h][0], p[h][1]);
            w[b][2 * h + 1] = Mma<F16>::pack(p[h][2], p[h][3]);
          }
        }
#pragma unroll
        for (int t = 0; t < kDimTiles; ++t) {
          const va_u32x4 v8 = C::f16x8(lds_read_tr8(lds0 + buffer + v_at + ((16 * t) ^ v_swz)));
#pragma unroll
          for (int b = 0; b < kBlocks; ++b) o[b][t] = Mma<F16>::run(v8, w[b], o[b][t]);
        }
      }
    }

    // ---- results: o[b][t][r] is dim 16 t + 4 kg + r of row row0 + 16 b + j, in units of 2^(e_ref - 127) ----
    const int flags0 = item[VA_I_LINK0 + VA_L_FLAGS], qref0 = item[VA_I_LINK0 + VA_L_QREF];
    const float unit = scale_value((uint32_t)e_ref);
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
      float l = l_run[b];
      l += __shfl_xor(l, 16, kWave);
      l += __shfl_xor(l, 32, kWave);
      const int iq = row_iq[b];
      if (iq >= n_q) continue;
      const float m = m_run[b] - kWideQOffset;
      const int hq = hk * G + row0 + 16 * b + j - iq * G;
      if (part_base < 0) {
        const long long out_row = (flags0 & VA_LINK_INDIRECT) ? (long long)a.qref_rows[qref0 + iq] : a.sub_worker[qref0 + iq];
        const long long at = (out_row * a.num_q_heads + hq) * (long long)kD;
#pragma unroll
        for (int t = 0; t < kDimTiles; ++t) {
          float y[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) y[k] = normalised(o[b][t][k], l) * unit;
          store_results4(a.out, at + 16 * t + 4 * kg, y, dtype, pieces);
        }
        if (kg == 0 && a.lse) a.lse[out_row * a.num_q_heads + hq] = log_sum(m, l, a.lse_base2);
      } else {
        const long long state = (long long)(part_base + iq) * a.num_q_heads + hq;
#pragma unroll
        for (int t = 0; t < kDimTiles; ++t) *(va_f32x4*)(a.part_acc + state * kD + 16 * t + 4 * kg) = o[b][t] * unit;
        if (kg == 0) {
          a.part_ml[state * 2 + 0] = m;
          a.part_ml[state * 2 + 1] = l;
        }
      }
    }
  }
}

template <int kD, typename C>
static int launch_quant_wide_one(const QuantAttnArgs& qa, int dtype, int n_slots, int pieces, hipStream_t stream) {
  const dim3 grid((unsigned)n_slots * (unsigned)qa.a.num_kv_heads), block(kWideQThreads);
  constexpr int bytes = WideQ<kD>::kLdsBytes;
  static std::atomic<unsigned long long> devices{0};
  hipError_t e = allow_lds(reinterpret_cast<const void*>(&attn_quant_wide_kernel<kD, C>), bytes, devices);
  if (e != hipSuccess) return va_fail(VA_ERR_HIP, "raising the LDS limit: %s", hipGetErrorString(e));
  hipLaunchKernelGGL((attn_quant_wide_kernel<kD, C>), grid, block, bytes, stream, qa, dtype, pieces);
  e = hipGetLastError();
  return e == hipSuccess ? VA_OK : va_fail(VA_ERR_HIP, "quantised attention launch: %s", hipGetErrorString(e));
}

template <typename C>
static int launch_quant_wide_coded(const QuantAttnArgs& qa, int dtype, int n_slots, int pieces, hipStream_t stream) {
  switch (qa.a.head_dim) {
    case 64:
      return launch_quant_wide_one<64, C>(qa, dtype, n_slots, pieces, stream);
    case 128:
      return launch_quant_wide_one<128, C>(qa, dtype, n_slots, pieces, stream);
    default:
      return launch_quant_wide_one<256, C>(qa, dtype, n_slots, pieces, stream);
  }
}

int launch_quant_wide(const QuantAttnArgs& qa, int dtype, int code_type, int n_slots, int pieces, hipStream_t stream) {
  return code_type == VA_CODE_E4M3 ? launch_quant_wide_coded<E4M3>(qa, dtype, n_slots, pieces, stream)
                                   : launch_quant_wide_coded<INT8>(qa, dtype, n_slots, pieces, stream);
}

}  // namespace va
