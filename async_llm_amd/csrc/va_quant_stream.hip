// Matrix-core view attention over a quantised pool: query tiles of up to 16 MFMA rows (decode tiles of 16 / G requests that
// read the same tokens, and prefill tiles of 16 / G new tokens), row = tile row R / G, head R % G.
//
//   S^T[32 tokens, 16 rows] = K . Q^T      v_mfma_f32_16x16x32_bf16, the codes of K as the A operand, converted to bf16 (exact;
//                                          the conversion of e4m3 takes 2^e_k along)
//   p = exp2(S * 2^e_k - max),     w = p * 2^e_v          (Q scaled by log2(e) / sqrt(D))
//   O^T[D, 16 rows] += V^T . W^T           the same product; V^T from transposing LDS reads of the codes
//
// Operands that are not codes are split into two bf16 numbers, x = hi + lo with an error of 2^-17 of x, and each product is
// taken twice: rounded to one bf16 a query or a weight would put an error of the size of the result's own rounding on it (a
// float16 result would lose three bits).  The range of bf16 is why no scale has to be normalised: w is whatever p * 2^e_v is.
// The matrix pipe has the time, the kernel is bound by HBM.
//
// Four independent waves a workgroup, each takes every fourth 32-token tile of the walk and brings it global -> LDS
// (global_load_lds) into a ring of its own: no barrier in the tile loop.  A tile is two halves of sixteen tokens, each one run
// of 16 * D bytes of a page, for K and for V: whole lines, requested non-temporally where no other tile reads them (6.8 TB/s for
// loads alone; as half lines straight to registers, which the products of K would take, 5.7).  A tile goes from LDS to
// registers at once, K before its products and V behind them, and its half of the buffer is requested anew: one buffer is
// enough, and two workgroups (three at 128, four at 64 dims) share a CU, so that an item's set-up and fold, about 5 us, run beside the
// walks of others.  (One workgroup with two buffers and two tiles that walk the same tokens, as the 16-bit kernel has them:
// 64 requests over a shared prompt 204 -> 247 us, 16 of short blocks 26 -> 36, a chunk of 333 tokens 97 -> 149; eight of 131072
// tokens 340 either way.)  8 requests of 131072 tokens 336 us (6.4 TB/s), 64 over 8192 shared tokens and blocks of 256..8192 191
// (1.04 GB from HBM; the prompt's sixteen tiles read 0.27 more from L2).
#include <hip/hip_runtime.h>

#include <type_traits>

#include "va_internal.h"
#include "va_launch.h"
#include "va_mfma_common.h"
#include "va_quant.h"
#include "va_quant_attn.h"
#include "va_quant_mfma.h"

namespace va {

template <int kD>
struct QuantRing {
  static constexpr int kPieces = kD / 64;       // 16-byte pieces of a token's row that a lane takes
  static constexpr int kSteps = kD / 32;        // contraction steps of K.Q^T
  static constexpr int kDimTiles = kD / 16;     // 16-dim tiles of the output
  static constexpr int kHalfBytes = 16 * kD;    // sixteen tokens of K (or V)
  static constexpr int kLoads = kHalfBytes / 1024;      // wave-level loads of a half
  static constexpr int kTileBytes = 4 * kHalfBytes;     // K, then V
  static constexpr int kScaleBytes = 64 * 4;            // a word per scale: 32 keys', 32 values'
  // Ring depth of a wave, in tiles.  Two at 64 dims, where LDS has the room: us with one / two, 8 requests of 60 k tokens 110 / 107,
  // 22 of 2 k shared and up to 14 k 45.2 / 44.5; 64 rows over 32768 shared tokens 222 / 232, over 1024 and short blocks 46.4 / 47.6.
  static constexpr int kBuffers = kD == 64 ? 2 : 1;
  static constexpr int kScaleSlots = 2 * kBuffers;      // scales stay in LDS while their tile is in registers
  static constexpr int kMinBlocks = kD == 64 ? 4 : kD == 128 ? 3 : 2;  // workgroups per CU
  static constexpr int kScaleOffset = kBuffers * kTileBytes;
  static constexpr int kWaveBytes = kScaleOffset + kScaleSlots * kScaleBytes;
  static constexpr int kQueryOffset = kQuantWaves * kWaveBytes;
  // Low parts of the query in registers, where there are any to spare (read from LDS for each tile at 128 dims: 28 rows of 7 k
  // shared and up to 16 k tokens 94.7 us instead of 92.5).
  static constexpr bool kKeepLow = kD < 256;
  static constexpr int kQueryBytes = (kKeepLow ? 2 : 1) * 16 * kD * 2;  // parts of a tile's query
  static constexpr int kLdsBytes = kQueryOffset + kQueryBytes;
  static_assert(kQuantWaves * QuantFold<kD>::kBytes <= kLdsBytes, "room for the waves' states");
  static_assert(kMinBlocks * kLdsBytes <= 160 * 1024, "the LDS of a CU");
  static constexpr int kLoadsPerTile = 4 * kLoads + 1;  // what the counter of outstanding loads sees of a tile
};

// One wave-level load of 1 KB with a cache policy (load_to_lds has none).
template <bool kOnce>
__device__ __forceinline__ void load_run_to_lds(const void* base, uint32_t lane_offset, uint32_t lds_base) {
  uint32_t saved;
#define VA_ONE_LOAD(policy)                                                                                              \
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" policy "\n\ts_mov_b32 m0, %0" \
               : "=&s"(saved)                                                                                            \
               : "v"(lane_offset), "s"(base), "s"(lds_base)                                                              \
               : "memory")
  if constexpr (kOnce) VA_ONE_LOAD(" nt"); else VA_ONE_LOAD("");
#undef VA_ONE_LOAD
}
template <int kD, typename C>
__device__ __forceinline__ void quant_stream_item(const QuantAttnArgs& qa, int dtype, int pieces) {
  const AttnArgs& a = qa.a;
  using Sh = QuantRing<kD>;
  using Words = const __attribute__((address_space(4))) int32_t*;
  constexpr int kPieces = Sh::kPieces, kSteps = Sh::kSteps, kDimTiles = Sh::kDimTiles, kLoads = Sh::kLoads, kBuffers = Sh::kBuffers;

  extern __shared__ va_u32x4 smem[];
  char* lds = (char*)smem;

  const ItemHead where = item_and_head(blockIdx.x, a.num_kv_heads);
  const Words item = (Words)a.items + (long long)where.item * VA_ITEM_WORDS;
  const int n_q = item[VA_I_N_Q], n_links = item[VA_I_N_LINKS], link_begin = item[VA_I_LINK_BEGIN], part_base = item[VA_I_PART_BASE];
  if (n_q == 0) return;  // padding item: keeps the launch order aligned with the die round-robin
  const int hk = where.head, G = a.num_q_heads / a.num_kv_heads;
  const int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int j = lane % 16, kg = lane / 16;  // MFMA row (token of a half, query row), contraction group
  const int row_iq = j / G;
  const uint8_t* kp = (const uint8_t*)a.k_pool;
  const uint8_t* vp = (const uint8_t*)a.v_pool;
  const int P = a.page_size, p_shift = qa.pages.shift;

  // This lane's part of wave-level load u of a half: row and piece, the piece that belongs at its LDS position; the
  // halves' swizzles differ by a bit of the position.  Loads of a group share one setting of M0, whose immediate offsets move
  // the pool address as well (grouped_lane_offset; the base gives the bias back).
  constexpr int kRowPieces = kD / 16;
  constexpr int kBias = 1024 * (kLoads - 1);
  auto ld_row = [&](int u) __attribute__((always_inline)) { return u * (64 / kRowPieces) + lane / kRowPieces; };
  auto ld_piece = [&](int u, int half) __attribute__((always_inline)) {
    return (lane % kRowPieces) ^ ring_swz<kD>(16 * half + ld_row(u));
  };
  uint32_t ld_off[2][kLoads];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int u = 0; u < kLoads; ++u)
      ld_off[h][u] = grouped_lane_offset((uint32_t)(ld_row(u) * kD + 16 * ld_piece(u, h) + kBias), u);
  // What it reads of a tile.  K: pieces 4 s + kg of token j of each half.  V: piece t of eight tokens, transposed.
  int k_at[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) k_at[h] = 16 * (kg ^ ring_swz<kD>(16 * h + j));
  const int v_token = (j / 2 < 4 ? 0 : 12) + 4 * kg + j / 2;  // tokens 4 kg .. + 3, then 16 + 4 kg .. + 3
  const int v_at = 2 * Sh::kHalfBytes + v_token * kD + 8 * (j % 2), v_swz = 16 * ring_swz<kD>(v_token);
  const uint32_t ring = __builtin_amdgcn_readfirstlane(lds_address(lds)) + (uint32_t)wave * Sh::kWaveBytes;
  char* query = lds + Sh::kQueryOffset;

  float m_run = kNegBig, l_run = 0.f;  // running maximum (log2 units) and sum, of this wave's tokens
  va_f32x4 o[kDimTiles];
#pragma unroll
  for (int t = 0; t < kDimTiles; ++t) o[t] = va_f32x4{0.f, 0.f, 0.f, 0.f};

  for (int li = 0; li < n_links; ++li) {
    const Words link = li == 0 ? item + VA_I_LINK0 : (Words)a.links + (long long)(link_begin + li) * VA_LINK_WORDS;
    const int lflags = link[VA_L_FLAGS], kv_begin = link[VA_L_KV_BEGIN], tok_begin = link[VA_L_TOK_BEGIN];
    const int tok_end = link[VA_L_TOK_END], causal_base = link[VA_L_CAUSAL_BASE], qref = link[VA_L_QREF];
    const bool slots = lflags & VA_LINK_SLOTS;
    const bool read_once = lflags & VA_LINK_ONCE;  // no other tile reads these rows: lines to evict first
    const bool whole = !slots && tok_begin % 16 == 0;  // halves lie inside a page
    const int t_stop = min(tok_end, causal_base + n_q);        // tokens any row of the tile sees
    const int t_row = min(tok_end, causal_base + row_iq + 1);  // tokens this lane's row sees
    const int t_all = min(tok_end, causal_base + 1);           // tokens every row sees
    const int t_last = t_stop - 1;
    const int n_all = t_stop > tok_begin ? (t_stop - tok_begin + kQuantTokens - 1) / kQuantTokens : 0;
    const int n_tiles = n_all > wave ? (n_all - wave + kQuantWaves - 1) / kQuantWaves : 0;  // this wave's
    auto first_token = [&](int i) __attribute__((always_inline)) { return tok_begin + (i * kQuantWaves + wave) * kQuantTokens; };
    // pages of tile i, read a tile ahead of its request (in scalar loads: a vector one would be waited for with all others)
    auto read_pages = [&](int i, int (&page)[2]) __attribute__((always_inline)) {
#pragma unroll
      for (int h = 0; h < 2; ++h) page[h] = ((Words)a.kv_indices)[kv_begin + (min(first_token(i) + 16 * h, t_last) >> p_shift)];
    };
    auto request_half = [&](const uint8_t* pool, long long base, const uint32_t* off, uint32_t dst, auto once) __attribute__((always_inline)) {
      const void* from = pool + (base - kBias);
      if constexpr (kLoads == 1) {
        load_run_to_lds<decltype(once)::value>(from, off[0], dst);
      } else {
        load_group_to_lds<kLoads, decltype(once)::value>(from, off, dst);
      }
    };
    // Request K (kind 0), or V and the scales (1), of tile i into buffer i % kBuffers.  Rows past the visible range repeat
    // the last visible token (masked).
    auto request = [&](int i, const int (&page)[2], auto kind) __attribute__((always_inline)) {
      constexpr int v = decltype(kind)::value;
      const uint8_t* pool = v ? vp : kp;
      const uint32_t dst = ring + (uint32_t)(i % kBuffers) * Sh::kTileBytes + v * 2 * Sh::kHalfBytes;
      const uint32_t scales = ring + Sh::kScaleOffset + (uint32_t)(i % Sh::kScaleSlots) * Sh::kScaleBytes;
      const uint8_t* of_scales = lane < 32 ? qa.k_scales : qa.v_scales;
      const int t0 = first_token(i);
      if (whole) {
        const bool full = t0 + kQuantTokens - 1 <= t_last;
        long long row[2];  // of a half's first token
#pragma unroll
        for (int h = 0; h < 2; ++h) row[h] = ((long long)page[h] * a.num_kv_heads + hk) * P + (min(t0 + 16 * h, t_last) & (P - 1));
        int place = j;
        if (full && read_once) {
#pragma unroll
          for (int h = 0; h < 2; ++h) request_half(pool, row[h] * kD, ld_off[h], dst + h * Sh::kHalfBytes, std::true_type{});
        } else if (full) {
#pragma unroll
          for (int h = 0; h < 2; ++h) request_half(pool, row[h] * kD, ld_off[h], dst + h * Sh::kHalfBytes, std::false_type{});
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int most = max(0, t_last - (t0 + 16 * h));  // last row of the half that is visible
            uint32_t off[kLoads];
#pragma unroll
            for (int u = 0; u < kLoads; ++u) off[u] = ld_off[h][u] - (uint32_t)(max(0, ld_row(u) - most) * kD);
            request_half(pool, row[h] * kD, off, dst + h * Sh::kHalfBytes, std::false_type{});
          }
          place = min(j, max(0, t_last - (t0 + 16 * (kg & 1))));
        }
        if constexpr (v) load_bytes_to_lds((unsigned long long)of_scales + (kg & 1 ? row[1] : row[0]) + place, scales);
      } else {  // every lane looks its tokens up, in vector loads (one after the other: few tokens come this way)
        auto row_of = [&](int t) __attribute__((always_inline)) {
          const int at = min(t, t_last), entry = a.kv_indices[kv_begin + (slots ? at : at >> p_shift)];
          const int page = slots ? entry >> p_shift : entry, place = (slots ? entry : at) & (P - 1);
          return ((long long)page * a.num_kv_heads + hk) * P + place;
        };
#pragma unroll 1
        for (int x = 0; x < 2 * kLoads; ++x) {
          const int h = x / kLoads, u = x % kLoads;
          load_to_lds(pool + row_of(t0 + 16 * h + ld_row(u)) * kD + 16 * ld_piece(u, h), dst + 1024 * x);
        }
        if constexpr (v) load_bytes_to_lds((unsigned long long)of_scales + row_of(t0 + lane % 32), scales);
      }
    };
    constexpr std::integral_constant<int, 0> kKeys{};
    constexpr std::integral_constant<int, 1> kValues{};

    // ---- set-up: first tiles on their way, then the query tile ----
    // (no barrier: a wave's ring is its own, and it has read the previous link's tiles)
    int next_page[2] = {0, 0}, page[kBuffers][2] = {};
    if (whole && n_tiles > 0) {
#pragma unroll
      for (int i = 0; i < kBuffers; ++i) read_pages(i, page[i]);
      read_pages(kBuffers, next_page);
    }
    const QuerySource source = query_source<kD>(a, n_q, lflags, qref);
#pragma unroll
    for (int i = 0; i < kBuffers; ++i)
      if (i < n_tiles) {
        request(i, page[i], kKeys);
        request(i, page[i], kValues);
      }
    const QueryPieces mine = turned_query<kD>(a, source, hk, dtype, pieces);
    if (li > 0) ring_barrier<kAnyInFlight>();  // every wave has read what lay there
    va_u32x4 q_hi[kSteps], q_lo[Sh::kKeepLow ? kSteps : 1];
    if constexpr (Sh::kKeepLow) {
      stage_query<kD>(mine, 0, query);
      stage_query<kD>(mine, 1, query + 32 * kD);
      ring_barrier<kAnyInFlight>();
#pragma unroll
      for (int s = 0; s < kSteps; ++s) q_hi[s] = staged_query<kD>(query, s), q_lo[s] = staged_query<kD>(query + 32 * kD, s);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) asm volatile("" : "+v"(q_hi[s]), "+v"(q_lo[s]));
    } else {  // one after the other through the same room
      stage_query<kD>(mine, 0, query);
      ring_barrier<kAnyInFlight>();
#pragma unroll
      for (int s = 0; s < kSteps; ++s) q_hi[s] = staged_query<kD>(query, s);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) asm volatile("" : "+v"(q_hi[s]));
      ring_barrier<kAnyInFlight>();
      stage_query<kD>(mine, 1, query);
      ring_barrier<kAnyInFlight>();
    }

    // ---- the tile loop ----
    for (int i = 0; i < n_tiles; ++i) {
      // The tile has landed once at most the loads of the kBuffers - 1 tiles requested after it are outstanding.
      if (i + kBuffers - 1 < n_tiles) {
        wave_wait_loads<(kBuffers - 1) * Sh::kLoadsPerTile>();
      } else {
        wave_wait_loads<0>();
      }
      const uint32_t buffer = (uint32_t)(i % kBuffers) * Sh::kTileBytes;
      const char* tile = lds + wave * Sh::kWaveBytes + buffer;
      const bool more = i + kBuffers < n_tiles;
      va_u32x4 kraw[2][kPieces];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int s = 0; s < kPieces; ++s) kraw[h][s] = *(const va_u32x4*)(tile + h * Sh::kHalfBytes + j * kD + (k_at[h] ^ (64 * s)));
      __builtin_amdgcn_sched_barrier(0);
      if (more) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        request(i + kBuffers, next_page, kKeys);
      }
      __builtin_amdgcn_sched_barrier(0);

      const char* scales = lds + wave * Sh::kWaveBytes + Sh::kScaleOffset + (i % Sh::kScaleSlots) * Sh::kScaleBytes;
      float of_token[2] = {1.f, 1.f};  // of this lane's token of each half, where the conversion takes it
      if constexpr (C::kScales)
#pragma unroll
        for (int h = 0; h < 2; ++h) of_token[h] = scale_value(*(const uint32_t*)(scales + 64 * h + 4 * j));
      va_f32x4 dots[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) dots[h] = va_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        va_u32x4 low;
        if constexpr (Sh::kKeepLow) low = q_lo[s]; else low = staged_query<kD>(query, s);
        va_u32x4 k8[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const va_u32x4 raw = kraw[h][s / 2];
          const va_u32x2 codes = s % 2 ? va_u32x2{raw[2], raw[3]} : va_u32x2{raw[0], raw[1]};
          if constexpr (C::kScales) k8[h] = C::bf16x8(codes, of_token[h]); else k8[h] = C::bf16x8(codes);
          dots[h] = Mma<BF16>::run(k8[h], q_hi[s], dots[h]);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) dots[h] = Mma<BF16>::run(k8[h], low, dots[h]);
      }
      __builtin_amdgcn_sched_barrier(0);
      va_u32x2 vraw[kDimTiles];
#pragma unroll
      for (int t = 0; t < kDimTiles; ++t) vraw[t] = lds_read_tr8(ring + buffer + v_at + ((16 * t) ^ v_swz));
      __builtin_amdgcn_sched_barrier(0);
      if (more) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        request(i + kBuffers, next_page, kValues);
        if (whole) read_pages(i + 1 + kBuffers, next_page);
      }
      __builtin_amdgcn_sched_barrier(0);

      // online softmax; this lane holds tokens 16 h + 4 kg + r of row j
      const int t0 = first_token(i);
      va_u32x4 vscale[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) vscale[h] = *(const va_u32x4*)(scales + 128 + 64 * h + 16 * kg);
      float sc[2][4], most = -INFINITY;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if constexpr (C::kScales) {
#pragma unroll
          for (int r = 0; r < 4; ++r) sc[h][r] = dots[h][r];
        } else {
          const va_u32x4 kscale = *(const va_u32x4*)(scales + 64 * h + 16 * kg);
#pragma unroll
          for (int r = 0; r < 4; ++r) sc[h][r] = dots[h][r] * scale_value(kscale[r]);
        }
      }
      if (t0 + kQuantTokens > t_all) {  // some row does not see some token, which may have any scale
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const bool seen = t0 + 16 * h + 4 * kg + r < t_row;
            sc[h][r] = seen ? sc[h][r] : -INFINITY;
            vscale[h][r] = seen ? vscale[h][r] : 0u;
          }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 4; ++r) most = fmaxf(most, sc[h][r]);
      if (__any(most > m_run + kQuantLeap)) {
        const float m_new = fmaxf(m_run, quant_group_max(most));
        const float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
        m_run = m_new;
        l_run *= alpha;
#pragma unroll
        for (int t = 0; t < kDimTiles; ++t) o[t] *= alpha;
      }
      va_u32x4 w_hi, w_lo;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float w[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float p = __builtin_amdgcn_exp2f(sc[h][r] - m_run);
          l_run += p;
          w[r] = p * scale_value(vscale[h][r]);
        }
        uint32_t x, y;
        split_pair(w[0], w[1], x, y);
        w_hi[2 * h] = x, w_lo[2 * h] = y;
        split_pair(w[2], w[3], x, y);
        w_hi[2 * h + 1] = x, w_lo[2 * h + 1] = y;
      }

      // O^T += V^T . W^T, the lane's contraction elements being tokens 4 kg .. + 3 and 16 + 4 kg .. + 3
#pragma unroll
      for (int t = 0; t < kDimTiles; ++t) {
        const va_u32x4 v8 = C::bf16x8(vraw[t]);
        o[t] = Mma<BF16>::run(v8, w_hi, o[t]);
        o[t] = Mma<BF16>::run(v8, w_lo, o[t]);
      }
    }
  }

  __syncthreads();  // every wave is done with its tiles and the query
  fold_and_finish<kD>(a, o, m_run, l_run, lds, n_q, part_base, item[VA_I_LINK0 + VA_L_QREF], item[VA_I_LINK0 + VA_L_FLAGS], hk, dtype, pieces);
}

template <int kD, typename C>
__global__ __launch_bounds__(kQuantThreads, QuantRing<kD>::kMinBlocks) void attn_quant_stream_kernel(QuantAttnArgs qa, int dtype, int pieces) {
  quant_stream_item<kD, C>(qa, dtype, pieces);
}
template <int kD, typename C>
__global__ __launch_bounds__(kQuantThreads, QuantRing<kD>::kMinBlocks) void attn_quant_stream_if_kernel(QuantAttnArgs qa, const int32_t* only_if, int dtype,
    int pieces) {
  if (*only_if) quant_stream_item<kD, C>(qa, dtype, pieces);
}

template <int kD, typename C>
static int launch_quant_stream_one(const QuantAttnArgs& qa, const int32_t* only_if, int dtype, int n_items, int pieces, hipStream_t stream) {
  const dim3 grid((unsigned)n_items * (unsigned)qa.a.num_kv_heads), block(kQuantThreads);
  constexpr int bytes = QuantRing<kD>::kLdsBytes;
  static std::atomic<unsigned long long> devices{0}, if_devices{0};
  hipError_t e = only_if ? allow_lds(reinterpret_cast<const void*>(&attn_quant_stream_if_kernel<kD, C>), bytes, if_devices)
                         : allow_lds(reinterpret_cast<const void*>(&attn_quant_stream_kernel<kD, C>), bytes, devices);
  if (e != hipSuccess) return va_fail(VA_ERR_HIP, "raising the LDS limit: %s", hipGetErrorString(e));
  if (only_if) {
    hipLaunchKernelGGL((attn_quant_stream_if_kernel<kD, C>), grid, block, bytes, stream, qa, only_if, dtype, pieces);
  } else {
    hipLaunchKernelGGL((attn_quant_stream_kernel<kD, C>), grid, block, bytes, stream, qa, dtype, pieces);
  }
  e = hipGetLastError();
  return e == hipSuccess ? VA_OK : va_fail(VA_ERR_HIP, "quantised attention launch: %s", hipGetErrorString(e));
}

template <typename C>
static int launch_quant_stream_coded(const QuantAttnArgs& qa, const int32_t* only_if, int dtype, int n_items, int pieces, hipStream_t stream) {
  switch (qa.a.head_dim) {
    case 64:
      return launch_quant_stream_one<64, C>(qa, only_if, dtype, n_items, pieces, stream);
    case 128:
      return launch_quant_stream_one<128, C>(qa, only_if, dtype, n_items, pieces, stream);
    default:
      return launch_quant_stream_one<256, C>(qa, only_if, dtype, n_items, pieces, stream);
  }
}

int launch_quant_mfma(const QuantAttnArgs& qa, const int32_t* only_if, int dtype, int code_type, int n_items, int q_tile, hipStream_t stream) {
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
  // The choice hangs on the page size alone, so that a recorded launch keeps its kernel.
  if (qa.pages.shift < 4) return launch_quant_scattered(qa, only_if, dtype, code_type, n_items, pieces, stream);
  return code_type == VA_CODE_E4M3 ? launch_quant_stream_coded<E4M3>(qa, only_if, dtype, n_items, pieces, stream)
                                   : launch_quant_stream_coded<INT8>(qa, only_if, dtype, n_items, pieces, stream);
}

}  // namespace va
