// Matrix-core view attention over a quantised pool whose tiles do not lie in one or two pages (pages of fewer than 16 tokens
// or of a number that no power of two is).  The mathematics and the split into waves are those of va_quant_stream.hip; what
// differs is how a tile arrives: every lane looks the tokens of its rows up, two tiles ahead, and takes its pieces of K and
// V to registers a tile ahead -- V while the tile before is taken apart, K behind its last product.
//   K: lane (j, kg) of a 16-token half takes bytes [64 s + 16 kg, + 16) of token j: the contraction elements of steps
//      2 s and 2 s + 1 of the products as they are.
//   V: the same pieces go through LDS (eight tokens of a dim in one ds_read_b64_tr_b8).
// Half lines a load cost it bandwidth (pages of 16 tokens: 5.7 TB/s, 6.8 in whole lines), which scattered rows do anyway: 8
// requests of 40 k tokens (0.6 GB) 105 us in pages of 16, here 128 to 134 in pages of 8 or 48 and 151 / 169 / 205 at 256 / 128 / 64
// dims in pages of one, whose scale bytes come in a line each.  Two, three and four workgroups a CU at these dims: 64 requests
// over 8192 tokens and blocks of 256..8192, pages of 8, two / now, 233 / 215 at 128 dims, 244 / 220 at 64.
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
struct ScatteredShape {
  static constexpr int kPieces = kD / 64;    // 16-byte pieces of a token's row that a lane takes
  static constexpr int kSteps = kD / 32;     // contraction steps of K.Q^T
  static constexpr int kDimTiles = kD / 16;  // 16-dim tiles of the output
  static constexpr int kTileBytes = kQuantTokens * kD;         // V of a tile
  static constexpr int kWaveBytes = kTileBytes + 2 * kQuantTokens * 4;  // and its scales, K then V
  static constexpr int kQueryBytes = 2 * 16 * kD * 2;          // hi and lo rows
  static constexpr int kMinBlocks = kD == 64 ? 4 : kD == 128 ? 3 : 2;  // workgroups per CU
  static constexpr int kLoopBytes = kQuantWaves * kWaveBytes + kQueryBytes;
  static constexpr int kFold = kQuantWaves * QuantFold<kD>::kBytes;
  static constexpr int kLdsBytes = kLoopBytes > kFold ? kLoopBytes : kFold;
};

// Piece c of token t of a V tile lies at position c ^ quant_swz(t): the sixteen tokens that a write covers spread over the
// banks, and so do the eight that a transposing read takes of one piece.
template <int kD>
__device__ __forceinline__ int quant_swz(int t) {
  if constexpr (kD == 256) return (t & 3) | (((t >> 4) & 1) << 2) | (((t >> 2) & 1) << 3);
  if constexpr (kD == 128) return ((t >> 1) & 3) | (((t >> 4) & 1) << 2);
  return ((t >> 2) & 3) ^ ((t >> 4) & 1);
}

template <int kD, typename C>
__device__ __forceinline__ void quant_scattered_item(const QuantAttnArgs& qa, int dtype, int pieces) {
  const AttnArgs& a = qa.a;
  using Sh = ScatteredShape<kD>;
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
  const int v_piece[2] = {16 * (kg ^ quant_swz<kD>(j)), 16 * (kg ^ quant_swz<kD>(16 + j))};  // (pieces 4 s + kg: s flips higher bits)
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
    // rows that no other tile reads are requested as lines to evict first
    const bool read_once = lflags & VA_LINK_ONCE;
    auto load_pieces = [&](const uint8_t* pool, va_u32x4 (&raw)[2][kPieces]) __attribute__((always_inline)) {
      if (read_once) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int s = 0; s < kPieces; ++s) raw[u][s] = __builtin_nontemporal_load((const va_u32x4*)(pool + row[u] * kD + 64 * s + 16 * kg));
      } else {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int s = 0; s < kPieces; ++s) raw[u][s] = *(const va_u32x4*)(pool + row[u] * kD + 64 * s + 16 * kg);
      }
    };
    auto load_v = [&]() __attribute__((always_inline)) {
      load_pieces(vp, vraw);
      // lanes 0 .. 31 the scales of the 32 keys, the others those of the values
      scale_byte = (lane < 32 ? qa.k_scales : qa.v_scales)[row[kg & 1]];
    };
    auto load_k = [&]() __attribute__((always_inline)) { load_pieces(kp, kraw); };
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
    {
      const QueryPieces own = turned_query<kD>(a, query_source<kD>(a, n_q, lflags, qref), hk, dtype, pieces);
      stage_query<kD>(own, 0, query);
      stage_query<kD>(own, 1, query + 32 * kD);
    }
    __syncthreads();
    // B operands: step 2 s + b holds dims [64 s + 16 kg + 8 b, + 8) of row j
    // (but at 64 dims they are read anew for every tile, and low parts are everywhere: held in registers they cost workgroups a
    // CU, which cover the latency of each other's loads)
    constexpr bool kKeepQuery = kD < 128;
    va_u32x4 q_hi[kKeepQuery ? kSteps : 1];
    if constexpr (kKeepQuery) {
#pragma unroll
      for (int s = 0; s < kSteps; ++s) q_hi[s] = staged_query<kD>(query, s);
    }

    // ---- the tile loop ----
    for (int i = 0; i < n_tiles; ++i) {
      // V and the scales to LDS, and the next ones on their way
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int s = 0; s < kPieces; ++s) *(va_u32x4*)(mine + (16 * u + j) * kD + (v_piece[u] ^ (64 * s))) = vraw[u][s];
      scales[lane] = scale_value(scale_byte);
      asm volatile("" ::: "memory");
      if (i + 1 < n_tiles) {
        load_v();
        read_entries(i + 2);
      }

      va_f32x4 dots[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) dots[u] = va_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const va_u32x4 high = kKeepQuery ? q_hi[kKeepQuery ? s : 0] : staged_query<kD>(query, s);
        const va_u32x4 low = staged_query<kD>(query + 32 * kD, s);
        va_u32x4 k8[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const va_u32x4 raw = kraw[u][s / 2];
          k8[u] = C::bf16x8(s % 2 ? va_u32x2{raw[2], raw[3]} : va_u32x2{raw[0], raw[1]});
          dots[u] = Mma<BF16>::run(k8[u], high, dots[u]);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) dots[u] = Mma<BF16>::run(k8[u], low, dots[u]);
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
          sc[u][r] = seen ? dots[u][r] * ks[r] : -INFINITY;
          vs[u][r] = seen ? v4[r] : 0.f;
          most = fmaxf(most, sc[u][r]);
        }
      }
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

  __syncthreads();  // every wave is done with its tiles and the query
  fold_and_finish<kD>(a, o, m_run, l_run, lds, n_q, part_base, item[VA_I_LINK0 + VA_L_QREF], item[VA_I_LINK0 + VA_L_FLAGS], hk, dtype, pieces);
}

template <int kD, typename C>
__global__ __launch_bounds__(kQuantThreads, ScatteredShape<kD>::kMinBlocks) void attn_quant_scattered_kernel(QuantAttnArgs qa, int dtype, int pieces) {
  quant_scattered_item<kD, C>(qa, dtype, pieces);
}
template <int kD, typename C>
__global__ __launch_bounds__(kQuantThreads, ScatteredShape<kD>::kMinBlocks) void attn_quant_scattered_if_kernel(QuantAttnArgs qa, const int32_t* only_if, int dtype,
    int pieces) {
  if (*only_if) quant_scattered_item<kD, C>(qa, dtype, pieces);
}

template <int kD, typename C>
static int launch_quant_scattered_one(const QuantAttnArgs& qa, const int32_t* only_if, int dtype, int n_items, int pieces, hipStream_t stream) {
  const dim3 grid((unsigned)n_items * (unsigned)qa.a.num_kv_heads), block(kQuantThreads);
  constexpr int bytes = ScatteredShape<kD>::kLdsBytes;
  static std::atomic<unsigned long long> devices{0}, if_devices{0};
  hipError_t e = only_if ? allow_lds(reinterpret_cast<const void*>(&attn_quant_scattered_if_kernel<kD, C>), bytes, if_devices)
                         : allow_lds(reinterpret_cast<const void*>(&attn_quant_scattered_kernel<kD, C>), bytes, devices);
  if (e != hipSuccess) return va_fail(VA_ERR_HIP, "raising the LDS limit: %s", hipGetErrorString(e));
  if (only_if) {
    hipLaunchKernelGGL((attn_quant_scattered_if_kernel<kD, C>), grid, block, bytes, stream, qa, only_if, dtype, pieces);
  } else {
    hipLaunchKernelGGL((attn_quant_scattered_kernel<kD, C>), grid, block, bytes, stream, qa, dtype, pieces);
  }
  e = hipGetLastError();
  return e == hipSuccess ? VA_OK : va_fail(VA_ERR_HIP, "quantised attention launch: %s", hipGetErrorString(e));
}

template <typename C>
static int launch_quant_scattered_coded(const QuantAttnArgs& qa, const int32_t* only_if, int dtype, int n_items, int pieces, hipStream_t stream) {
  switch (qa.a.head_dim) {
    case 64:
      return launch_quant_scattered_one<64, C>(qa, only_if, dtype, n_items, pieces, stream);
    case 128:
      return launch_quant_scattered_one<128, C>(qa, only_if, dtype, n_items, pieces, stream);
    default:
      return launch_quant_scattered_one<256, C>(qa, only_if, dtype, n_items, pieces, stream);
  }
}

int launch_quant_scattered(const QuantAttnArgs& qa, const int32_t* only_if, int dtype, int code_type, int n_items, int pieces, hipStream_t stream) {
  return code_type == VA_CODE_E4M3 ? launch_quant_scattered_coded<E4M3>(qa, only_if, dtype, n_items, pieces, stream)
                                   : launch_quant_scattered_coded<INT8>(qa, only_if, dtype, n_items, pieces, stream);
}

}  // namespace va
