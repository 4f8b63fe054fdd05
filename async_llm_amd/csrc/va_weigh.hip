// Attention weights by cached token: for every token and kv head the sum, over all rows and q heads that see the token, of
// exp(score - lse), added to the sums of former steps.
//
//   S^T[16 tokens, 16 rows] = K . Q^T    v_mfma_f32_16x16x32, keys as the A operand (a lane's element of the result: four tokens of
//                                        one row)
//   sum[token] += exp2(S - lse2[row])    no running maximum: the log-sum is known, so rows may come in any order and split
//
// The keys of a workgroup's tokens are loaded once and stay in registers while the rows' queries pass by; a lane's sums stay in
// registers too, and its rows are added up across lanes at the end.  Sums are 32-bit numbers that users compare and add up over many
// steps, so queries are not rounded to 16 bits: they come as sums of 16-bit numbers (bf16: three, which hold all 24 bits; float16:
// two of a row brought into its range by a power of two, 22 bits) and each product is taken that often.  A first pass over the
// packed rows (weigh_rows_kernel) turns them, scales them by log2(e) / sqrt(D) and writes those parts as the matrix cores read
// them.  Codes of a quantised pool become bf16, scale and all, exactly.
//
// Where a chunk's rows are split among workgroups each writes partial sums, and weigh_join_kernel adds them in their order.
#include <hip/hip_runtime.h>

#include "va_device.h"
#include "va_internal.h"
#include "va_launch.h"
#include "va_mfma_common.h"
#include "va_quant.h"
#include "va_weigh.h"

namespace va {

constexpr int kWeighThreads = 256, kWeighWaves = kWeighThreads / kWave;
constexpr int kWeighGroups = VA_WEIGH_CHUNK / (16 * kWeighWaves);  // groups of 16 tokens of a wave
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
  const int32_t* joins;
  const int32_t* pages;
  const int32_t* sub_rows;
  const int32_t* lo;
  const int32_t* hi;
  int n_rows, n_tiles;
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
enum { kRows32 = 0, kRowsF16 = 2, kRowsBF16 = 3 };  // 32-bit rows, or how many 16-bit parts

// 16-bit parts: element d of row j belongs to step 2 (d / 64) + (d / 8) % 2, contraction group (d / 16) % 4, so that a lane's
// pieces of two steps are neighbours in the row: [tile][part][step][lane] of 16 bytes, lane 16 * group + j.
template <int kParts>
__global__ __launch_bounds__(kWeighThreads) void weigh_rows_kernel(WeighArgs a) {
  __shared__ float x[16][kWeighMaxDim + 1];
  const int tile = blockIdx.x, hk = blockIdx.y, D = a.head_dim, G = a.num_q_heads / a.num_kv_heads;
  const int j = threadIdx.x / 16, c = threadIdx.x % 16;
  const int pair = tile * 16 + j, row = pair / G, hq = hk * G + pair - row * G;
  const int sub = a.sub_rows[row];
  const long long worker = sub < 0 ? 0 : a.sub_worker[sub];
  if (sub >= 0) {
    const Pos3 pos = load_pos(a.sub_loc, a.sub_loc_axis_stride, sub);
    const long long at = worker * a.q_row_stride + (long long)hq * D;
    for (int i = c; i < a.rope.half; i += 16) {
      float cs, sn;
      rope_cos_sin(a.rope, pos, i, cs, sn);
      const float x1 = weigh_activation(a.q, at + i, a.dtype), x2 = weigh_activation(a.q, at + i + a.rope.half, a.dtype);
      x[j][i] = (mul_rounded(cs, x1) - mul_rounded(sn, x2)) * a.scale_log2;
      x[j][i + a.rope.half] = (mul_rounded(cs, x2) + mul_rounded(sn, x1)) * a.scale_log2;
    }
    for (int d = 2 * a.rope.half + c; d < D; d += 16) x[j][d] = weigh_activation(a.q, at + d, a.dtype) * a.scale_log2;
  } else {
    for (int d = c; d < D; d += 16) x[j][d] = 0.f;
  }
  __syncthreads();
  float scale = 1.f, up = 1.f;
  if constexpr (kParts == kRowsF16) {  // the largest element to 2^10 .. 2^11
    float most = 0.f;
    for (int d = c; d < D; d += 16) most = fmaxf(most, fabsf(x[j][d]));
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) most = fmaxf(most, __shfl_xor(most, off, kWave));
    const int e = most > 0.f && most < INFINITY ? min(max(10 - ((int)(__float_as_uint(most) >> 23) - 127), -100), 100) : 0;
    up = __uint_as_float((uint32_t)(127 + e) << 23), scale = __uint_as_float((uint32_t)(127 - e) << 23);
  }
  if constexpr (kParts == kRows32) {
    float* to = (float*)a.queries + ((long long)hk * a.n_tiles * 16 + pair) * D;
    for (int d = c; d < D; d += 16) to[d] = x[j][d];
  } else {
    for (int piece = c; piece < D / 8; piece += 16) {
      const int step = 2 * (piece / 8) + piece % 2, group = piece % 8 / 2;
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = x[j][8 * piece + e] * up;
#pragma unroll
      for (int part = 0; part < kParts; ++part) {
        va_u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (kParts == kRowsF16) {
            w[e] = Mma<F16>::pack(y[2 * e], y[2 * e + 1]);
            y[2 * e] -= F16::load(__builtin_bit_cast(__half, (uint16_t)w[e])), y[2 * e + 1] -= F16::load(__builtin_bit_cast(__half, (uint16_t)(w[e] >> 16)));
          } else {
            w[e] = Mma<BF16>::pack(y[2 * e], y[2 * e + 1]);
            y[2 * e] -= __uint_as_float(w[e] << 16), y[2 * e + 1] -= __uint_as_float(w[e] & 0xffff0000u);
          }
        }
        *(va_u32x4*)(a.queries + ((((long long)hk * a.n_tiles + tile) * kParts + part) * (D / 32) + step) * 1024 + (16 * group + j) * 16) = w;
      }
    }
  }
  if (c == 0) {
    WeighRow r{0.f, scale, 0, 0};
    if (sub >= 0) {
      const float lse = a.lse[worker * a.num_q_heads + hq];
      r.minus_lse = a.lse_base2 ? -lse : -lse * kLog2e;
      if (lse != -INFINITY) r.lo = a.lo[row], r.hi = a.hi[row];
    }
    a.rows[(long long)hk * a.n_tiles * 16 + pair] = r;
  }
}

// ---------------------------------------------------------------------------
// matrix cores
// ---------------------------------------------------------------------------
// Pool element types: what their keys are in the products.
template <typename E>
struct WeighKeys {
  using M = E;
  static constexpr bool kCodes = false;
  static constexpr int kParts = kRowsBF16;
};
template <>
struct WeighKeys<F16> {
  using M = F16;
  static constexpr bool kCodes = false;
  static constexpr int kParts = kRowsF16;
};
template <>
struct WeighKeys<E4M3> {
  using M = BF16;
  static constexpr bool kCodes = true;
  static constexpr int kParts = kRowsBF16;
  static __device__ __forceinline__ va_u32x4 keys(va_u32x2 codes, float scale) { return E4M3::bf16x8(codes, scale); }
};
template <>
struct WeighKeys<INT8> {
  using M = BF16;
  static constexpr bool kCodes = true;
  static constexpr int kParts = kRowsBF16;
  static __device__ __forceinline__ va_u32x4 keys(va_u32x2 codes, float scale) {  // (bf16 has the eight bits of a code)
    float x[8];
    INT8::unpack4(codes[0], x), INT8::unpack4(codes[1], x + 4);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] *= scale;
    return va_u32x4{Mma<BF16>::pack(x[0], x[1]), Mma<BF16>::pack(x[2], x[3]), Mma<BF16>::pack(x[4], x[5]), Mma<BF16>::pack(x[6], x[7])};
  }
};

template <int kD, typename C>
__global__ __launch_bounds__(kWeighThreads) void weigh_mfma_kernel(WeighArgs a) {
  using K = WeighKeys<C>;
  using M = Mma<typename K::M>;
  constexpr int kParts = K::kParts, kSteps = kD / 32;
  const ItemHead where = item_and_head(blockIdx.x, a.num_kv_heads);
  const int32_t* item = a.items + (long long)where.item * VA_WEIGH_ITEM_WORDS;
  const int n_tok = item[VA_WI_N_TOK], hk = where.head;
  if (n_tok == 0) return;
  const int page_begin = item[VA_WI_PAGES], first = item[VA_WI_FIRST], tile_end = item[VA_WI_TILE_END], partial = item[VA_WI_PARTIAL];
  const int lane = threadIdx.x % kWave, j = lane % 16, kg = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int w0 = 16 * kWeighGroups * wave;  // first token of the wave, in the chunk
  if (w0 >= n_tok) return;

  va_u32x4 keys[kWeighGroups][kSteps];
#pragma unroll
  for (int g = 0; g < kWeighGroups; ++g) {
    const uint32_t slot = weigh_slot(a, page_begin, first + min(w0 + 16 * g + j, n_tok - 1));
    if constexpr (K::kCodes) {
      const long long row = quant_row(a.page_map, slot, hk, a.num_kv_heads);
      const float scale = scale_value(a.k_scales[row]);
      va_u32x4 raw[kSteps / 2];
#pragma unroll
      for (int s = 0; s < kSteps / 2; ++s) raw[s] = *(const va_u32x4*)((const uint8_t*)a.k_pool + row * kD + 64 * s + 16 * kg);
#pragma unroll
      for (int s = 0; s < kSteps / 2; ++s) {
        keys[g][2 * s] = K::keys(va_u32x2{raw[s][0], raw[s][1]}, scale);
        keys[g][2 * s + 1] = K::keys(va_u32x2{raw[s][2], raw[s][3]}, scale);
      }
    } else {
      const uint16_t* row = (const uint16_t*)a.k_pool + (long long)slot * a.pool_row_stride + (long long)hk * kD;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) keys[g][s] = *(const va_u32x4*)(row + 64 * (s / 2) + 16 * kg + 8 * (s % 2));
    }
  }

  const int t_wave = first + w0, t_end = min(t_wave + 16 * kWeighGroups, first + n_tok);
  float sum[kWeighGroups][4];
#pragma unroll
  for (int g = 0; g < kWeighGroups; ++g)
#pragma unroll
    for (int r = 0; r < 4; ++r) sum[g][r] = 0.f;
  for (int tile = item[VA_WI_TILE_BEGIN]; tile < tile_end; ++tile) {
    const long long at = (long long)hk * a.n_tiles + tile;
    const WeighRow row = a.rows[at * 16 + j];
    if (!__any(row.lo < t_end && row.hi > t_wave)) continue;
    const va_u32x4* queries = (const va_u32x4*)(a.queries + at * (kParts * kSteps * 1024)) + lane;
    va_f32x4 dots[kWeighGroups];
#pragma unroll
    for (int g = 0; g < kWeighGroups; ++g) dots[g] = va_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int part = kParts - 1; part >= 0; --part)  // (small ones first)
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const va_u32x4 q = queries[(part * kSteps + s) * kWave];
#pragma unroll
        for (int g = 0; g < kWeighGroups; ++g) dots[g] = M::run(keys[g][s], q, dots[g]);
      }
    const bool all = !__any(row.lo > t_wave || row.hi < t_end);
#pragma unroll
    for (int g = 0; g < kWeighGroups; ++g)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float p = __builtin_amdgcn_exp2f(fmaf(dots[g][r], row.scale, row.minus_lse));
        const int t = t_wave + 16 * g + 4 * kg + r;
        sum[g][r] += all || (t >= row.lo && t < row.hi) ? p : 0.f;
      }
  }
#pragma unroll
  for (int g = 0; g < kWeighGroups; ++g) {
#pragma unroll
    for (int r = 0; r < 4; ++r) sum[g][r] = group_sum<16>(sum[g][r]);
    // lane j < 4 has token 4 kg + j
    const float mine = j == 0 ? sum[g][0] : j == 1 ? sum[g][1] : j == 2 ? sum[g][2] : sum[g][3];
    const int t = w0 + 16 * g + 4 * kg + j;
    if (j < 4 && t < n_tok) {
      if (partial >= 0) {
        a.partials[hk * a.n_partials + partial + t] = mine;
      } else {
        const long long to = hk * a.num_slots + weigh_slot(a, page_begin, first + t);
        a.weights_out[to] = a.weights_in[to] + mine;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// vector ALU: any type, alignment and head_dim up to kWeighMaxDim
// ---------------------------------------------------------------------------
constexpr int kWeighBatch = 4;  // rows of a wave at a time

template <typename C>
__global__ __launch_bounds__(kWeighThreads) void weigh_generic_kernel(WeighArgs a) {
  extern __shared__ float lds[];  // [64 tokens][D + 1], then [waves][64]
  const ItemHead where = item_and_head(blockIdx.x, a.num_kv_heads);
  const int32_t* item = a.items + (long long)where.item * VA_WEIGH_ITEM_WORDS;
  const int n_tok = item[VA_WI_N_TOK], hk = where.head, D = a.head_dim;
  if (n_tok == 0) return;
  const int page_begin = item[VA_WI_PAGES], first = item[VA_WI_FIRST], partial = item[VA_WI_PARTIAL];
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
    for (int pair = item[VA_WI_TILE_BEGIN] * 16 + wave * kWeighBatch; pair < item[VA_WI_TILE_END] * 16; pair += kWeighWaves * kWeighBatch) {
      const float* q = (const float*)a.queries + ((long long)hk * a.n_tiles * 16 + pair) * D;
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

__global__ __launch_bounds__(VA_WEIGH_CHUNK) void weigh_join_kernel(WeighArgs a) {
  const int32_t* join = a.joins + (long long)blockIdx.x * VA_WEIGH_JOIN_WORDS;
  const int n_tok = join[VA_WJ_N_TOK], n_parts = join[VA_WJ_N_PARTS], hk = blockIdx.y, t = threadIdx.x;
  if (t >= n_tok) return;
  const float* from = a.partials + hk * a.n_partials + join[VA_WJ_PARTIAL] + t;
  float sum = 0.f;
  for (int p = 0; p < n_parts; ++p) sum += from[(long long)p * n_tok];
  const long long to = hk * a.num_slots + weigh_slot(a, join[VA_WJ_PAGES], join[VA_WJ_FIRST] + t);
  a.weights_out[to] = a.weights_in[to] + sum;
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
static int weigh_launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? VA_OK : va_fail(VA_ERR_HIP, "%s launch: %s", what, hipGetErrorString(e));
}

template <typename C>
static int launch_weigh(const WeighArgs& a, int n_items, bool matrix, hipStream_t stream) {
  const dim3 rows_grid((unsigned)a.n_tiles, (unsigned)a.num_kv_heads), grid((unsigned)n_items * (unsigned)a.num_kv_heads), block(kWeighThreads);
  if constexpr (!std::is_same_v<C, F32>) {
    if (matrix) {
      hipLaunchKernelGGL(weigh_rows_kernel<WeighKeys<C>::kParts>, rows_grid, block, 0, stream, a);
      switch (a.head_dim) {
        case 64:
          hipLaunchKernelGGL((weigh_mfma_kernel<64, C>), grid, block, 0, stream, a);
          break;
        case 128:
          hipLaunchKernelGGL((weigh_mfma_kernel<128, C>), grid, block, 0, stream, a);
          break;
        default:
          hipLaunchKernelGGL((weigh_mfma_kernel<256, C>), grid, block, 0, stream, a);
      }
      return weigh_launched("attention weights");
    }
  }
  const int bytes = (64 * (a.head_dim + 1) + 64 * kWeighWaves) * 4;
  static std::atomic<unsigned long long> devices{0};
  const hipError_t e = allow_lds(reinterpret_cast<const void*>(&weigh_generic_kernel<C>), (64 * (kWeighMaxDim + 1) + 64 * kWeighWaves) * 4, devices);
  if (e != hipSuccess) return va_fail(VA_ERR_HIP, "raising the LDS limit: %s", hipGetErrorString(e));
  hipLaunchKernelGGL(weigh_rows_kernel<kRows32>, rows_grid, block, 0, stream, a);
  hipLaunchKernelGGL(weigh_generic_kernel<C>, grid, block, (unsigned)bytes, stream, a);
  return weigh_launched("attention weights");
}

static int weigh(WeighArgs& a, int code_type, int num_pages, const int32_t* plan_dev, const int32_t* h, void* workspace, int64_t workspace_bytes,
                 const VaShape* shape, const VaRope* rope, hipStream_t stream) {
  if (!h || h[VA_WH_MAGIC] != VA_WEIGH_MAGIC) return va_fail(VA_ERR_ARG, "not a plan of attention weights");
  if (h[VA_WH_HQ] != shape->num_q_heads || h[VA_WH_HKV] != shape->num_kv_heads || h[VA_WH_D] != shape->head_dim ||
      h[VA_WH_PAGE] != shape->page_size || h[VA_WH_DTYPE] != shape->dtype || (num_pages >= 0 && h[VA_WH_POOL_PAGES] != num_pages))
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
  const bool rows16 = code_type >= 0 || (a.pool_row_stride % 8 == 0 && (uintptr_t)a.k_pool % 16 == 0);
  const bool matrix = dims && rows16;
  if (code_type == VA_CODE_E4M3) {
    rc = launch_weigh<E4M3>(a, n_items, matrix, stream);
  } else if (code_type == VA_CODE_INT8) {
    rc = launch_weigh<INT8>(a, n_items, matrix, stream);
  } else {
    switch (shape->dtype) {
      case VA_F32:
        rc = launch_weigh<F32>(a, n_items, false, stream);
        break;
      case VA_F16:
        rc = launch_weigh<F16>(a, n_items, matrix, stream);
        break;
      case VA_BF16:
        rc = launch_weigh<BF16>(a, n_items, matrix, stream);
        break;
      default:
        rc = va_fail(VA_ERR_ARG, "unknown dtype %d", (int)shape->dtype);
    }
  }
  if (rc || h[VA_WH_N_JOINS] == 0) return rc;
  hipLaunchKernelGGL(weigh_join_kernel, dim3((unsigned)h[VA_WH_N_JOINS], (unsigned)hkv), dim3(VA_WEIGH_CHUNK), 0, stream, a);
  return weigh_launched("joining attention weights");
}

}  // namespace va

extern "C" int va_weigh(const void* q_dev, int64_t q_row_stride, const void* k_pool_dev, int64_t pool_row_stride, const int32_t* plan_dev,
                        const int32_t* plan_header_host, const int64_t* sub_worker_dev, const int64_t* sub_loc_dev, int64_t sub_loc_axis_stride,
                        const float* lse_dev, int32_t lse_base2, const float* weights_in_dev, float* weights_out_dev, void* workspace_dev,
                        int64_t workspace_bytes, const VaShape* shape, const VaRope* rope, void* stream) {
  if (!shape || shape->num_kv_heads <= 0 || shape->num_q_heads <= 0 || shape->num_q_heads % shape->num_kv_heads || shape->head_dim <= 0 || shape->page_size <= 0)
    return va_fail(VA_ERR_ARG, "bad shape");
  if (pool_row_stride < (int64_t)shape->num_kv_heads * shape->head_dim) return va_fail(VA_ERR_ARG, "pool rows overlap");
  va::WeighArgs a{};
  a.q = q_dev, a.q_row_stride = q_row_stride, a.k_pool = k_pool_dev, a.pool_row_stride = pool_row_stride, a.sub_worker = sub_worker_dev;
  a.sub_loc = sub_loc_dev, a.sub_loc_axis_stride = sub_loc_axis_stride, a.lse = lse_dev, a.lse_base2 = lse_base2;
  a.weights_in = weights_in_dev, a.weights_out = weights_out_dev;
  return va::weigh(a, -1, -1, plan_dev, plan_header_host, workspace_dev, workspace_bytes, shape, rope, (hipStream_t)stream);
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
