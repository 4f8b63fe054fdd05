// View attention of many new tokens over a quantised pool, by rows read back once.
//
// A prefill chunk reads every token of its view for hundreds of rows: the products are what it costs, and the 16-bit
// kernel's wide tiles (va_mfma_wide.hip) run them at a rate that a kernel which converts codes beside them did not come
// near: four chunks of 300 to 1500 tokens over 8000 at 128 dims 675 us, with tiles of 16 rows over codes 1473, with
// wide tiles over codes 960 to 1140.  Reading back is a tenth of it (47 k tokens, 94 MB of codes).
//
// It runs in float16 whatever the activations are: codes have four (eight) bits, so eleven hold them, and a bf16 query or
// weight would put an error on the result that is as large as its own rounding (0.0034 against 0.0017 of it, in bf16).  A float16 one does
// the same to float16 results (0.00036 against 0.00021), which the Python op therefore leaves to the codes.  Range is
// what float16 lacks; it is given by powers of two, exactly:
//   K' = K 2^-b,  q' = q 2^b,  V' = V 2^-s,  out = out' 2^s
// with b and s from the largest scales among the rows, found by a pass over the scale bytes.  Beside float16's relative
// errors (under mRoPE its kernels round cosines, sines, products and their sum to it, each) this leaves absolute ones of 2^-25,
// half of its smallest step: 2^-39 of the largest value for V' and out'; 2^-17 / sqrt(D) of a score for each q' element below
// 2^-14 (K' is at most 2^8) and 2^-25 q' / sqrt(D) for each K' element below it; and 2^-33 of a value for each token's weight,
// whose largest is taken as 2^8 (F16Lifted in va_mfma_common.h).
//
// One b and one s serve all heads and requests of a launch, whose rows need not be of a size.  Where float16 would lose what
// codes keep, the launch says so in the scratch's first word, and its results are taken from the codes (va_attention_if_q8):
//   * a query element is over kMostQuery = 2^9 in front of its rotation, |q_i| max|K| > 1.1e5: below it the errors of all D
//     elements of K' add up to 2^-12 of a score at most, whatever their size, and nothing overflows;
//   * a value row's scale is more than kMostSpread = 16 powers of two under the largest one, and the row is not zero: above
//     that its codes are exact in V' (e4m3 the multiples of 2^(6 - 9 - 16), int8 of 2^(7 - 16)), and the row's largest is over
//     2^-4, 2^21 times the absolute error.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "va_internal.h"
#include "va_launch.h"
#include "va_quant.h"
#include "va_quant_attn.h"

namespace va {

constexpr int kBackGroups = 64;  // workgroups of the pass over the scales: a lane each to fold them

template <typename C>
struct BackScale;  // log2 of what a code of the largest scale counts: K' up to 224 or 254, V' (and with it out') up to 28672 or 16256
template <>
struct BackScale<E4M3> {
  static constexpr int kKey = -1, kValue = 6;
};
template <>
struct BackScale<INT8> {
  static constexpr int kKey = 1, kValue = 7;
};

// The least of the largest scales: rows that are all smaller lie lower in float16, and the powers that undo it, 2^(scale - 127 -
// kKey) and 2^(scale - 127 - kValue), stay normal numbers of 32 bits.
constexpr uint32_t kLeastTop = 8;
static_assert((int)kLeastTop - 127 - BackScale<INT8>::kValue >= -126 && (int)kLeastTop - 127 - BackScale<E4M3>::kValue >= -126 &&
              (int)kLeastTop - 127 - BackScale<INT8>::kKey >= -126, "powers of two that are not normal numbers");

struct BackArgs {
  const uint8_t* codes[2];
  const uint8_t* scales[2];
  const int64_t* slots;
  long long n_slots;
  uint32_t num_slots;
  int num_kv_heads, head_dim;
  PageMap pages;
  int32_t* beyond;  // whether float16 does not hold the launch's numbers
  uint32_t* tops;   // [kBackGroups][2]: largest scale bytes of keys and values
  __half* rows[2];
  const void* q;
  long long q_row_stride;
  __half* q16;
  long long n_rows;
  int q_width, dtype;
};

__device__ __forceinline__ bool back_slot(const BackArgs& a, long long i, uint32_t& slot) {
  const long long s = a.slots[i];
  slot = (uint32_t)s;
  return s >= 0 && s < (long long)a.num_slots;
}

// The largest scales of a stride of the slots (255 marks rows of NaN), or kLeastTop.
__global__ __launch_bounds__(256) void quant_top_kernel(BackArgs a) {
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.beyond = 0;
  uint32_t top[2] = {kLeastTop, kLeastTop};
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < a.n_slots; i += kBackGroups * 256ll) {
    uint32_t slot;
    if (!back_slot(a, i, slot)) continue;
    const long long row = quant_row(a.pages, slot, 0, a.num_kv_heads);
    for (int h = 0; h < a.num_kv_heads; ++h) {
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const uint32_t e = a.scales[w][row + (long long)h * a.pages.size];
        if (e != 255u) top[w] = max(top[w], e);
      }
    }
  }
  __shared__ uint32_t of_wave[4][2];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) top[w] = max(top[w], (uint32_t)__shfl_xor((int)top[w], off, kWave));
    if (threadIdx.x % kWave == 0) of_wave[threadIdx.x / kWave][w] = top[w];
  }
  __syncthreads();
  if (threadIdx.x < 2)
    a.tops[2 * blockIdx.x + threadIdx.x] = max(max(of_wave[0][threadIdx.x], of_wave[1][threadIdx.x]),
                                               max(of_wave[2][threadIdx.x], of_wave[3][threadIdx.x]));
}
__device__ __forceinline__ int back_top(const uint32_t* tops, int which) {  // (by a whole wave)
  static_assert(kBackGroups == kWave, "a lane a group");
  uint32_t top = tops[2 * (threadIdx.x % kWave) + which];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, off, kWave));
  return (int)top;
}

constexpr float kMostQuery = 512.f;
constexpr int kMostSpread = 16;
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)min(254, max(0, e + 127)) << 23); }

// K (blockIdx.y 0), V (1) and the queries (2) as float16, eight elements a thread.
template <typename C>
__global__ __launch_bounds__(256) void quant_back_kernel(BackArgs a, long long rows_threads, long long q_threads, int pieces) {
  const long long idx = blockIdx.x * 256ll + threadIdx.x;
  const int which = blockIdx.y;
  const int top = back_top(a.tops, which == 1 ? 1 : 0);
  bool beyond = which == 2 && top - 127 - BackScale<C>::kKey > 127;  // (no scale of this library's stores)
  union {
    uint4 raw;
    __half e[8];
  } y;
  if (which < 2) {
    if (idx >= rows_threads) return;
    const int per_head = a.head_dim / 8, per_row = a.num_kv_heads * per_head;
    const long long i = idx / per_row;
    const int u = (int)(idx - i * per_row), h = u / per_head, d0 = 8 * (u - h * per_head);
    y.raw = make_uint4(0, 0, 0, 0);
    uint32_t slot;
    if (back_slot(a, i, slot)) {
      const long long r = quant_row(a.pages, slot, h, a.num_kv_heads);
      const uint2 codes = *(const uint2*)((which ? a.codes[1] : a.codes[0]) + r * a.head_dim + d0);
      // A row of NaN goes to the keys, whose products are masked: a NaN among the values would reach those that do not see it.
      const uint32_t ek = a.scales[0][r], ev = a.scales[1][r], e = which ? ev : ek;
      const bool nan = ek == 255u || ev == 255u;
      const float f = nan ? 0.f : power_of_two((int)e - top + (which ? BackScale<C>::kValue : BackScale<C>::kKey));
      float x[8];
      C::unpack4(codes.x, x);
      C::unpack4(codes.y, x + 4);
#pragma unroll
      for (int k = 0; k < 8; ++k) y.e[k] = nan && !which ? __float2half_rn(NAN) : __float2half_rn(x[k] * f);
      beyond = which && !nan && (int)e < top - kMostSpread && ((codes.x | codes.y) & C::kNotZero) != 0;
    }
    *(uint4*)((which ? a.rows[1] : a.rows[0]) + idx * 8) = y.raw;
  } else {
    if (idx >= q_threads) return;
    const int per_row = a.q_width / 8;
    const long long row = idx / per_row, at = row * a.q_row_stride + (idx - row * per_row) * 8;
    const float f = power_of_two(top - 127 - BackScale<C>::kKey);
    auto query = [&](float x) __attribute__((always_inline)) {
      beyond = beyond || fabsf(x * f) > kMostQuery;  // (a NaN makes one of its own row either way)
      return __float2half_rn(x * f);
    };
    if (pieces) {
      const uint4 w = *(const uint4*)((const uint16_t*)a.q + at);
      const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint16_t b = (uint16_t)(words[k / 2] >> (16 * (k % 2)));
        y.e[k] = query(a.dtype == VA_BF16 ? BF16::load(b) : __half2float(__builtin_bit_cast(__half, b)));
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) y.e[k] = query(activation(a.q, at + k, a.dtype));
    }
    *(uint4*)(a.q16 + idx * 8) = y.raw;
  }
  if (beyond) *a.beyond = 1;  // (all that write it write the same)
}

// Results in the activations' type, eight elements a thread.  A row that a NaN reached has NaN for its lse (the attention's
// kernels leave -inf where the sum of its weights is no number).
template <typename C>
__global__ __launch_bounds__(256) void quant_results_kernel(const __half* from, void* out, float* lse, const uint32_t* tops,
                                                            long long threads, int head_dim, int dtype, int pieces) {
  const long long idx = blockIdx.x * 256ll + threadIdx.x;
  const float f = power_of_two(back_top(tops, 1) - 127 - BackScale<C>::kValue);
  if (idx >= threads) return;
  union {
    uint4 raw;
    __half e[8];
  } x;
  x.raw = *(const uint4*)(from + idx * 8);
  float y[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) y[k] = __half2float(x.e[k]) * f;
  if (lse && y[0] != y[0] && idx % (head_dim / 8) == 0) lse[idx / (head_dim / 8)] = NAN;
  if (pieces) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = dtype == VA_BF16 ? Mma<BF16>::pack(y[2 * k], y[2 * k + 1]) : Mma<F16>::pack(y[2 * k], y[2 * k + 1]);
    *(uint4*)((uint16_t*)out + idx * 8) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) store_activation(out, idx * 8 + k, y[k], dtype);
  }
}

struct BackLayout {
  int64_t tops, rows[2], q, out, bytes;
};
static BackLayout back_layout(int64_t n_slots, int64_t n_rows, const VaShape* s) {
  auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
  const int64_t kv = up(2 * n_slots * s->num_kv_heads * s->head_dim), q = up(2 * n_rows * s->num_q_heads * s->head_dim);
  BackLayout l;
  l.tops = 256;  // (behind the word that says whether float16 holds the launch)
  l.rows[0] = l.tops + up(kBackGroups * 2 * 4);
  l.rows[1] = l.rows[0] + kv;
  l.q = l.rows[1] + kv;
  l.out = l.q + q;
  l.bytes = l.out + q;
  return l;
}

template <typename C>
static int launch_quant_back(const BackArgs& a, int pieces, hipStream_t stream) {
  const long long rows_threads = a.n_slots * a.num_kv_heads * (a.head_dim / 8), q_threads = a.n_rows * (a.q_width / 8);
  const long long blocks = (std::max(rows_threads, q_threads) + 255) / 256;
  if (blocks > 0x7fffffffLL) return va_fail(VA_ERR_ARG, "too many rows");
  hipLaunchKernelGGL(quant_top_kernel, dim3(kBackGroups), dim3(256), 0, stream, a);
  hipLaunchKernelGGL((quant_back_kernel<C>), dim3((unsigned)blocks, 3), dim3(256), 0, stream, a, rows_threads, q_threads, pieces);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? VA_OK : va_fail(VA_ERR_HIP, "read-back launch: %s", hipGetErrorString(e));
}

template <typename C>
static int launch_quant_results(const __half* from, void* out, float* lse, const uint32_t* tops, long long n, int head_dim,
                                int dtype, hipStream_t stream) {
  const int pieces = (uintptr_t)out % 16 == 0;
  hipLaunchKernelGGL((quant_results_kernel<C>), dim3((unsigned)((n / 8 + 255) / 256)), dim3(256), 0, stream, from, out, lse,
                     tops, n / 8, head_dim, dtype, pieces);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? VA_OK : va_fail(VA_ERR_HIP, "results launch: %s", hipGetErrorString(e));
}

}  // namespace va

extern "C" int64_t va_read_back_bytes(int64_t n_slots, int64_t n_rows, const VaShape* shape) {
  if (!shape || n_slots < 0 || n_rows < 0) return va_fail(VA_ERR_ARG, "bad shape");
  return va::back_layout(n_slots, n_rows, shape).bytes;
}

extern "C" int va_attention_read_back_q8(const void* q_dev, int64_t q_row_stride, const VaQuantPool* pool,
                                         const int64_t* slots_dev, int64_t n_slots, const int32_t* plan_dev,
                                         const int32_t* plan_header_host, const int32_t* kv_indices_dev,
                                         const int64_t* sub_worker_dev, const int64_t* sub_loc_dev,
                                         int64_t sub_loc_axis_stride, void* out_dev, float* lse_dev, int32_t lse_base2,
                                         void* workspace_dev, int64_t workspace_bytes, void* scratch_dev,
                                         int64_t scratch_bytes, const VaShape* shape, const VaRope* rope, void* stream) {
  if (!shape || !plan_header_host || !plan_dev) return va_fail(VA_ERR_ARG, "null plan or shape");
  int rc = va::check_quant_pool(pool, shape);
  if (rc) return rc;
  const int32_t* h = plan_header_host;
  if (h[VA_H_MAGIC] != VA_PLAN_MAGIC) return va_fail(VA_ERR_ARG, "plan header has no magic word");
  if (h[VA_H_N_ROWS] == 0) return VA_OK;
  if (shape->num_q_heads <= 0 || shape->num_q_heads % shape->num_kv_heads)
    return va_fail(VA_ERR_ARG, "num_q_heads must be a multiple of num_kv_heads");
  if ((shape->dtype != VA_F16 && shape->dtype != VA_BF16) || h[VA_H_KERNEL] != VA_KERNEL_MFMA)
    return va_fail(VA_ERR_ARG, "rows are read back for 16-bit activations and matrix-core plans");
  if (n_slots < 0 || !q_dev || !out_dev || (n_slots > 0 && !slots_dev)) return va_fail(VA_ERR_ARG, "null pointer");
  const int64_t n_rows = h[VA_H_N_ROWS];
  const va::BackLayout l = va::back_layout(n_slots, n_rows, shape);
  if (!scratch_dev || scratch_bytes < l.bytes || (uintptr_t)scratch_dev % 256)
    return va_fail(VA_ERR_CAPACITY, "read-back needs %lld bytes of scratch on a 256-byte boundary, got %lld", (long long)l.bytes,
                   (long long)scratch_bytes);
  char* scratch = (char*)scratch_dev;
  hipStream_t s = (hipStream_t)stream;
  const int width = shape->num_q_heads * shape->head_dim;
  va::BackArgs a{{(const uint8_t*)pool->k_codes_dev, (const uint8_t*)pool->v_codes_dev},
                 {pool->k_scales_dev, pool->v_scales_dev}, slots_dev, n_slots,
                 (uint32_t)pool->num_pages * (uint32_t)shape->page_size, shape->num_kv_heads, shape->head_dim,
                 va::page_map(shape->page_size), (int32_t*)scratch, (uint32_t*)(scratch + l.tops),
                 {(__half*)(scratch + l.rows[0]), (__half*)(scratch + l.rows[1])},
                 q_dev, q_row_stride, (__half*)(scratch + l.q), n_rows, width, shape->dtype};
  const int pieces = (uintptr_t)q_dev % 16 == 0 && q_row_stride % 8 == 0;
  const bool e4m3 = pool->code_type == VA_CODE_E4M3;
  rc = e4m3 ? va::launch_quant_back<va::E4M3>(a, pieces, s) : va::launch_quant_back<va::INT8>(a, pieces, s);
  if (rc) return rc;
  VaShape half = *shape;
  half.dtype = VA_F16;
  rc = va::attention_launches(a.q16, width, a.rows[0], a.rows[1], (int64_t)shape->num_kv_heads * shape->head_dim, plan_dev, h,
                              kv_indices_dev, sub_worker_dev, sub_loc_dev, sub_loc_axis_stride, scratch + l.out, lse_dev,
                              lse_base2, workspace_dev, workspace_bytes, &half, rope, 1, stream);
  if (rc) return rc;
  const __half* from = (const __half*)(scratch + l.out);
  return e4m3 ? va::launch_quant_results<va::E4M3>(from, out_dev, lse_dev, a.tops, n_rows * width, shape->head_dim, shape->dtype, s)
              : va::launch_quant_results<va::INT8>(from, out_dev, lse_dev, a.tops, n_rows * width, shape->head_dim, shape->dtype, s);
}
