// Rotation of the queries and keys of a step by position, and the cos|sin table of the same frequencies.
//
//   angle(row, i) = pos[row] * f_i,  c = factor cos(angle), s = factor sin(angle)
//   (a, b) -> (a c - b s, b c + a s)   for the pairs (i, i + h) or (2 i, 2 i + 1) of every head, h = rotary_dim / 2
//
// The product of position and frequency is taken in 64 bits, in quarter turns (the frequencies come divided by pi / 2): the nearest
// whole number of them comes off exactly, so an angle at position 2^22 is as good as one at 1.  32 bits would be off by
// position * 2^-25 quarter turns there.  Cosines and sines, products and sums are 32-bit numbers, rounded once to the element type.
//
// A workgroup takes a token, or a few where a token's heads are few: it works their angles out once, a thread a pair, for all heads
// through LDS, then each thread takes units of 2 * kVec elements -- the two 16-byte pieces that hold both halves of kVec pairs, or
// two neighbouring ones -- of any token and head.  Bound by HBM, 2 * (Hq + Hkv) * head_dim elements a token: 16384 rows of 64 + 16 heads
// of 64 in 32 bits 120 us, 5.6 TB/s; 64 rows of 16 + 4 heads of 256 4 us.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>

#include "va_device.h"
#include "va_internal.h"
#include "va_launch.h"

namespace va {

typedef uint32_t va_rot_u32x4 __attribute__((ext_vector_type(4)));

constexpr int kRotThreads = 256;
constexpr int kRotPairs = 1024;  // (token, pair) angles of a workgroup

// Turns of whole positions by frequencies in quarter turns.
__device__ __forceinline__ float2 turn_at(double position, double quarters, float factor) {
  const double t = position * quarters, k = rint(t);
  const float r = (float)((t - k) * 1.57079632679489655800);
  float s, c;
  sin_cos_of_quadrant(r, (int)(k - 4.0 * floor(0.25 * k)), s, c);
  return make_float2(factor * c, factor * s);
}

struct RotateArgs {
  const void* x[2];  // q, k
  void* y[2];
  long long x_stride[2], y_stride[2];  // elements between rows
  int heads[2];
  const void* positions;
  int positions_i64;
  long long n_rows;
  int tokens;      // of a workgroup
  int head_dim, half;
  int units;       // of a head: pairs first, then what passes through
  uint32_t per_unit, per_head;  // ceil(2^32 / units), ceil(2^32 / heads)
  const double* quarters;
  float factor;
};

template <typename E, int kVec, bool kNeighbours, bool kPast>  // kPast: reads go past the caches
__global__ __launch_bounds__(kRotThreads) void rotate_kernel(RotateArgs a) {
  using S = typename E::storage;
  __shared__ float2 turns[kRotPairs];
  const long long first = (long long)blockIdx.x * a.tokens;
  const int n_tok = (int)min((long long)a.tokens, a.n_rows - first);
  for (int i = threadIdx.x; i < n_tok * a.half; i += kRotThreads) {
    const int t = i / a.half;
    const long long p = a.positions_i64 ? ((const int64_t*)a.positions)[first + t] : ((const int32_t*)a.positions)[first + t];
    turns[i] = turn_at((double)p, a.quarters[i - t * a.half], a.factor);
  }
  __syncthreads();
  const int heads = a.heads[0] + a.heads[1], pair_units = a.half / kVec;
  const int tasks = n_tok * heads * a.units;
  for (int task = threadIdx.x; task < tasks; task += kRotThreads) {
    const int row = a.units == 1 ? task : (int)__umulhi((uint32_t)task, a.per_unit), unit = task - row * a.units;
    const int t = heads == 1 ? row : (int)__umulhi((uint32_t)row, a.per_head), head = row - t * heads;
    const int which = head >= a.heads[0], h = head - (which ? a.heads[0] : 0);
    const S* from = (const S*)a.x[which] + (first + t) * a.x_stride[which] + (long long)h * a.head_dim;
    S* to = (S*)a.y[which] + (first + t) * a.y_stride[which] + (long long)h * a.head_dim;
    const bool turned = unit < pair_units;
    const int d0 = turned && !kNeighbours ? unit * kVec : 2 * unit * kVec;
    const int d1 = turned && !kNeighbours ? d0 + a.half : d0 + kVec;
    S lo[kVec], hi[kVec];
    if constexpr (kVec > 1) {
      const va_rot_u32x4 *p = (const va_rot_u32x4*)(from + d0), *q = (const va_rot_u32x4*)(from + d1);
      if constexpr (kPast) {
        *(va_rot_u32x4*)lo = __builtin_nontemporal_load(p), *(va_rot_u32x4*)hi = __builtin_nontemporal_load(q);
      } else {
        *(va_rot_u32x4*)lo = *p, *(va_rot_u32x4*)hi = *q;
      }
    } else {
      lo[0] = from[d0], hi[0] = from[d1];
    }
    if (turned) {
      float x[2 * kVec];
#pragma unroll
      for (int e = 0; e < kVec; ++e) x[e] = E::load(lo[e]), x[kVec + e] = E::load(hi[e]);
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const float2 cs = turns[t * a.half + unit * kVec + e];
        float& p = kNeighbours ? x[2 * e] : x[e];
        float& q = kNeighbours ? x[2 * e + 1] : x[kVec + e];
        const float y = p * cs.x - q * cs.y;
        q = q * cs.x + p * cs.y;
        p = y;
      }
#pragma unroll
      for (int e = 0; e < kVec; ++e) lo[e] = E::store(x[e]), hi[e] = E::store(x[kVec + e]);
    }
    if constexpr (kVec > 1) {
      *(va_rot_u32x4*)(to + d0) = *(va_rot_u32x4*)lo;
      *(va_rot_u32x4*)(to + d1) = *(va_rot_u32x4*)hi;
    } else {
      to[d0] = lo[0], to[d1] = hi[0];
    }
  }
}

__global__ __launch_bounds__(256) void rotary_table_kernel(const double* quarters, int half, float factor, long long first, long long n_rows,
                                                           float* table) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n_rows * half) return;
  const long long row = i / half;
  const int pair = (int)(i - row * half);
  const float2 cs = turn_at((double)(first + row), quarters[pair], factor);
  table[row * 2 * half + pair] = cs.x;
  table[row * 2 * half + half + pair] = cs.y;
}

static uint32_t reciprocal(int d) { return (uint32_t)(((1ull << 32) + d - 1) / d); }

template <typename E>
static int launch_rotate(RotateArgs& a, bool neighbours, hipStream_t stream) {
  constexpr int kWide = 16 / (int)sizeof(typename E::storage);
  bool wide = a.head_dim % (2 * kWide) == 0 && a.half % kWide == 0;
  for (int i = 0; i < 2; ++i)
    wide = wide && (!a.heads[i] || ((uintptr_t)a.x[i] % 16 == 0 && (uintptr_t)a.y[i] % 16 == 0 && a.x_stride[i] % kWide == 0 &&
                                    a.y_stride[i] % kWide == 0));
  const int heads = a.heads[0] + a.heads[1];
  a.units = a.head_dim / 2 / (wide ? kWide : 1);
  a.per_unit = reciprocal(a.units), a.per_head = reciprocal(heads);
  // (the quotients by reciprocals are exact below 2^32 / divisor)
  const long long row_tasks = (long long)heads * a.units;
  if (row_tasks * std::max(a.units, heads) >= (1ll << 31)) return va_fail(VA_ERR_ARG, "%d heads of %d dims are more than a workgroup counts", heads, a.head_dim);
  // As many tokens as give every thread a unit (16384 rows of 8 + 2 heads of 128: 15.1 us with four, 18.3 with one; of 64 + 16
  // heads of 64 in 32 bits 132 and 122), and one where there are few, so that all CUs have some.
  long long most = std::min<long long>((kRotThreads + row_tasks - 1) / row_tasks, (1ll << 31) / (row_tasks * std::max(a.units, heads)));
  if (a.half) most = std::min<long long>(most, kRotPairs / a.half);
  a.tokens = (int)std::max<long long>(1, std::min(most, a.n_rows / 2048));
  const long long groups = (a.n_rows + a.tokens - 1) / a.tokens;
  if (groups > 0x7fffffffLL) return va_fail(VA_ERR_ARG, "too many rows for one launch");
  // Rows and results that the 256 MB of the last cache do not hold (16384 rows of 32 + 8 heads of 128: 53 us past the caches, 61
  // through them; 4099 such rows, which it holds, 20.6 and 15.7).
  const bool past = wide && 2 * a.n_rows * heads * a.head_dim * (long long)sizeof(typename E::storage) > 256ll << 20;
  const dim3 grid((unsigned)groups), block(kRotThreads);
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, stream, a); };
  if (past) {
    neighbours ? launch(rotate_kernel<E, kWide, true, true>) : launch(rotate_kernel<E, kWide, false, true>);
  } else if (wide) {
    neighbours ? launch(rotate_kernel<E, kWide, true, false>) : launch(rotate_kernel<E, kWide, false, false>);
  } else {
    neighbours ? launch(rotate_kernel<E, 1, true, false>) : launch(rotate_kernel<E, 1, false, false>);
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? VA_OK : va_fail(VA_ERR_HIP, "rotation launch: %s", hipGetErrorString(e));
}

}  // namespace va

extern "C" int va_rotate_qk(const void* q_dev, int64_t q_row_stride, int32_t num_q_heads, void* out_q_dev, int64_t out_q_row_stride,
                            const void* k_dev, int64_t k_row_stride, int32_t num_k_heads, void* out_k_dev, int64_t out_k_row_stride,
                            const void* positions_dev, int32_t positions_are_i64, int64_t n_rows, int32_t head_dim, int32_t dtype,
                            const VaTurns* turns, void* stream) {
  if (!turns) return va_fail(VA_ERR_ARG, "null rotation description");
  const int rotary = turns->rotary_dim;
  if (n_rows < 0 || num_q_heads < 0 || num_k_heads < 0 || head_dim <= 0 || head_dim % 2) return va_fail(VA_ERR_ARG, "bad shape");
  if (rotary < 0 || rotary > head_dim || rotary % 2)
    return va_fail(VA_ERR_ARG, "rotary_dim %d must be even and within head_dim %d", rotary, head_dim);
  if (rotary / 2 > va::kRotPairs) return va_fail(VA_ERR_ARG, "rotary_dim %d is over %d", rotary, 2 * va::kRotPairs);
  if ((int64_t)num_q_heads + num_k_heads > INT32_MAX) return va_fail(VA_ERR_ARG, "too many heads");
  if (n_rows == 0 || num_q_heads + num_k_heads == 0) return VA_OK;
  if ((num_q_heads && (!q_dev || !out_q_dev)) || (num_k_heads && (!k_dev || !out_k_dev)) || (rotary && (!turns->quarters_dev || !positions_dev)))
    return va_fail(VA_ERR_ARG, "null pointer");
  if ((num_q_heads && n_rows > 1 && out_q_row_stride < (int64_t)num_q_heads * head_dim) ||
      (num_k_heads && n_rows > 1 && out_k_row_stride < (int64_t)num_k_heads * head_dim))
    return va_fail(VA_ERR_ARG, "output rows overlap");
  va::RotateArgs a{{q_dev, k_dev}, {out_q_dev, out_k_dev}, {q_row_stride, k_row_stride}, {out_q_row_stride, out_k_row_stride},
                   {num_q_heads, num_k_heads}, positions_dev, positions_are_i64, n_rows, 1, head_dim, rotary / 2, 0, 0, 0,
                   turns->quarters_dev, turns->factor};
  const bool neighbours = turns->neighbours != 0;
  switch (dtype) {
    case VA_F32:
      return va::launch_rotate<va::F32>(a, neighbours, (hipStream_t)stream);
    case VA_F16:
      return va::launch_rotate<va::F16>(a, neighbours, (hipStream_t)stream);
    case VA_BF16:
      return va::launch_rotate<va::BF16>(a, neighbours, (hipStream_t)stream);
    default:
      return va_fail(VA_ERR_ARG, "unknown dtype %d", (int)dtype);
  }
}

extern "C" int va_rotary_table(const VaTurns* turns, int64_t first_position, int64_t n_rows, float* table_dev, void* stream) {
  if (!turns) return va_fail(VA_ERR_ARG, "null rotation description");
  if (n_rows < 0 || turns->rotary_dim < 0 || turns->rotary_dim % 2 || turns->rotary_dim / 2 > va::kRotPairs) return va_fail(VA_ERR_ARG, "bad shape");
  const int half = turns->rotary_dim / 2;
  if (n_rows == 0 || half == 0) return VA_OK;
  if (!turns->quarters_dev || !table_dev) return va_fail(VA_ERR_ARG, "null pointer");
  const long long groups = n_rows > (1ll << 40) ? 1ll << 40 : (n_rows * half + 255) / 256;
  if (groups > 0x7fffffffLL) return va_fail(VA_ERR_ARG, "too many rows for one launch");
  hipLaunchKernelGGL(va::rotary_table_kernel, dim3((unsigned)groups), dim3(256), 0, (hipStream_t)stream, turns->quarters_dev, half, turns->factor,
                     first_position, n_rows, table_dev);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? VA_OK : va_fail(VA_ERR_HIP, "rotary table launch: %s", hipGetErrorString(e));
}
