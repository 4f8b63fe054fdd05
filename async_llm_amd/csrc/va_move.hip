// Tokens of a pool move to other slots in every layer, each key turned by a shift of its own: what eviction left of a block, put
// together, with the positions that the tokens have there.
//
//   k[dst] = round(R(shift_i) k[src]),  v[dst] = v[src],  weights[dst] = weights[src]
//
// Keys are rotated as 32-bit copies and rounded once; a key whose shift is 0 is copied bit for bit.  As in the copy with one shift
// (va_block_copy.hip) a workgroup owns kMoveTokens tokens of a layer and a thread a 16-byte piece position of the row, with which
// it walks the tokens; what differs is that every token has its own cosines and sines, looked up once a workgroup, in LDS.
// Bound by HBM: 4 * layers * kv_heads * head_dim * sizeof(element) bytes per token.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "va_copy_pieces.h"
#include "va_device.h"
#include "va_internal.h"
#include "va_launch.h"
#include "va_token_weights.h"

namespace va {

// Tokens of a workgroup, whose loads are in flight together: 12556 tokens of 4 layers of 4 heads of 256 87 us (4.7 TB/s), 95 with one,
// 92 with eight.
constexpr int kMoveTokens = 4;
constexpr int kMoveTurnBytes = 48 * 1024;

struct MoveArgs {
  void* k_pool;
  void* v_pool;
  long long pool_row_stride;  // elements between token slots
  long long layer_stride;     // elements between the pools of consecutive layers
  const int64_t* src;
  const int64_t* dst;
  const int64_t* shifts;  // null: nothing rotates
  long long n_tokens, num_slots;
  int tokens;  // of a workgroup
  int num_kv_heads, head_dim;
  RopeDev rope;
  TokenWeights weights;
};

template <typename E, int kVec>
__global__ __launch_bounds__(1024) void move_kernel(MoveArgs a) {
  using S = typename E::storage;
  using P = Piece<S, kVec>;
  extern __shared__ float2 turns[];  // [token][pair]
  __shared__ long long from[kMoveTokens], to[kMoveTokens];  // pool rows; a token that is skipped goes to -1
  __shared__ int still[kMoveTokens];
  const long long layer = blockIdx.y;
  const long long t0 = (long long)blockIdx.x * a.tokens;
  const int n_tok = (int)min((long long)a.tokens, a.n_tokens - t0);
  const int D = a.head_dim, half = a.shifts ? a.rope.half : 0;

  if ((int)threadIdx.x < n_tok) {
    const long long s = a.src[t0 + threadIdx.x], d = a.dst[t0 + threadIdx.x];
    const bool ok = s >= 0 && s < a.num_slots && d >= 0 && d < a.num_slots;
    from[threadIdx.x] = ok ? s : 0, to[threadIdx.x] = ok ? d : -1;
    still[threadIdx.x] = !a.shifts || a.shifts[t0 + threadIdx.x] == 0;
  }
  for (int i = threadIdx.x; i < n_tok * half; i += blockDim.x) {
    const int t = i / half;
    const long long shift = a.shifts[t0 + t];
    float c, s;
    rope_cos_sin(a.rope, Pos3{shift, shift, shift}, i - t * half, c, s);
    turns[i] = make_float2(c, s);
  }
  __syncthreads();
  if (layer == 0 && a.weights.sums)
    for (int i = threadIdx.x; i < n_tok * a.num_kv_heads; i += blockDim.x) {
      const int h = i / n_tok, t = i - h * n_tok;
      if (to[t] >= 0) move_weights(a.weights, h + 1, from[t], to[t], h, 1);
    }

  const int pair_pieces = half / kVec, pass_pieces = (D - 2 * half) / kVec;  // per head
  const int n_pair = a.num_kv_heads * pair_pieces, n_pass = a.num_kv_heads * pass_pieces, n_v = a.num_kv_heads * D / kVec;
  S* kp = (S*)a.k_pool + layer * a.layer_stride;
  S* vp = (S*)a.v_pool + layer * a.layer_stride;
  for (int task = threadIdx.x; task < n_pair + n_pass + n_v; task += blockDim.x) {
    if (task < n_pair) {
      const int h = task / pair_pieces, j = task - h * pair_pieces;
      const long long off = (long long)h * D + (long long)j * kVec;
      P x1[kMoveTokens], x2[kMoveTokens];
#pragma unroll
      for (int u = 0; u < kMoveTokens; ++u) {
        const S* row = kp + from[min(u, n_tok - 1)] * a.pool_row_stride + off;
        x1[u] = load_piece<S, kVec>(row);
        x2[u] = load_piece<S, kVec>(row + half);
      }
#pragma unroll
      for (int u = 0; u < kMoveTokens; ++u)
        if (u < n_tok && to[u] >= 0) {
          if (!still[u])
#pragma unroll
            for (int e = 0; e < kVec; ++e) {
              const float2 cs = turns[u * half + j * kVec + e];
              float r1, r2;
              rope_pair<F32>(a.rope, cs.x, cs.y, E::load(x1[u].v[e]), E::load(x2[u].v[e]), r1, r2);
              x1[u].v[e] = E::store(r1);
              x2[u].v[e] = E::store(r2);
            }
          S* row = kp + to[u] * a.pool_row_stride + off;
          store_piece<S, kVec>(row, x1[u]);
          store_piece<S, kVec>(row + half, x2[u]);
        }
    } else {
      // plain pieces: the rest of K, then V
      S* pool = kp;
      long long off;
      const int t = task - n_pair;
      if (t < n_pass) {
        const int h = t / pass_pieces, j = t - h * pass_pieces;
        off = (long long)h * D + 2 * half + (long long)j * kVec;
      } else {
        pool = vp;
        off = (long long)(t - n_pass) * kVec;
      }
      P x[kMoveTokens];
#pragma unroll
      for (int u = 0; u < kMoveTokens; ++u) x[u] = load_piece<S, kVec>(pool + from[min(u, n_tok - 1)] * a.pool_row_stride + off);
#pragma unroll
      for (int u = 0; u < kMoveTokens; ++u)
        if (u < n_tok && to[u] >= 0) store_piece<S, kVec>(pool + to[u] * a.pool_row_stride + off, x[u]);
    }
  }
}

// A thread per token and head.
__global__ __launch_bounds__(256) void move_weights_kernel(TokenWeights weights, const int64_t* src, const int64_t* dst, long long n) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const long long s = src[i], d = dst[i];
  if (s >= 0 && s < weights.slots && d >= 0 && d < weights.slots) move_weights(weights, (int)blockIdx.y + 1, s, d, (int)blockIdx.y, 1);
}

int launch_move_weights(const TokenWeights& w, int heads, const int64_t* src, const int64_t* dst, long long n, hipStream_t stream) {
  if (heads > 65535 || n > 0x7fffffffLL * 256) return va_fail(VA_ERR_ARG, "too many tokens or heads for one launch");
  hipLaunchKernelGGL(move_weights_kernel, dim3((unsigned)((n + 255) / 256), (unsigned)heads), dim3(256), 0, stream, w, src, dst, n);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? VA_OK : va_fail(VA_ERR_HIP, "moving weights: %s", hipGetErrorString(e));
}

// A thread per slot and head: weights[h][slots[i]] = 0.
__global__ __launch_bounds__(256) void clear_weights_kernel(TokenWeights weights, const int64_t* slots, long long n) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const long long slot = slots[i];
  if (slot >= 0 && slot < weights.slots) weights.sums[(long long)blockIdx.y * weights.slots + slot] = 0.f;
}

template <typename E>
static int launch_move(MoveArgs& a, int num_layers, hipStream_t stream) {
  using S = typename E::storage;
  constexpr int kWide = 16 / (int)sizeof(S);
  const int half = a.shifts ? a.rope.half : 0;
  auto aligned = [](const void* p) { return ((uintptr_t)p & 15) == 0; };
  const bool wide = a.head_dim % kWide == 0 && half % kWide == 0 && a.pool_row_stride % kWide == 0 &&
                    a.layer_stride % kWide == 0 && aligned(a.k_pool) && aligned(a.v_pool);
  const int vec = wide ? kWide : 1;
  const long long tasks = (long long)a.num_kv_heads * (half / vec + (a.head_dim - 2 * half) / vec + a.head_dim / vec);
  if (tasks > 0x7fffffffLL || half * (int)sizeof(float2) > kMoveTurnBytes) return va_fail(VA_ERR_ARG, "rows of %d heads of %d dims are too long", a.num_kv_heads, a.head_dim);
  const unsigned threads = (unsigned)std::min<long long>(1024, (tasks + 63) / 64 * 64);
  a.tokens = half ? std::min(kMoveTokens, kMoveTurnBytes / (half * (int)sizeof(float2))) : kMoveTokens;
  const long long groups = (a.n_tokens + a.tokens - 1) / a.tokens;
  if (groups > 0x7fffffffLL || num_layers > 65535) return va_fail(VA_ERR_ARG, "too many tokens or layers for one launch");
  const dim3 grid((unsigned)groups, (unsigned)num_layers);
  const unsigned bytes = (unsigned)(a.tokens * half * (int)sizeof(float2));
  if (wide) {
    hipLaunchKernelGGL((move_kernel<E, kWide>), grid, dim3(threads), bytes, stream, a);
  } else {
    hipLaunchKernelGGL((move_kernel<E, 1>), grid, dim3(threads), bytes, stream, a);
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? VA_OK : va_fail(VA_ERR_HIP, "move launch: %s", hipGetErrorString(e));
}

}  // namespace va

extern "C" int va_move_kv(void* k_pool_dev, void* v_pool_dev, int64_t pool_row_stride, int64_t layer_stride, int32_t num_layers,
                          int64_t num_slots, const int64_t* src_slots_dev, const int64_t* dst_slots_dev, const int64_t* shifts_dev,
                          int64_t n_tokens, float* weights_dev, const VaShape* shape, const VaRope* rope, void* stream) {
  if (!shape) return va_fail(VA_ERR_ARG, "null shape");
  if (n_tokens < 0 || num_layers < 0 || num_slots < 0) return va_fail(VA_ERR_ARG, "negative count");
  if (n_tokens == 0 || num_slots == 0 || (num_layers == 0 && !weights_dev)) return VA_OK;
  if ((num_layers && (!k_pool_dev || !v_pool_dev)) || !src_slots_dev || !dst_slots_dev) return va_fail(VA_ERR_ARG, "null pointer");
  if (shape->num_kv_heads <= 0 || shape->head_dim <= 0) return va_fail(VA_ERR_ARG, "bad shape");
  const va::TokenWeights weights{weights_dev, (long long)num_slots};
  if (num_layers == 0) return va::launch_move_weights(weights, shape->num_kv_heads, src_slots_dev, dst_slots_dev, n_tokens, (hipStream_t)stream);
  if (pool_row_stride < (int64_t)shape->num_kv_heads * shape->head_dim)
    return va_fail(VA_ERR_ARG, "pool rows overlap: stride %lld < %d elements", (long long)pool_row_stride,
                   shape->num_kv_heads * shape->head_dim);
  va::MoveArgs a{k_pool_dev, v_pool_dev, pool_row_stride, layer_stride, src_slots_dev, dst_slots_dev, nullptr, n_tokens, num_slots, 1,
                 shape->num_kv_heads, shape->head_dim, va::RopeDev{}, weights};
  if (shifts_dev) {
    const int rc = va::make_rope(rope, shape->head_dim, &a.rope);
    if (rc) return rc;
    if (a.rope.half > 0) a.shifts = shifts_dev;  // (nothing rotates: a plain copy)
  }
  switch (shape->dtype) {
    case VA_F32:
      return va::launch_move<va::F32>(a, num_layers, (hipStream_t)stream);
    case VA_F16:
      return va::launch_move<va::F16>(a, num_layers, (hipStream_t)stream);
    case VA_BF16:
      return va::launch_move<va::BF16>(a, num_layers, (hipStream_t)stream);
    default:
      return va_fail(VA_ERR_ARG, "unknown dtype %d", (int)shape->dtype);
  }
}

extern "C" int va_clear_weights(float* weights_dev, int32_t num_heads, int64_t num_slots, const int64_t* slots_dev, int64_t n, void* stream) {
  if (num_heads < 0 || num_slots < 0 || n < 0) return va_fail(VA_ERR_ARG, "negative count");
  if (num_heads == 0 || num_slots == 0 || n == 0) return VA_OK;
  if (!weights_dev || !slots_dev) return va_fail(VA_ERR_ARG, "null pointer");
  if (num_heads > 65535 || n > 0x7fffffffLL * 256) return va_fail(VA_ERR_ARG, "too many slots or heads for one launch");
  hipLaunchKernelGGL(va::clear_weights_kernel, dim3((unsigned)((n + 255) / 256), (unsigned)num_heads), dim3(256), 0, (hipStream_t)stream,
                     va::TokenWeights{weights_dev, (long long)num_slots}, slots_dev, n);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? VA_OK : va_fail(VA_ERR_HIP, "clearing weights: %s", hipGetErrorString(e));
}
