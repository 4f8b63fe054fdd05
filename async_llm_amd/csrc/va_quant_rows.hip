// Rows of a quantised pool: writing them (rotation and quantisation), reading them back, moving them to other slots
// (the keys rotated by a shift on the way).  All three are bound by HBM, or by their launch where rows are few.
#include <hip/hip_runtime.h>

#include "va_internal.h"
#include "va_launch.h"
#include "va_quant.h"

namespace va {

int check_quant_pool(const VaQuantPool* pool, const VaShape* shape) {
  if (!pool || !shape) return va_fail(VA_ERR_ARG, "null pool or shape");
  if (pool->code_type != VA_CODE_E4M3 && pool->code_type != VA_CODE_INT8)
    return va_fail(VA_ERR_ARG, "unknown code type %d", pool->code_type);
  if (!pool->k_codes_dev || !pool->v_codes_dev || !pool->k_scales_dev || !pool->v_scales_dev)
    return va_fail(VA_ERR_ARG, "null pool array");
  if ((uintptr_t)pool->k_codes_dev % 16 || (uintptr_t)pool->v_codes_dev % 16)
    return va_fail(VA_ERR_ARG, "code arrays must start on 16-byte boundaries");
  if (shape->num_kv_heads <= 0 || shape->page_size <= 0 || pool->num_pages < 0)
    return va_fail(VA_ERR_ARG, "bad shape");
  const int d = shape->head_dim;
  if (d != 16 && d != 32 && d != 64 && d != 128 && d != 256)
    return va_fail(VA_ERR_ARG, "head_dim %d unsupported (16, 32, 64, 128 or 256)", d);
  if ((int64_t)pool->num_pages * shape->page_size > 0x7fffffffLL)
    return va_fail(VA_ERR_ARG, "a pool of %d pages of %d tokens has more slots than 32 bits address", pool->num_pages, shape->page_size);
  return VA_OK;
}

static int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? VA_OK : va_fail(VA_ERR_HIP, "%s launch: %s", what, hipGetErrorString(e));
}

// Largest magnitude, as bits, over the kLanes lanes of a row (neighbours, aligned).
template <int kLanes>
__device__ __forceinline__ uint32_t top_of_row(uint32_t top) {
#pragma unroll
  for (int off = kLanes / 2; off > 0; off >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, off, kWave));
  return top;
}

// Eight activations at `p` (16-byte aligned) as fp32.
template <typename E>
__device__ __forceinline__ void load8(const typename E::storage* p, float* x) {
  using S = typename E::storage;
  constexpr int kPieces = 8 * sizeof(S) / 16;
  union {
    uint4 raw[kPieces];
    S e[8];
  } u;
#pragma unroll
  for (int i = 0; i < kPieces; ++i) u.raw[i] = ((const uint4*)p)[i];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = E::load(u.e[i]);
}

__device__ __forceinline__ uint32_t top8(const float* x) {
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(x[k]) & 0x7fffffffu);
  return top;
}

// Codes of eight elements of a row with this scale.
template <typename C>
__device__ __forceinline__ uint2 codes8(const float* x, int scale) {
  if (scale == 255) return make_uint2(0, 0);
  const float f = inverse_scale(scale);
  float y[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) y[k] = limited<C>(x[k]) * f;
  return make_uint2(C::pack4(y[0], y[1], y[2], y[3]), C::pack4(y[4], y[5], y[6], y[7]));
}

struct StoreArgs {
  const void* x[2];  // k, v
  long long x_stride[2];
  uint8_t* codes[2];
  uint8_t* scales[2];
  const void* dst;
  int dst_is_i64;
  const int64_t* pos;
  long long pos_axis_stride;
  long long n_rows;
  uint32_t num_slots;
  int num_kv_heads, head_dim;
  PageMap pages;
  RopeDev rope;
};

__device__ __forceinline__ bool slot_of_row(const void* dst, int is_i64, long long row, uint32_t num_slots, uint32_t& slot) {
  const long long s = is_i64 ? ((const long long*)dst)[row] : (long long)((const int*)dst)[row];
  slot = (uint32_t)s;
  return s >= 0 && s < (long long)num_slots;
}

// Any alignment and rotary width: a wave per (row, head) of k (blockIdx.y 0) or v (1), a lane every 64th element.
template <typename E, typename C>
__global__ __launch_bounds__(256) void quant_store_kernel(StoreArgs a) {
  const long long unit = (long long)blockIdx.x * 4 + threadIdx.x / kWave;
  const int lane = threadIdx.x % kWave, which = blockIdx.y;
  const long long row = unit / a.num_kv_heads;
  if (row >= a.n_rows) return;
  const int h = (int)(unit - row * a.num_kv_heads), D = a.head_dim;
  uint32_t slot;
  if (!slot_of_row(a.dst, a.dst_is_i64, row, a.num_slots, slot)) return;
  const typename E::storage* x = (const typename E::storage*)(which ? a.x[1] : a.x[0]) +
                                 row * (which ? a.x_stride[1] : a.x_stride[0]) + (long long)h * D;
  const int rotary = which ? 0 : a.rope.rotary_dim, half = rotary / 2;
  Pos3 p{0, 0, 0};
  if (rotary) p = load_pos(a.pos, a.pos_axis_stride, row);
  float y[4];
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int d = lane + 64 * k;
    y[k] = 0.f;
    if (d < D) {
      if (d < rotary) {
        const int i = d < half ? d : d - half;
        float c, s, y1, y2;
        rope_cos_sin(a.rope, p, i, c, s);
        const float x1 = E::load(x[i]), x2 = E::load(x[i + half]);
        y1 = mul_rounded(c, x1) - mul_rounded(s, x2);
        y2 = mul_rounded(c, x2) + mul_rounded(s, x1);
        y[k] = d < half ? y1 : y2;
      } else {
        y[k] = E::load(x[d]);
      }
      top = max(top, __float_as_uint(y[k]) & 0x7fffffffu);
    }
  }
  const int scale = scale_of<C>(top_of_row<kWave>(top));
  const long long r = quant_row(a.pages, slot, h, a.num_kv_heads);
  uint8_t* codes = (which ? a.codes[1] : a.codes[0]) + r * D;
  const float f = inverse_scale(scale);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int d = lane + 64 * k;
    if (d < D) codes[d] = scale == 255 ? (uint8_t)0 : (uint8_t)C::pack4(limited<C>(y[k]) * f, 0.f, 0.f, 0.f);
  }
  if (lane == 0) (which ? a.scales[1] : a.scales[0])[r] = (uint8_t)scale;
}

// The same where rows start on 16-byte boundaries and rotary_dim is a multiple of 16: a row is kD / 16 neighbouring
// lanes with sixteen elements each, two pieces of eight that rotate together or lie side by side, and one
// store of codes for each piece.  64 rows of 4 heads of 256 dims are 32 workgroups: the launch is all there is; long
// runs are bound by HBM.
template <typename E, typename C, int kD>
__global__ __launch_bounds__(256) void quant_store_vec_kernel(StoreArgs a) {
  using S = typename E::storage;
  constexpr int kLanes = kD / 16;
  const unsigned idx = blockIdx.x * 256u + threadIdx.x;  // (the launcher keeps the units within 32 bits)
  const int x = idx % kLanes, which = blockIdx.y;
  const unsigned unit = idx / kLanes;
  const long long row = unit / (unsigned)a.num_kv_heads;
  const int h = (int)(unit - (unsigned)row * (unsigned)a.num_kv_heads);
  uint32_t slot;
  if (row >= a.n_rows || !slot_of_row(a.dst, a.dst_is_i64, row, a.num_slots, slot)) return;  // (whole rows leave)
  const S* in = (const S*)(which ? a.x[1] : a.x[0]) + row * (which ? a.x_stride[1] : a.x_stride[0]) + (long long)h * kD;
  const int pairs = which ? 0 : a.rope.rotary_dim / 16;  // lanes whose pieces rotate together
  const int d0 = x < pairs ? 8 * x : 16 * x, d1 = x < pairs ? 8 * x + a.rope.half : 16 * x + 8;
  float lo[8], hi[8];
  load8<E>(in + d0, lo);
  load8<E>(in + d1, hi);
  if (x < pairs) {
    float c[8], s[8];
    turns8(a.rope, load_pos(a.pos, a.pos_axis_stride, row), d0, c, s);
    turn8(c, s, lo, hi);
  }
  const int scale = scale_of<C>(top_of_row<kLanes>(max(top8(lo), top8(hi))));
  const long long r = quant_row(a.pages, slot, h, a.num_kv_heads);
  uint8_t* codes = (which ? a.codes[1] : a.codes[0]) + r * kD;
  *(uint2*)(codes + d0) = codes8<C>(lo, scale);
  *(uint2*)(codes + d1) = codes8<C>(hi, scale);
  if (x == 0) (which ? a.scales[1] : a.scales[0])[r] = (uint8_t)scale;
}

template <typename E, typename C>
static int launch_quant_store(const StoreArgs& a, hipStream_t stream) {
  constexpr int kVec = 16 / sizeof(typename E::storage);
  const bool pieces = (uintptr_t)a.x[0] % 16 == 0 && (uintptr_t)a.x[1] % 16 == 0 && a.x_stride[0] % kVec == 0 &&
                      a.x_stride[1] % kVec == 0 && a.rope.rotary_dim % 16 == 0 &&
                      (a.rope.rotary_dim == 0 || a.rope.mode != VA_ROPE_TABLE || (uintptr_t)a.rope.cos_sin % 16 == 0);
  const long long units = a.n_rows * a.num_kv_heads;
  if (pieces && units * (a.head_dim / 16) < 0x7fffff00LL) {
    const dim3 grid((unsigned)((units * (a.head_dim / 16) + 255) / 256), 2), block(256);
    switch (a.head_dim) {
#define VA_CASE(D) \
  case D:          \
    hipLaunchKernelGGL((quant_store_vec_kernel<E, C, D>), grid, block, 0, stream, a); \
    break;
      VA_CASE(16) VA_CASE(32) VA_CASE(64) VA_CASE(128) VA_CASE(256)
#undef VA_CASE
    }
    return launched("quantising store");
  }
  if (units > 4 * 0x7fffffffLL) return va_fail(VA_ERR_ARG, "too many rows");
  hipLaunchKernelGGL((quant_store_kernel<E, C>), dim3((unsigned)((units + 3) / 4), 2), dim3(256), 0, stream, a);
  return launched("quantising store");
}

// ---------------------------------------------------------------------------
// reading back
// ---------------------------------------------------------------------------
struct LoadArgs {
  const uint8_t* codes[2];
  const uint8_t* scales[2];
  void* out[2];
  long long out_stride;
  const int64_t* slots;
  long long n_rows;
  uint32_t num_slots;
  int num_kv_heads, head_dim, first;
  PageMap pages;
};

// A thread takes eight codes, neighbours neighbouring ones of a row, heads and rows after one another.  Bound by HBM: a
// view of 254 MB (a third codes, the rest written) 41 us, 6.1 TB/s; with stores that stay in the caches 66.
template <typename E, typename C>
__global__ __launch_bounds__(256) void quant_load_kernel(LoadArgs a, int per_head, int per_row) {
  using S = typename E::storage;
  const unsigned idx = blockIdx.x * 256u + threadIdx.x;
  const long long row = idx / (unsigned)per_row;
  if (row >= a.n_rows) return;
  const int u = (int)(idx - (unsigned)row * (unsigned)per_row), h = u / per_head, d0 = 8 * (u - h * per_head);
  const int which = a.first + blockIdx.y;
  union {
    uint4 raw[8 * sizeof(S) / 16];
    S e[8];
  } y;
  const long long s = a.slots[row];
  if (s >= 0 && s < (long long)a.num_slots) {
    const long long r = quant_row(a.pages, (uint32_t)s, h, a.num_kv_heads);
    const uint2 codes = *(const uint2*)((which ? a.codes[1] : a.codes[0]) + r * a.head_dim + d0);
    const float f = scale_value((which ? a.scales[1] : a.scales[0])[r]);
    float x[8];
    C::unpack4(codes.x, x);
    C::unpack4(codes.y, x + 4);
#pragma unroll
    for (int k = 0; k < 8; ++k) y.e[k] = E::store(x[k] * f);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) y.e[k] = E::store(0.f);
  }
  S* out = (S*)(which ? a.out[1] : a.out[0]) + row * a.out_stride + (long long)h * a.head_dim + d0;
  if (((uintptr_t)out & 15) == 0) {
#pragma unroll
    for (int i = 0; i < (int)(8 * sizeof(S) / 16); ++i)
      __builtin_nontemporal_store(__builtin_bit_cast(va_u32x4, y.raw[i]), (va_u32x4*)out + i);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) out[k] = y.e[k];
  }
}

template <typename E, typename C>
static int launch_quant_load(const LoadArgs& a_in, hipStream_t stream) {
  LoadArgs a = a_in;
  const int per_head = a.head_dim / 8, per_row = a.num_kv_heads * per_head;
  a.first = a.out[0] ? 0 : 1;
  const unsigned kinds = (a.out[0] ? 1 : 0) + (a.out[1] ? 1 : 0);
  // (runs of rows whose threads 32 bits count)
  const long long most = 0x7fffff00LL / per_row;
  for (long long at = 0; at < a_in.n_rows; at += most) {
    a.n_rows = a_in.n_rows - at < most ? a_in.n_rows - at : most;
    a.slots = a_in.slots + at;
    for (int w = 0; w < 2; ++w)
      if (a_in.out[w]) a.out[w] = (typename E::storage*)a_in.out[w] + at * a.out_stride;
    hipLaunchKernelGGL((quant_load_kernel<E, C>), dim3((unsigned)((a.n_rows * per_row + 255) / 256), kinds), dim3(256), 0,
                       stream, a, per_head, per_row);
    const int rc = launched("read-back");
    if (rc) return rc;
  }
  return VA_OK;
}

// ---------------------------------------------------------------------------
// copy with a shift
// ---------------------------------------------------------------------------
constexpr int kQuantCopyTokens = 16;  // tokens per workgroup
constexpr int kQuantCopyBatch = 4;    // heads whose loads are in flight together

struct QuantCopyArgs {
  uint8_t* codes[2];
  uint8_t* scales[2];
  long long code_layer_stride, scale_layer_stride;
  const int64_t* src;
  const int64_t* dst;
  long long n_tokens;
  long long shift;  // 0: nothing rotates
  uint32_t num_slots;
  int num_kv_heads;
  PageMap pages;
  RopeDev rope;
};

// A workgroup moves the keys (blockIdx.z 0) or values (1) of kQuantCopyTokens tokens of a layer.  As in the store a row is
// kD / 16 neighbouring lanes; a thread keeps its token and its place in the row, so the slots and the turns of its pairs
// are looked up once, and walks the heads: neighbouring rows of a wave are neighbouring tokens of a page, one run of
// memory.  Bound by HBM: 12556 tokens of 4 layers of 4 heads of 256 dims (207 MB read and written) 39 us, 5.3 TB/s; with a thread
// walking sixteen tokens of its head 66 us, with stores that stay in the caches 49.  Small copies are bound by the trip
// slot, scale and codes, store: 5.6 us for 4.3 MB (17 with walks).  kTurn: keys are rotated (rotary_dim a multiple of 16);
// otherwise they move code for code like the values.
template <typename C, int kD, bool kTurn>
__global__ __launch_bounds__(256) void quant_copy_kernel(QuantCopyArgs a) {
  constexpr int kLanes = kD / 16, kHeads = 256 / kLanes / kQuantCopyTokens;  // heads side by side
  const int x = threadIdx.x % kLanes, which = blockIdx.z;
  const long long layer = blockIdx.y, i = (long long)blockIdx.x * kQuantCopyTokens + threadIdx.x / kLanes % kQuantCopyTokens;
  if (i >= a.n_tokens) return;  // (whole rows leave)
  const long long src = a.src[i], dst = a.dst[i];
  if (src < 0 || src >= (long long)a.num_slots || dst < 0 || dst >= (long long)a.num_slots) return;
  uint8_t* codes = (which ? a.codes[1] : a.codes[0]) + layer * a.code_layer_stride;
  uint8_t* scales = (which ? a.scales[1] : a.scales[0]) + layer * a.scale_layer_stride;
  const long long from = quant_row(a.pages, (uint32_t)src, 0, a.num_kv_heads);
  const long long to = quant_row(a.pages, (uint32_t)dst, 0, a.num_kv_heads);
  const int first = threadIdx.x / (kLanes * kQuantCopyTokens);
  if (!kTurn || which) {
    for (int h0 = first; h0 < a.num_kv_heads; h0 += kQuantCopyBatch * kHeads) {
      va_u32x4 row[kQuantCopyBatch];
      uint8_t e[kQuantCopyBatch];
#pragma unroll
      for (int u = 0; u < kQuantCopyBatch; ++u) {
        const long long r = from + (long long)min(h0 + u * kHeads, a.num_kv_heads - 1) * a.pages.size;
        row[u] = *(const va_u32x4*)(codes + r * kD + 16 * x);
        e[u] = scales[r];
      }
#pragma unroll
      for (int u = 0; u < kQuantCopyBatch; ++u) {
        if (h0 + u * kHeads >= a.num_kv_heads) break;
        const long long r = to + (long long)(h0 + u * kHeads) * a.pages.size;
        __builtin_nontemporal_store(row[u], (va_u32x4*)(codes + r * kD + 16 * x));
        if (x == 0) scales[r] = e[u];
      }
    }
    return;
  }
  const bool turns = x < a.rope.rotary_dim / 16;
  const int d0 = turns ? 8 * x : 16 * x, d1 = turns ? 8 * x + a.rope.half : 16 * x + 8;
  float c[8], s[8];
  if (turns) turns8(a.rope, Pos3{a.shift, a.shift, a.shift}, d0, c, s);
  for (int h0 = first; h0 < a.num_kv_heads; h0 += kQuantCopyBatch * kHeads) {
    uint2 lo[kQuantCopyBatch], hi[kQuantCopyBatch];
    uint32_t e[kQuantCopyBatch];
#pragma unroll
    for (int u = 0; u < kQuantCopyBatch; ++u) {
      const long long r = from + (long long)min(h0 + u * kHeads, a.num_kv_heads - 1) * a.pages.size;
      lo[u] = *(const uint2*)(codes + r * kD + d0);
      hi[u] = *(const uint2*)(codes + r * kD + d1);
      e[u] = scales[r];
    }
#pragma unroll
    for (int u = 0; u < kQuantCopyBatch; ++u) {
      const int h = h0 + u * kHeads;
      float p[8], q[8];
      const float f = scale_value(e[u]);
      C::unpack4(lo[u].x, p), C::unpack4(lo[u].y, p + 4), C::unpack4(hi[u].x, q), C::unpack4(hi[u].y, q + 4);
#pragma unroll
      for (int k = 0; k < 8; ++k) p[k] *= f, q[k] *= f;
      if (turns) turn8(c, s, p, q);
      e[u] = scale_of<C>(top_of_row<kLanes>(max(top8(p), top8(q))));
      lo[u] = codes8<C>(p, e[u]);
      hi[u] = codes8<C>(q, e[u]);
      if (h < a.num_kv_heads) {
        const long long r = to + (long long)h * a.pages.size;
        __builtin_nontemporal_store(__builtin_bit_cast(va_u32x2, lo[u]), (va_u32x2*)(codes + r * kD + d0));
        __builtin_nontemporal_store(__builtin_bit_cast(va_u32x2, hi[u]), (va_u32x2*)(codes + r * kD + d1));
        if (x == 0) scales[r] = (uint8_t)e[u];
      }
    }
  }
}

// Rotary widths that no multiple of 16 is: a wave per (token, head) of a layer, a lane every 64th element; a rotating key
// is read whole before it is written, so rows may be rewritten in place.
template <typename C>
__global__ __launch_bounds__(256) void quant_copy_any_kernel(QuantCopyArgs a, int D) {
  const long long unit = (long long)blockIdx.x * 4 + threadIdx.x / kWave, layer = blockIdx.y;
  const int lane = threadIdx.x % kWave;
  const long long i = unit / a.num_kv_heads;
  if (i >= a.n_tokens) return;
  const int h = (int)(unit - i * a.num_kv_heads);
  const long long src = a.src[i], dst = a.dst[i];
  if (src < 0 || src >= (long long)a.num_slots || dst < 0 || dst >= (long long)a.num_slots) return;
  const long long from = quant_row(a.pages, (uint32_t)src, h, a.num_kv_heads), to = quant_row(a.pages, (uint32_t)dst, h, a.num_kv_heads);
  const Pos3 p{a.shift, a.shift, a.shift};
  uint8_t* codes = a.codes[0] + layer * a.code_layer_stride;
  uint8_t* scales = a.scales[0] + layer * a.scale_layer_stride;
  const float f = scale_value(scales[from]);
  auto element = [&](int d) __attribute__((always_inline)) {
    float x[4];
    C::unpack4(codes[from * D + d], x);
    return x[0] * f;
  };
  float y[4];
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int d = lane + 64 * k;
    y[k] = 0.f;
    if (d < D) {
      y[k] = element(d);
      if (d < a.rope.rotary_dim) {
        const bool first = d < a.rope.half;
        const float other = element(first ? d + a.rope.half : d - a.rope.half);
        float c, s;
        rope_cos_sin(a.rope, p, first ? d : d - a.rope.half, c, s);
        y[k] = first ? mul_rounded(c, y[k]) - mul_rounded(s, other) : mul_rounded(c, y[k]) + mul_rounded(s, other);
      }
      top = max(top, __float_as_uint(y[k]) & 0x7fffffffu);
    }
  }
  const int scale = scale_of<C>(top_of_row<kWave>(top));  // (every lane has read its elements when the wave is here)
  const float inv = inverse_scale(scale);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int d = lane + 64 * k;
    if (d < D) codes[to * D + d] = scale == 255 ? (uint8_t)0 : (uint8_t)C::pack4(limited<C>(y[k]) * inv, 0.f, 0.f, 0.f);
  }
  if (lane == 0) scales[to] = (uint8_t)scale;
  const uint8_t* v_from = a.codes[1] + layer * a.code_layer_stride + from * D;
  uint8_t* v_to = a.codes[1] + layer * a.code_layer_stride + to * D;
  for (int d = lane; d < D; d += 64) v_to[d] = v_from[d];
  if (lane == 0) a.scales[1][layer * a.scale_layer_stride + to] = a.scales[1][layer * a.scale_layer_stride + from];
}

template <typename C>
static int launch_quant_copy(const QuantCopyArgs& a, int head_dim, int num_layers, hipStream_t stream) {
  const bool turn = a.shift != 0 && a.rope.half > 0;
  const bool pieces = !turn || (a.rope.rotary_dim % 16 == 0 && (a.rope.mode != VA_ROPE_TABLE || (uintptr_t)a.rope.cos_sin % 16 == 0));
  if (num_layers > 65535) return va_fail(VA_ERR_ARG, "too many layers for one launch");
  if (!pieces) {
    const long long groups = (a.n_tokens * a.num_kv_heads + 3) / 4;
    if (groups > 0x7fffffffLL) return va_fail(VA_ERR_ARG, "too many tokens for one launch");
    hipLaunchKernelGGL(quant_copy_any_kernel<C>, dim3((unsigned)groups, (unsigned)num_layers), dim3(256), 0, stream, a, head_dim);
    return launched("quantised copy");
  }
  const long long groups = (a.n_tokens + kQuantCopyTokens - 1) / kQuantCopyTokens;
  if (groups > 0x7fffffffLL) return va_fail(VA_ERR_ARG, "too many tokens for one launch");
  const dim3 grid((unsigned)groups, (unsigned)num_layers, 2), block(256);
  switch (head_dim) {
#define VA_CASE(D)                                                                            \
  case D:                                                                                     \
    if (turn) {                                                                               \
      hipLaunchKernelGGL((quant_copy_kernel<C, D, true>), grid, block, 0, stream, a);         \
    } else {                                                                                  \
      hipLaunchKernelGGL((quant_copy_kernel<C, D, false>), grid, block, 0, stream, a);        \
    }                                                                                         \
    break;
    VA_CASE(16) VA_CASE(32) VA_CASE(64) VA_CASE(128) VA_CASE(256)
#undef VA_CASE
  }
  return launched("quantised copy");
}

}  // namespace va

#define VA_DISPATCH_ROWS(dtype, code, CALL)                                                        \
  switch (2 * (dtype) + (code)) {                                                                  \
    case 2 * VA_F32 + VA_CODE_E4M3: { using E = va::F32; using C = va::E4M3; rc = CALL; } break;   \
    case 2 * VA_F32 + VA_CODE_INT8: { using E = va::F32; using C = va::INT8; rc = CALL; } break;   \
    case 2 * VA_F16 + VA_CODE_E4M3: { using E = va::F16; using C = va::E4M3; rc = CALL; } break;   \
    case 2 * VA_F16 + VA_CODE_INT8: { using E = va::F16; using C = va::INT8; rc = CALL; } break;   \
    case 2 * VA_BF16 + VA_CODE_E4M3: { using E = va::BF16; using C = va::E4M3; rc = CALL; } break; \
    case 2 * VA_BF16 + VA_CODE_INT8: { using E = va::BF16; using C = va::INT8; rc = CALL; } break; \
    default: rc = va_fail(VA_ERR_ARG, "unknown dtype %d", (int)(dtype));                           \
  }

extern "C" int va_store_kv_rope_q8(const void* k_dev, const void* v_dev, int64_t k_row_stride, int64_t v_row_stride,
                                   const VaQuantPool* pool, const void* out_loc_dev, int32_t out_loc_is_i64,
                                   const int64_t* pos_dev, int64_t pos_axis_stride, int64_t n_rows,
                                   const VaShape* shape, const VaRope* rope, void* stream) {
  int rc = va::check_quant_pool(pool, shape);
  if (rc) return rc;
  if (n_rows < 0) return va_fail(VA_ERR_ARG, "bad shape");
  if (n_rows == 0) return VA_OK;
  if (!k_dev || !v_dev || !out_loc_dev || !rope) return va_fail(VA_ERR_ARG, "null pointer");
  if (!pos_dev && rope->rotary_dim > 0) return va_fail(VA_ERR_ARG, "rotation needs positions");
  va::StoreArgs a{{k_dev, v_dev}, {k_row_stride, v_row_stride}, {(uint8_t*)pool->k_codes_dev, (uint8_t*)pool->v_codes_dev},
                  {pool->k_scales_dev, pool->v_scales_dev}, out_loc_dev, out_loc_is_i64, pos_dev, pos_axis_stride, n_rows,
                  (uint32_t)pool->num_pages * (uint32_t)shape->page_size, shape->num_kv_heads, shape->head_dim,
                  va::page_map(shape->page_size), va::RopeDev{}};
  rc = va::make_rope(rope, shape->head_dim, &a.rope);
  if (rc) return rc;
  VA_DISPATCH_ROWS(shape->dtype, pool->code_type, (va::launch_quant_store<E, C>(a, (hipStream_t)stream)));
  return rc;
}

extern "C" int va_load_kv_q8(const VaQuantPool* pool, const int64_t* slots_dev, int64_t n_rows, void* out_k_dev,
                             void* out_v_dev, int64_t out_row_stride, const VaShape* shape, void* stream) {
  int rc = va::check_quant_pool(pool, shape);
  if (rc) return rc;
  if (n_rows < 0) return va_fail(VA_ERR_ARG, "bad shape");
  if (n_rows == 0 || (!out_k_dev && !out_v_dev)) return VA_OK;
  if (!slots_dev) return va_fail(VA_ERR_ARG, "null pointer");
  if (out_row_stride < (int64_t)shape->num_kv_heads * shape->head_dim) return va_fail(VA_ERR_ARG, "output rows overlap");
  va::LoadArgs a{{(const uint8_t*)pool->k_codes_dev, (const uint8_t*)pool->v_codes_dev}, {pool->k_scales_dev, pool->v_scales_dev},
                 {out_k_dev, out_v_dev}, out_row_stride, slots_dev, n_rows, (uint32_t)pool->num_pages * (uint32_t)shape->page_size,
                 shape->num_kv_heads, shape->head_dim, 0, va::page_map(shape->page_size)};
  VA_DISPATCH_ROWS(shape->dtype, pool->code_type, (va::launch_quant_load<E, C>(a, (hipStream_t)stream)));
  return rc;
}

extern "C" int va_copy_shift_kv_q8(const VaQuantPool* pool, int64_t code_layer_stride, int64_t scale_layer_stride,
                                   int32_t num_layers, const int64_t* src_slots_dev, const int64_t* dst_slots_dev,
                                   int64_t n_tokens, int64_t position_shift, const VaShape* shape, const VaRope* rope,
                                   void* stream) {
  int rc = va::check_quant_pool(pool, shape);
  if (rc) return rc;
  if (n_tokens < 0 || num_layers < 0) return va_fail(VA_ERR_ARG, "negative count");
  if (n_tokens == 0 || num_layers == 0) return VA_OK;
  if (!src_slots_dev || !dst_slots_dev) return va_fail(VA_ERR_ARG, "null pointer");
  if (num_layers > 1 && code_layer_stride % 16) return va_fail(VA_ERR_ARG, "code arrays must start on 16-byte boundaries");
  va::QuantCopyArgs a{{(uint8_t*)pool->k_codes_dev, (uint8_t*)pool->v_codes_dev}, {pool->k_scales_dev, pool->v_scales_dev},
                      code_layer_stride, scale_layer_stride, src_slots_dev, dst_slots_dev, n_tokens, position_shift,
                      (uint32_t)pool->num_pages * (uint32_t)shape->page_size, shape->num_kv_heads,
                      va::page_map(shape->page_size), va::RopeDev{}};
  if (position_shift != 0) {
    rc = va::make_rope(rope, shape->head_dim, &a.rope);
    if (rc) return rc;
  }
  return pool->code_type == VA_CODE_E4M3 ? va::launch_quant_copy<va::E4M3>(a, shape->head_dim, num_layers, (hipStream_t)stream)
                                         : va::launch_quant_copy<va::INT8>(a, shape->head_dim, num_layers, (hipStream_t)stream);
}
