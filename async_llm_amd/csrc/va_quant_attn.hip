// View attention over a quantised pool: the entry point and the vector-ALU kernel.
//
// The plans, the partial states and their merge are those of the 16-bit path; only what a token's K and V rows are differs:
//   score = (q . code_k) * 2^e_k / sqrt(d),   out += weight * 2^e_v * code_v.
// The scales stay out of the products over dims (codes are exact in fp32 and bf16 alike).
#include <hip/hip_runtime.h>

#include "va_internal.h"
#include "va_launch.h"
#include "va_quant.h"
#include "va_quant_attn.h"

namespace va {

// Any activation type, head_dim a power of two from 16 to 256, any number of q heads per kv head: float32 activations and
// what the matrix-core kernel rejects.  One workgroup of four waves per (work item, kv head), tile rows one after another,
// four q heads a pass.  A token's K (and V) row is sixteen codes for each of kD / 16 adjacent lanes, a wave takes
// 1024 / kD tokens a step and two steps together; the next two are requested before their products, the first ones before the
// queries are rotated.  Every lane group keeps maxima and sums of its own; the workgroup's maximum is found at the end of the
// chain, and what is left are plain sums.
//
// Small steps are a chain of trips (item, link, page, codes; row, query, turns) and a fold, so what counts is their number:
// one row, 2 kv heads of 128 dims, 1900 tokens 8.1 us (12.7 where codes were requested behind the query and lane groups joined
// pair by pair, each with its rescaling, by shuffles); eight rows of 3000 tokens, 4 heads of 256 dims 26 (32 for the step), 32 rows
// of 12000, 8 heads of 128 dims 320 (399): the vector ALU's products.
constexpr int kAnyHeads = 4;
constexpr int kAnyThreads = 256;
constexpr int kAnyWaves = kAnyThreads / kWave;
constexpr int kAnyAhead = 2;

// Lane exchanges on the vector ALU (a shuffle is a trip through LDS).
template <int kCtrl>
__device__ __forceinline__ float lane_of_row(float x) {
  return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), kCtrl, 0xf, 0xf, true));
}
// Sum over kLanes neighbouring lanes, in all of them: neighbours, pairs, then mirrored halves of 8 and of 16.
template <int kLanes>
__device__ __forceinline__ float neighbour_sum(float x) {
  if constexpr (kLanes >= 2) x += lane_of_row<0xB1>(x);
  if constexpr (kLanes >= 4) x += lane_of_row<0x4E>(x);
  if constexpr (kLanes >= 8) x += lane_of_row<0x141>(x);
  if constexpr (kLanes >= 16) x += lane_of_row<0x140>(x);
  return x;
}
// f over the lanes of a row of 16 that lie a multiple of kStep apart, in all of them: rotations by kStep, twice it, ...
template <int kStep, typename F>
__device__ __forceinline__ float over_row(float x, F f) {
  if constexpr (kStep <= 1) x = f(x, lane_of_row<0x121>(x));
  if constexpr (kStep <= 2) x = f(x, lane_of_row<0x122>(x));
  if constexpr (kStep <= 4) x = f(x, lane_of_row<0x124>(x));
  if constexpr (kStep <= 8) x = f(x, lane_of_row<0x128>(x));
  return x;
}
template <typename F>
__device__ __forceinline__ float over_rows16(float x, F f) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = f(__uint_as_float(r[0]), __uint_as_float(r[1]));
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return f(__uint_as_float(s[0]), __uint_as_float(s[1]));
}

template <int kD, typename C>
__global__ __launch_bounds__(kAnyThreads) void attn_quant_any_kernel(QuantAttnArgs qa, int dtype) {
  const AttnArgs& a = qa.a;
  using Words = const __attribute__((address_space(4))) int32_t*;  // read only while a launch runs
  using Longs = const __attribute__((address_space(4))) int64_t*;
  constexpr int kVec = 16;
  constexpr int kLPT = kD / kVec;  // lanes per token
  constexpr int kTPW = kWave / kLPT;
  static_assert(kAnyHeads == kWave / 16, "a head for each row of 16 lanes");

  __shared__ float q_s[kAnyHeads][kD];
  __shared__ __align__(16) float acc_s[kAnyWaves][kAnyHeads][kD];
  __shared__ float m_s[kAnyWaves][kAnyHeads], l_s[kAnyWaves][kAnyHeads];

  const ItemHead where = item_and_head(blockIdx.x, a.num_kv_heads);
  const Words item = (Words)a.items + (long long)where.item * VA_ITEM_WORDS;
  const int hk = where.head, G = a.num_q_heads / a.num_kv_heads;
  const int n_q = item[VA_I_N_Q];
  if (n_q == 0) return;  // padding item: keeps the launch order aligned with the die round-robin
  const int part_base = item[VA_I_PART_BASE], link_begin = item[VA_I_LINK_BEGIN], n_links = item[VA_I_N_LINKS];
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const int li = lane % kLPT, lg = lane / kLPT;
  const uint8_t* kp = (const uint8_t*)a.k_pool;
  const uint8_t* vp = (const uint8_t*)a.v_pool;
  const auto larger = [](float x, float y) { return fmaxf(x, y); };
  const auto sum = [](float x, float y) { return x + y; };

  for (int iq = 0; iq < n_q; ++iq) {
    long long out_row = -1;
    for (int hb = 0; hb < G; hb += kAnyHeads) {
      float m[kAnyHeads], l[kAnyHeads], acc[kAnyHeads][kVec];
#pragma unroll
      for (int g = 0; g < kAnyHeads; ++g) {
        m[g] = kNegBig;
        l[g] = 0.f;
#pragma unroll
        for (int e = 0; e < kVec; ++e) acc[g][e] = 0.f;
      }
      for (int lk = 0; lk < n_links; ++lk) {
        const Words link = (Words)a.links + (long long)(link_begin + lk) * VA_LINK_WORDS;
        const int lflags = link[VA_L_FLAGS], qref = link[VA_L_QREF], kv_begin = link[VA_L_KV_BEGIN];
        const int t_end = min(link[VA_L_TOK_END], link[VA_L_CAUSAL_BASE] + iq + 1);
        const bool slots = lflags & VA_LINK_SLOTS;
        int t0 = link[VA_L_TOK_BEGIN] + wave * kTPW;
        constexpr int kStep = kAnyAhead * kAnyWaves * kTPW;
        uint4 kraw[kAnyAhead], vraw[kAnyAhead];
        uint8_t ks[kAnyAhead], vs[kAnyAhead];
        // (past the range the last token's rows, whose products are masked)
        const auto request = [&](int t0) __attribute__((always_inline)) {
#pragma unroll
          for (int u = 0; u < kAnyAhead; ++u) {
            const long long row = quant_token_row(qa, kv_begin, min(t0 + u * kAnyWaves * kTPW + lg, t_end - 1), slots, hk);
            kraw[u] = *(const uint4*)(kp + row * kD + li * kVec);
            vraw[u] = *(const uint4*)(vp + row * kD + li * kVec);
            ks[u] = qa.k_scales[row];
            vs[u] = qa.v_scales[row];
          }
        };
        if (t0 < t_end) request(t0);

        // this row's query for the link, rotated in fp32
        const int subrow = (lflags & VA_LINK_INDIRECT) ? ((Words)a.qrefs)[qref + iq] : qref + iq;
        const long long src_row = ((Longs)a.sub_worker)[subrow];
        out_row = src_row;
        const Pos3 p = load_pos(a.sub_loc, a.sub_loc_axis_stride, subrow);
        __syncthreads();
        for (int e = threadIdx.x; e < kAnyHeads * kD; e += kAnyThreads) {
          const int g = e / kD, d = e - g * kD;
          float val = 0.f;
          if (hb + g < G) {
            const long long at = src_row * a.q_row_stride + (long long)(hk * G + hb + g) * kD;
            val = activation(a.q, at + d, dtype);
            if (d < a.rope.rotary_dim) {
              const bool first = d < a.rope.half;
              const float other = activation(a.q, at + (first ? d + a.rope.half : d - a.rope.half), dtype);
              float c, s;
              rope_cos_sin(a.rope, p, first ? d : d - a.rope.half, c, s);
              val = first ? mul_rounded(c, val) - mul_rounded(s, other) : mul_rounded(c, val) + mul_rounded(s, other);
            }
          }
          q_s[g][d] = val;
        }
        __syncthreads();
        float qr[kAnyHeads][kVec];
#pragma unroll
        for (int g = 0; g < kAnyHeads; ++g)
#pragma unroll
          for (int e = 0; e < kVec; ++e) qr[g][e] = q_s[g][li * kVec + e];

        for (; t0 < t_end; t0 += kStep) {
          float sc[kAnyAhead][kAnyHeads], vscale[kAnyAhead];
          uint4 v[kAnyAhead];
          bool live[kAnyAhead];
#pragma unroll
          for (int u = 0; u < kAnyAhead; ++u) {
            live[u] = t0 + u * kAnyWaves * kTPW + lg < t_end;
            float kf[kVec];
            C::unpack4(kraw[u].x, kf), C::unpack4(kraw[u].y, kf + 4), C::unpack4(kraw[u].z, kf + 8), C::unpack4(kraw[u].w, kf + 12);
            const float kscale = scale_value(ks[u]) * a.scale_log2;
#pragma unroll
            for (int g = 0; g < kAnyHeads; ++g) {
              float d = 0.f;
#pragma unroll
              for (int e = 0; e < kVec; ++e) d = fmaf(qr[g][e], kf[e], d);
              sc[u][g] = live[u] ? neighbour_sum<kLPT>(d) * kscale : -INFINITY;
            }
            v[u] = vraw[u];
            vscale[u] = live[u] ? scale_value(vs[u]) : 0.f;  // (a token that the row does not see may have any scale)
          }
          if (t0 + kStep < t_end) request(t0 + kStep);
          float pr[kAnyAhead][kAnyHeads];
#pragma unroll
          for (int g = 0; g < kAnyHeads; ++g) {
            const float m_new = fmaxf(m[g], fmaxf(sc[0][g], sc[1][g]));
            const float alpha = exp2f(m[g] - m_new);
            m[g] = m_new;
#pragma unroll
            for (int u = 0; u < kAnyAhead; ++u) pr[u][g] = exp2f(sc[u][g] - m_new);
            l[g] = fmaf(l[g], alpha, pr[0][g] + pr[1][g]);
#pragma unroll
            for (int e = 0; e < kVec; ++e) acc[g][e] *= alpha;
          }
#pragma unroll
          for (int u = 0; u < kAnyAhead; ++u) {
            float vf[kVec];
            C::unpack4(v[u].x, vf), C::unpack4(v[u].y, vf + 4), C::unpack4(v[u].z, vf + 8), C::unpack4(v[u].w, vf + 12);
#pragma unroll
            for (int g = 0; g < kAnyHeads; ++g) {
              const float weight = pr[u][g] * vscale[u];
#pragma unroll
              for (int e = 0; e < kVec; ++e) acc[g][e] = fmaf(weight, vf[e], acc[g][e]);
            }
          }
        }
      }

      // One maximum for the workgroup, then plain sums: over the lane groups of a row of 16, then over the rows, whose
      // swaps leave row r with head r.
#pragma unroll
      for (int g = 0; g < kAnyHeads; ++g) {
        const float top = over_rows16(over_row<kLPT>(m[g], larger), larger);
        if (lane == 0) m_s[wave][g] = top;
      }
      __syncthreads();
      float top[kAnyHeads];
#pragma unroll
      for (int g = 0; g < kAnyHeads; ++g) {
        top[g] = m_s[0][g];
#pragma unroll
        for (int w = 1; w < kAnyWaves; ++w) top[g] = fmaxf(top[g], m_s[w][g]);
        const float s = exp2f(m[g] - top[g]);
        const float ll = over_rows16(over_row<kLPT>(l[g] * s, sum), sum);
        if (lane == 0) l_s[wave][g] = ll;
#pragma unroll
        for (int e = 0; e < kVec; ++e) acc[g][e] *= s;
      }
      float mine[kVec];
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        float pair[2];
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(acc[g][e]), __float_as_uint(acc[g + 2][e]), false, false);
          pair[g] = __uint_as_float(r[0]) + __uint_as_float(r[1]);  // low half: head g, high half: g + 2
        }
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(pair[0]), __float_as_uint(pair[1]), false, false);
        mine[e] = over_row<kLPT>(__uint_as_float(r[0]) + __uint_as_float(r[1]), sum);
      }
      if (lane % 16 < kLPT) {
#pragma unroll
        for (int e = 0; e < kVec; e += 4)
          *(float4*)&acc_s[wave][lane / 16][li * kVec + e] = make_float4(mine[e], mine[e + 1], mine[e + 2], mine[e + 3]);
      }
      __syncthreads();
      // the waves
      for (int e = threadIdx.x; e < kAnyHeads * kD; e += kAnyThreads) {
        const int g = e / kD, d = e - g * kD;
        if (hb + g >= G) continue;
        float ll = 0.f, av = 0.f, mm = m_s[0][g];
#pragma unroll
        for (int w = 0; w < kAnyWaves; ++w) {
          mm = fmaxf(mm, m_s[w][g]);
          ll += l_s[w][g];
          av += acc_s[w][g][d];
        }
        const int hq = hk * G + hb + g;
        if (part_base < 0) {
          store_activation(a.out, (out_row * a.num_q_heads + hq) * (long long)kD + d, normalised(av, ll), dtype);
          if (d == 0 && a.lse) a.lse[out_row * a.num_q_heads + hq] = log_sum(mm, ll, a.lse_base2);
        } else {
          const long long slot = (long long)(part_base + iq) * a.num_q_heads + hq;
          a.part_acc[slot * kD + d] = av;
          if (d == 0) {
            a.part_ml[slot * 2 + 0] = mm;
            a.part_ml[slot * 2 + 1] = ll;
          }
        }
      }
    }
  }
}

template <typename C>
static int launch_quant_any(const QuantAttnArgs& qa, int dtype, int n_items, hipStream_t stream) {
  const dim3 grid((unsigned)n_items * (unsigned)qa.a.num_kv_heads), block(kAnyThreads);
  switch (qa.a.head_dim) {
#define VA_CASE(D) \
  case D:          \
    hipLaunchKernelGGL((attn_quant_any_kernel<D, C>), grid, block, 0, stream, qa, dtype); \
    break;
    VA_CASE(16) VA_CASE(32) VA_CASE(64) VA_CASE(128) VA_CASE(256)
#undef VA_CASE
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? VA_OK : va_fail(VA_ERR_HIP, "attention launch: %s", hipGetErrorString(e));
}

}  // namespace va

static int attention_q8(const int32_t* only_if, const void* q_dev, int64_t q_row_stride, const VaQuantPool* pool,
                        const int32_t* plan_dev, const int32_t* plan_header_host, const int32_t* kv_indices_dev,
                        const int64_t* sub_worker_dev, const int64_t* sub_loc_dev, int64_t sub_loc_axis_stride,
                        void* out_dev, float* lse_dev, int32_t lse_base2, void* workspace_dev,
                        int64_t workspace_bytes, const VaShape* shape, const VaRope* rope, void* stream) {
  if (!shape || !plan_header_host || !plan_dev) return va_fail(VA_ERR_ARG, "null plan or shape");
  int rc = va::check_quant_pool(pool, shape);
  if (rc) return rc;
  if (shape->dtype != VA_F32 && shape->dtype != VA_F16 && shape->dtype != VA_BF16)
    return va_fail(VA_ERR_ARG, "unknown dtype %d", (int)shape->dtype);
  const int32_t* h = plan_header_host;
  if (h[VA_H_MAGIC] != VA_PLAN_MAGIC) return va_fail(VA_ERR_ARG, "plan header has no magic word");
  if (h[VA_H_N_ROWS] == 0) return VA_OK;
  if (h[VA_H_N_WIDE] != 0) return va_fail(VA_ERR_ARG, "a plan over a quantised pool has no wide items (wide_tile < 0)");
  if (only_if && (h[VA_H_N_PARTIALS] > 0 || h[VA_H_N_EMPTY_ROWS] > 0))
    return va_fail(VA_ERR_ARG, "a launch under a condition takes plans without partial states and empty rows");
  if (only_if && h[VA_H_KERNEL] != VA_KERNEL_MFMA) return va_fail(VA_ERR_ARG, "a launch under a condition takes matrix-core plans");
  va::QuantAttnArgs qa;
  va::MergeArgs m;
  rc = va::plan_arguments(q_dev, q_row_stride, pool->k_codes_dev, pool->v_codes_dev, 0, plan_dev, h, kv_indices_dev,
                          sub_worker_dev, sub_loc_dev, sub_loc_axis_stride, out_dev, lse_dev, lse_base2, workspace_dev,
                          workspace_bytes, shape, rope, &qa.a, &m);
  if (rc) return rc;
  qa.k_scales = pool->k_scales_dev;
  qa.v_scales = pool->v_scales_dev;
  qa.pages = va::page_map(shape->page_size);
  m.keep_nan = 1;
  hipStream_t s = (hipStream_t)stream;
  const int n_items = h[VA_H_N_ITEMS];
  if (n_items > 0) {
    if (h[VA_H_KERNEL] == VA_KERNEL_MFMA)
      rc = va::launch_quant_mfma(qa, only_if, shape->dtype, pool->code_type, n_items, h[VA_H_Q_TILE], s);
    else
      rc = pool->code_type == VA_CODE_E4M3 ? va::launch_quant_any<va::E4M3>(qa, shape->dtype, n_items, s)
                                           : va::launch_quant_any<va::INT8>(qa, shape->dtype, n_items, s);
    if (rc) return rc;
  }
  if (h[VA_H_N_PARTIALS] > 0 || h[VA_H_N_EMPTY_ROWS] > 0)
    rc = va::launch_merge_typed(m, shape->dtype, h[VA_H_N_ROWS], h[VA_H_MERGE_WAVES], s);
  return rc;
}

extern "C" int va_attention_q8(const void* q_dev, int64_t q_row_stride, const VaQuantPool* pool, const int32_t* plan_dev,
                               const int32_t* plan_header_host, const int32_t* kv_indices_dev,
                               const int64_t* sub_worker_dev, const int64_t* sub_loc_dev, int64_t sub_loc_axis_stride,
                               void* out_dev, float* lse_dev, int32_t lse_base2, void* workspace_dev,
                               int64_t workspace_bytes, const VaShape* shape, const VaRope* rope, void* stream) {
  return attention_q8(nullptr, q_dev, q_row_stride, pool, plan_dev, plan_header_host, kv_indices_dev, sub_worker_dev, sub_loc_dev,
                      sub_loc_axis_stride, out_dev, lse_dev, lse_base2, workspace_dev, workspace_bytes, shape, rope, stream);
}

extern "C" int va_attention_if_q8(const int32_t* condition_dev, const void* q_dev, int64_t q_row_stride, const VaQuantPool* pool,
                                  const int32_t* plan_dev, const int32_t* plan_header_host, const int32_t* kv_indices_dev,
                                  const int64_t* sub_worker_dev, const int64_t* sub_loc_dev, int64_t sub_loc_axis_stride,
                                  void* out_dev, float* lse_dev, int32_t lse_base2, const VaShape* shape, const VaRope* rope,
                                  void* stream) {
  if (!condition_dev) return va_fail(VA_ERR_ARG, "null condition");
  return attention_q8(condition_dev, q_dev, q_row_stride, pool, plan_dev, plan_header_host, kv_indices_dev, sub_worker_dev,
                      sub_loc_dev, sub_loc_axis_stride, out_dev, lse_dev, lse_base2, nullptr, 0, shape, rope, stream);
}
