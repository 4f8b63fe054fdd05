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
// 1024 / kD tokens a step, kAhead steps are in flight together.  Every lane group keeps a softmax state of its own; they are
// folded by shuffles and through LDS at the end of the chain.
constexpr int kAnyHeads = 4;
constexpr int kAnyThreads = 256;
constexpr int kAnyWaves = kAnyThreads / kWave;
constexpr int kAnyAhead = 2;

template <int kD, typename C>
__global__ __launch_bounds__(kAnyThreads) void attn_quant_any_kernel(QuantAttnArgs qa, int dtype) {
  const AttnArgs& a = qa.a;
  constexpr int kVec = 16;
  constexpr int kLPT = kD / kVec;  // lanes per token
  constexpr int kTPW = kWave / kLPT;

  __shared__ float q_s[kAnyHeads][kD];
  __shared__ float acc_s[kAnyWaves][kAnyHeads][kD];
  __shared__ float ml_s[kAnyWaves][kAnyHeads][2];

  const ItemHead where = item_and_head(blockIdx.x, a.num_kv_heads);
  const int32_t* item = a.items + (long long)where.item * VA_ITEM_WORDS;
  const int hk = where.head, G = a.num_q_heads / a.num_kv_heads;
  const int n_q = item[VA_I_N_Q];
  if (n_q == 0) return;  // padding item: keeps the launch order aligned with the die round-robin
  const int part_base = item[VA_I_PART_BASE];
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const int li = lane % kLPT, lg = lane / kLPT;
  const uint8_t* kp = (const uint8_t*)a.k_pool;
  const uint8_t* vp = (const uint8_t*)a.v_pool;

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
      for (int lk = 0; lk < item[VA_I_N_LINKS]; ++lk) {
        const int32_t* link = a.links + (long long)(item[VA_I_LINK_BEGIN] + lk) * VA_LINK_WORDS;
        const int lflags = link[VA_L_FLAGS];
        const int subrow = (lflags & VA_LINK_INDIRECT) ? a.qrefs[link[VA_L_QREF] + iq] : link[VA_L_QREF] + iq;
        const long long src_row = a.sub_worker[subrow];
        out_row = src_row;
        const Pos3 p = load_pos(a.sub_loc, a.sub_loc_axis_stride, subrow);

        // this row's query for the link, rotated in fp32
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

        const int t_end = min(link[VA_L_TOK_END], link[VA_L_CAUSAL_BASE] + iq + 1);
        const int kv_begin = link[VA_L_KV_BEGIN];
        const bool slots = lflags & VA_LINK_SLOTS;
        for (int t0 = link[VA_L_TOK_BEGIN] + wave * kTPW; t0 < t_end; t0 += kAnyAhead * kAnyWaves * kTPW) {
          bool live[kAnyAhead];
          uint4 kraw[kAnyAhead], vraw[kAnyAhead];
          float ks[kAnyAhead], vs[kAnyAhead];
#pragma unroll
          for (int u = 0; u < kAnyAhead; ++u) {
            const int t = t0 + u * kAnyWaves * kTPW + lg;
            live[u] = t < t_end;
            const long long row = quant_token_row(qa, kv_begin, live[u] ? t : t_end - 1, slots, hk);
            kraw[u] = *(const uint4*)(kp + row * kD + li * kVec);
            vraw[u] = *(const uint4*)(vp + row * kD + li * kVec);
            ks[u] = scale_value(qa.k_scales[row]);
            vs[u] = scale_value(qa.v_scales[row]);
          }
#pragma unroll
          for (int u = 0; u < kAnyAhead; ++u) {
            if (t0 + u * kAnyWaves * kTPW >= t_end) break;  // (wave-uniform: the step lies past the range)
            float kf[kVec], vf[kVec], sc[kAnyHeads];
            C::unpack4(kraw[u].x, kf), C::unpack4(kraw[u].y, kf + 4), C::unpack4(kraw[u].z, kf + 8), C::unpack4(kraw[u].w, kf + 12);
            C::unpack4(vraw[u].x, vf), C::unpack4(vraw[u].y, vf + 4), C::unpack4(vraw[u].z, vf + 8), C::unpack4(vraw[u].w, vf + 12);
#pragma unroll
            for (int g = 0; g < kAnyHeads; ++g) {
              float d = 0.f;
#pragma unroll
              for (int e = 0; e < kVec; ++e) d = fmaf(qr[g][e], kf[e], d);
              d = group_sum<kLPT>(d);
              sc[g] = live[u] ? d * (ks[u] * a.scale_log2) : -INFINITY;
            }
#pragma unroll
            for (int g = 0; g < kAnyHeads; ++g) {
              const float m_new = fmaxf(m[g], sc[g]);
              const float alpha = exp2f(m[g] - m_new);
              const float pr = exp2f(sc[g] - m_new), weight = live[u] ? pr * vs[u] : 0.f;
              m[g] = m_new;
              l[g] = l[g] * alpha + pr;
#pragma unroll
              for (int e = 0; e < kVec; ++e) acc[g][e] = fmaf(weight, vf[e], acc[g][e] * alpha);
            }
          }
        }
      }

      // the lane groups of the wave
#pragma unroll
      for (int off = kLPT; off < kWave; off <<= 1) {
#pragma unroll
        for (int g = 0; g < kAnyHeads; ++g) {
          const float m_o = __shfl_xor(m[g], off, kWave), l_o = __shfl_xor(l[g], off, kWave);
          const float m_new = fmaxf(m[g], m_o);
          const float sa = exp2f(m[g] - m_new), sb = exp2f(m_o - m_new);
          l[g] = l[g] * sa + l_o * sb;
#pragma unroll
          for (int e = 0; e < kVec; ++e) acc[g][e] = acc[g][e] * sa + __shfl_xor(acc[g][e], off, kWave) * sb;
          m[g] = m_new;
        }
      }
      __syncthreads();
      if (lg == 0) {
#pragma unroll
        for (int g = 0; g < kAnyHeads; ++g) {
#pragma unroll
          for (int e = 0; e < kVec; ++e) acc_s[wave][g][li * kVec + e] = acc[g][e];
          if (li == 0) {
            ml_s[wave][g][0] = m[g];
            ml_s[wave][g][1] = l[g];
          }
        }
      }
      __syncthreads();
      // the waves
      for (int e = threadIdx.x; e < kAnyHeads * kD; e += kAnyThreads) {
        const int g = e / kD, d = e - g * kD;
        if (hb + g >= G) continue;
        float mm = kNegBig;
#pragma unroll
        for (int w = 0; w < kAnyWaves; ++w) mm = fmaxf(mm, ml_s[w][g][0]);
        float ll = 0.f, av = 0.f;
#pragma unroll
        for (int w = 0; w < kAnyWaves; ++w) {
          const float sw = exp2f(ml_s[w][g][0] - mm);
          ll += ml_s[w][g][1] * sw;
          av += acc_s[w][g][d] * sw;
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

extern "C" int va_attention_q8(const void* q_dev, int64_t q_row_stride, const VaQuantPool* pool, const int32_t* plan_dev,
                               const int32_t* plan_header_host, const int32_t* kv_indices_dev,
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
      rc = va::launch_quant_mfma(qa, shape->dtype, pool->code_type, n_items, h[VA_H_Q_TILE], s);
    else
      rc = pool->code_type == VA_CODE_E4M3 ? va::launch_quant_any<va::E4M3>(qa, shape->dtype, n_items, s)
                                           : va::launch_quant_any<va::INT8>(qa, shape->dtype, n_items, s);
    if (rc) return rc;
  }
  if (h[VA_H_N_PARTIALS] > 0 || h[VA_H_N_EMPTY_ROWS] > 0)
    rc = va::launch_merge_typed(m, shape->dtype, h[VA_H_N_ROWS], h[VA_H_MERGE_WAVES], s);
  return rc;
}
