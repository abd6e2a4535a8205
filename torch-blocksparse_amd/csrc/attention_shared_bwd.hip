// Attention with score rules whose keys have a part that all heads share, backward (attention_rules_bwd.h), and the sum of that part's gradient over the key heads.
// Measured: bf16 2 x 16 x 4001 x (128 + 64), causal, five documents: rows 201 us (vector operations 23 % of the cycles, matrix units 23 %), columns 252 (23 %, 25 %), that sum 6 (of 32 MB); one
// wavefront a SIMD, whose products wait for each other.  Two a SIMD spill 90 to 250 bytes a lane in the rows of 128 elements.
#include "attention_rules_bwd.h"

namespace bsp {
namespace {

// dkx[z][l] = sum over the key heads of kx_heads[z][head][l], in their order; four elements a thread.  Bound by reading the heads' once, 256 bytes a position.
template <typename T> __global__ void __launch_bounds__(256) k_shared_sum(const float *heads, int kv_heads, int L, T *to, int64_t to_sz, int64_t to_ld) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, in = (int64_t)L * (kShared / 4);
  const int z = (int)blockIdx.y, e = (int)(id % (kShared / 4)) * 4;
  if (id >= in) return;
  const float *from = heads + (int64_t)z * kv_heads * L * kShared + 4 * id;
  f32x4 sum = *reinterpret_cast<const f32x4 *>(from);
#pragma unroll 4
  for (int h = 1; h < kv_heads; h++) {
    const f32x4 v = *reinterpret_cast<const f32x4 *>(from + (int64_t)h * L * kShared);
#pragma unroll
    for (int i = 0; i < 4; i++) sum[i] += v[i];
  }
  T *dst = to + z * to_sz + id / (kShared / 4) * to_ld + e;
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<f32x4 *>(dst) = sum;
  } else {
    union { u32x2 raw; T e[4]; } pk;
#pragma unroll
    for (int i = 0; i < 4; i++) pk.e[i] = from_float<T>(sum[i]);
    *reinterpret_cast<u32x2 *>(dst) = pk.raw;
  }
}
template <typename T> void shared_sum(const bsp_attention_rules_call *call, const bsp_attention_shared_part *part, hipStream_t st) {
  const int64_t *s = part->strides;
  hipLaunchKernelGGL(k_shared_sum<T>, dim3((unsigned)cdiv(call->length * (kShared / 4), 256), (unsigned)call->Z), dim3(256), 0, st, part->dk_heads, call->kv_heads, (int)call->length,
                     reinterpret_cast<T *>(part->dk), s[8], s[9]);
}

}  // namespace
}  // namespace bsp

using namespace bsp;

extern "C" int bsp_attention_shared_bwd(const bsp_attention_rules_call *call, const bsp_attention_shared_part *part, const void *d_o, const void *q, const void *k, const void *v, const void *o,
                                        void *dq, void *dk, void *dv, float *neg_delta, const int32_t *d_items, int n_items, float *partial, int n_slots, const int32_t *d_split,
                                        int n_split, void *stream) {
  RuleArgs a;
  int rc = rules_bwd_args(call, d_o, q, k, v, o, dq, dk, dv, neg_delta, d_items, n_items, partial, n_slots, d_split, n_split, a);
  if (rc != BSP_OK) return rc;
  rc = shared_args(call, part, true, a);
  if (rc != BSP_OK) return rc;
  if ((dk != nullptr) != (part->dk != nullptr) || (dk && !part->dk_heads)) return BSP_ERR_ARG;
  if (dk && (call->Z > 65535 || (int64_t)a.Z * n_split * (16 * (2 * call->D + kShared)) >= ((int64_t)1 << 32))) return BSP_ERR_UNSUPPORTED;
  const hipStream_t st = as_stream(stream);
  rc = launch_rules_bwd<kShared>(call->dtype, call->D, a, false, st);
  if (rc != BSP_OK) return rc;
  if (dk) {
    rules_bwd_columns(call, dk, dv, d_items, n_items, partial, n_slots, d_split, n_split, a);
    rc = launch_rules_bwd<kShared>(call->dtype, call->D, a, true, st);
    if (rc != BSP_OK) return rc;
    if (call->dtype == BSP_F16) shared_sum<f16>(call, part, st);
    else if (call->dtype == BSP_BF16) shared_sum<bf16>(call, part, st);
    else shared_sum<float>(call, part, st);
  }
  BSP_LAUNCH_CHECK();
  return BSP_OK;
}
