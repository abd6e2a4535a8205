// Attention with score rules whose keys have a part that all heads share (the expanded form of latent attention), forward: logits of scale * (q . k + qx . kx), qx
// [Z, H, L, 64] and kx [Z, L, 64], by the kernels of attention_rules_fwd.h: the part is 64 elements more of a key in the ring and two products more of a tile's scores.  Measured: bf16, causal,
// 16 heads x 8192 x (128 + 64): 505 us, 680 TFLOP/s of what is visible (vector operations 35 % of the cycles, matrix units 41 %); 2 x 16 x 4001 in five documents 135 us (27 %, 21 %: the longest
// document's lines).
#include "attention_rules_fwd.h"

namespace bsp {

int shared_args(const bsp_attention_rules_call *call, const bsp_attention_shared_part *part, bool backward, RuleArgs &a) {
  if (!part || !part->q || !part->k || (backward && !part->dq)) return BSP_ERR_ARG;
  const void *ptrs[] = {part->q, part->k, part->dq, part->dk, part->dk_heads};
  for (const void *p : ptrs)
    if (reinterpret_cast<uintptr_t>(p) & 15) return BSP_ERR_ARG;
  const int64_t unit = call->dtype == BSP_F32 ? 4 : 8, size = call->dtype == BSP_F32 ? 4 : 2, *s = part->strides;
  for (int i = 0; i < 10; i++)
    if (s[i] % unit) return BSP_ERR_ARG;
  // rows are fetched by byte offsets of 32 bits from a head's first
  const int rows[] = {2, 4, 7, 9};
  for (int i = 0; i < (backward ? part->dk ? 4 : 3 : 2); i++)
    if (s[rows[i]] < kShared || s[rows[i]] > (((int64_t)1 << 32) - 1) / (size * (call->length + 64))) return BSP_ERR_ARG;
  a.qx = part->q; a.qx_sz = s[0]; a.qx_sh = s[1]; a.qx_ld = s[2];
  a.kx = part->k; a.kx_sz = s[3]; a.kx_ld = s[4];
  a.ox = part->dq; a.ox_sz = s[5]; a.ox_sh = s[6]; a.ox_ld = s[7];
  a.kx_heads = part->dk_heads;
  return BSP_OK;
}

}  // namespace bsp

using namespace bsp;

extern "C" int bsp_attention_shared_fwd(const bsp_attention_rules_call *call, const bsp_attention_shared_part *part, const void *q, const void *k, const void *v, void *o, void *stream) {
  RuleArgs a;
  int rc = rules_fwd_args(call, q, k, v, o, a);
  if (rc != BSP_OK) return rc;
  rc = shared_args(call, part, false, a);
  if (rc != BSP_OK) return rc;
  const hipStream_t st = as_stream(stream);
  rules_ranges(a, call->ranges, st);
  rc = launch_rules_fwd<kShared>(call->dtype, call->D, a, st);
  if (rc != BSP_OK) return rc;
  BSP_LAUNCH_CHECK();
  return BSP_OK;
}
