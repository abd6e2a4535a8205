// Attention with score rules, backward: the kernels of attention_rules_bwd.h and what the calls are checked for.
#include "attention_rules_bwd.h"

using namespace bsp;

static inline bool off16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

int bsp::rules_bwd_args(const bsp_attention_rules_call *call, const void *d_o, const void *q, const void *k, const void *v, const void *o, void *dq, void *dk, void *dv, float *neg_delta,
                        const int32_t *d_items, int n_items, float *partial, int n_slots, const int32_t *d_split, int n_split, RuleArgs &a) {
  const int rc = rules_args(call, a);
  if (rc != BSP_OK) return rc;
  const int64_t *s = call->strides;
  if (!d_o || !q || !k || !v || !o || !dq || !neg_delta || !call->stats || (call->dtype != BSP_F32 && (!call->o_rest || off16(call->o_rest))) || (dk != nullptr) != (dv != nullptr)) return BSP_ERR_ARG;
  const void *ptrs[] = {d_o, q, k, v, o, dq, dk, dv, partial};
  for (const void *p : ptrs)
    if (off16(p)) return BSP_ERR_ARG;
  for (int i = 2; i < 24; i += 3)
    if (!s[i] && (dk || i < 18)) return BSP_ERR_ARG;
  if (dk && (!d_items || n_items <= 0 || n_slots < 0 || n_split < 0 || (n_slots > 0) != (n_split > 0) || (n_slots > 0 && (!partial || !d_split)))) return BSP_ERR_ARG;
  if (dk && ((int64_t)a.Z * call->kv_heads * n_items >= ((int64_t)1 << 25) - 64 || (int64_t)a.Z * n_split * (32 * call->D) >= ((int64_t)1 << 32) || a.rows * 2 * a.G >= ((int64_t)1 << 30))) return BSP_ERR_UNSUPPORTED;
  a.q = q; a.k = k; a.v = v; a.d_o = d_o; a.o_in = o; a.delta = neg_delta;
  a.oin_sz = s[9]; a.oin_sh = s[10]; a.oin_ld = s[11];
  a.do_sz = s[12]; a.do_sh = s[13]; a.do_ld = s[14];
  a.o = dq; a.o_sz = s[15]; a.o_sh = s[16]; a.o_ld = s[17];
  return BSP_OK;
}

void bsp::rules_bwd_columns(const bsp_attention_rules_call *call, void *dk, void *dv, const int32_t *d_items, int n_items, float *partial, int n_slots, const int32_t *d_split, int n_split, RuleArgs &a) {
  const int64_t *s = call->strides;
  a.o = dk; a.o_sz = s[18]; a.o_sh = s[19]; a.o_ld = s[20];
  a.o2 = dv; a.o2_sz = s[21]; a.o2_sh = s[22]; a.o2_ld = s[23];
  a.lut = d_items; a.R = n_items;
  a.partial = partial; a.n_slots = n_slots; a.split_lut = d_split; a.n_split = n_split;
}

extern "C" int bsp_attention_rules_bwd(const bsp_attention_rules_call *call, const void *d_o, const void *q, const void *k, const void *v, const void *o,
                                       void *dq, void *dk, void *dv, float *neg_delta, const int32_t *d_items, int n_items, float *partial, int n_slots,
                                       const int32_t *d_split, int n_split, void *stream) {
  RuleArgs a;
  const int rc = rules_bwd_args(call, d_o, q, k, v, o, dq, dk, dv, neg_delta, d_items, n_items, partial, n_slots, d_split, n_split, a);
  if (rc != BSP_OK) return rc;
  const hipStream_t st = as_stream(stream);
  int rl = launch_rules_bwd<0>(call->dtype, call->D, a, false, st);
  if (rl != BSP_OK) return rl;
  if (dk) {
    rules_bwd_columns(call, dk, dv, d_items, n_items, partial, n_slots, d_split, n_split, a);
    rl = launch_rules_bwd<0>(call->dtype, call->D, a, true, st);
    if (rl != BSP_OK) return rl;
  }
  BSP_LAUNCH_CHECK();
  return BSP_OK;
}
