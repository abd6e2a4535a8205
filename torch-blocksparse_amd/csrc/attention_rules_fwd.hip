// Attention with score rules, forward: the kernels of attention_rules_fwd.h and what the calls are checked for.
#include "attention_rules_fwd.h"

namespace bsp {
namespace {

// The range of document numbers in each group of sixteen positions (see RuleArgs)
__global__ void __launch_bounds__(256) k_rules_ranges(const int32_t *docs, int64_t docs_sz, int L, int groups, int Z, int32_t *out) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= (int64_t)Z * groups) return;
  const int z = (int)(at / groups), first = (int)(at % groups) * 16;
  int lo = 0x7fffffff, hi = -1;
  bool none = false;
#pragma unroll
  for (int i = 0; i < 16; i++) {
    const int p = first + i < L ? first + i : L - 1, d = docs[z * docs_sz + p];
    none |= d < 0;
    lo = d < lo ? d : lo;
    hi = d > hi ? d : hi;
  }
  out[2 * at] = none ? -1 : lo;
  out[2 * at + 1] = hi < 0 ? -1 : hi;
}

}  // namespace

int rules_args(const bsp_attention_rules_call *c, RuleArgs &a) {
  if (!c || c->Z <= 0 || c->H <= 0 || c->kv_heads <= 0 || c->H % c->kv_heads || c->length <= 0 || c->length >= (1 << 24) || !c->d_rows) return BSP_ERR_ARG;
  if ((c->dtype != BSP_F16 && c->dtype != BSP_BF16 && c->dtype != BSP_F32) || (c->D != 64 && c->D != 128)) return BSP_ERR_UNSUPPORTED;
  if (c->H / c->kv_heads > 127 || !scores_ok(c->scale, c->softcap)) return BSP_ERR_ARG;
  if ((c->documents != nullptr) != (c->ranges != nullptr) || (c->prefix && !c->causal)) return BSP_ERR_ARG;
  const int64_t lines = c->lines, unit = c->dtype == BSP_F32 ? 4 : 8, size = c->dtype == BSP_F32 ? 4 : 2;
  if (lines < (c->length + 63) / 64 || lines > (1 << 18)) return BSP_ERR_ARG;
  if ((int64_t)c->Z * c->H * lines >= ((int64_t)1 << 25) - 64) return BSP_ERR_UNSUPPORTED;   // (a grid has fewer than 2^32 threads, 128 a line)
  for (int i = 0; i < 24; i++)
    if (c->strides[i] % unit) return BSP_ERR_ARG;
  // the rows of q, k, v and do are fetched by byte offsets of 32 bits from a head's first
  for (int i = 2; i < 24; i += 3)
    if (c->strides[i] != 0 && (c->strides[i] < c->D || c->strides[i] > (((int64_t)1 << 32) - 1) / (size * (c->length + 64)))) return BSP_ERR_ARG;
  a = RuleArgs{};
  a.Z = c->Z; a.H = c->H; a.G = c->H / c->kv_heads; a.L = (int)c->length; a.R = (int)lines;
  a.rows = lines * 64;
  const int64_t *s = c->strides;
  a.q_sz = s[0]; a.q_sh = s[1]; a.q_ld = s[2];
  a.k_sz = s[3]; a.k_sh = s[4]; a.k_ld = s[5];
  a.v_sz = s[6]; a.v_sh = s[7]; a.v_ld = s[8];
  logit_args(a, c->scale, c->softcap);
  a.slopes = c->slopes; a.causal = c->causal; a.prefix = c->prefix;
  a.docs = c->documents; a.docs_sz = c->documents_stride; a.ranges = c->ranges; a.groups = (int)((c->length + 15) / 16);
  a.ref = c->stats; a.o_rest = c->o_rest; a.lut = c->d_rows;
  return BSP_OK;
}

}  // namespace bsp

using namespace bsp;

static inline bool off16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

int bsp::rules_fwd_args(const bsp_attention_rules_call *call, const void *q, const void *k, const void *v, void *o, RuleArgs &a) {
  const int rc = rules_args(call, a);
  if (rc != BSP_OK) return rc;
  const int64_t *s = call->strides;
  if (!q || !k || !v || !o || off16(q) || off16(k) || off16(v) || off16(o) || !s[2] || !s[5] || !s[8] || !s[11]) return BSP_ERR_ARG;
  if (call->stats && call->dtype != BSP_F32 && (!call->o_rest || off16(call->o_rest))) return BSP_ERR_ARG;
  a.q = q; a.k = k; a.v = v; a.o = o;
  a.o_sz = s[9]; a.o_sh = s[10]; a.o_ld = s[11];
  return BSP_OK;
}

void bsp::rules_ranges(const RuleArgs &a, int32_t *ranges, hipStream_t st) {
  if (a.docs) hipLaunchKernelGGL(k_rules_ranges, dim3((unsigned)cdiv((int64_t)a.Z * a.groups, 256)), dim3(256), 0, st, a.docs, a.docs_sz, a.L, a.groups, a.Z, ranges);
}

extern "C" int bsp_attention_rules_fwd(const bsp_attention_rules_call *call, const void *q, const void *k, const void *v, void *o, void *stream) {
  RuleArgs a;
  const int rc = rules_fwd_args(call, q, k, v, o, a);
  if (rc != BSP_OK) return rc;
  const hipStream_t st = as_stream(stream);
  rules_ranges(a, call->ranges, st);
  const int rl = launch_rules_fwd<0>(call->dtype, call->D, a, st);
  if (rl != BSP_OK) return rl;
  BSP_LAUNCH_CHECK();
  return BSP_OK;
}
