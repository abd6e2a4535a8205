// Forward pass of attention with score rules (attention_rules.h): one sweep over a line's tiles with a running maximum and sum
// per row.  As in attention_fwd.hip the maximum moves only when a lane's exponentials of a step add up to more than 8192.
// Stores o and, for the backward pass, per row `ref` and `factor` with p = exp2(y - ref) * factor: ref = m + log2 l rounded to one
// float, factor what the rounding left out (1 in 16-bit types while |ref| < 64, where it is below 2^-18).  16-bit types keep what the rounding of o left out
// as well.
// Measured: a causal prompt of 8192 positions in 16 heads of 128 (8 key heads), bf16, capped scores: 396 us, 695 TFLOP/s, vector operations 53 % of the cycles, matrix
// units 29 %, which two wavefronts a SIMD overlap little (more do not fit the registers); fp16 8 x 16 x 4096 over blocks of 16 with stride 64 and a bias by distance: 153 us,
// 70 % and 21 %.
#include "attention_rules.h"

namespace bsp {
namespace {

// (four wavefronts a SIMD leave 128 registers, which a bias or documents overrun)
template <typename T, int D, bool BIAS, bool DOCS> constexpr int fwd_waves() { return sizeof(T) == 4 ? (D == 64 ? 2 : 1) : D == 64 ? (BIAS || DOCS ? 3 : 4) : 2; }

template <typename T, int D, bool CAP, bool BIAS, bool DOCS, int PAIRS>
__global__ void __launch_bounds__(128 * PAIRS, (fwd_waves<T, D, BIAS, DOCS>())) k_rules_fwd(RuleArgs a) {
  typedef Geo<T, D> Q;
  constexpr int MT = D / 32;
  extern __shared__ __attribute__((aligned(1024))) unsigned char all_smem[];
  const int group = PAIRS == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 7);
  unsigned char *smem = all_smem + group * pair_lds<T, D, PAIRS>(), *extra = smem + Q::RING;                // per stage: the documents of its 32 keys, twice
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane((tid >> 6) & 1);
  const int l32 = lane & 31, half = lane >> 5;
  const Place place = rules_place(blockIdx.x, a.Z * a.H, a.R);
  if (place.unit < 0) return;
  const int line = a.R - 1 - place.item;                // (the last lines first, which in a causal layout are the longest)
  const HeadOf head(place.unit, a.Z, a.G);
  const int h = head.h, z = head.z, hk = head.hk;
  const table_ptr lut = as_table(a.lut);
  const int row = line * 64 + 32 * wave + l32, row_in = row < a.L ? row : a.L - 1;
  bool dead;
  LineRules<DOCS> rules;
  rules.init(a, z, line, row, dead);
  f32x16 o[MT];
#pragma unroll
  for (int mt = 0; mt < MT; mt++) o[mt] = zeros16();
  float m = dead ? 0.f : -INFINITY, l = 0.f;

  Walk<DOCS> walk;
  walk.init(a.lut + lut[2 * (h * a.R + line) + 1], line * 64 < a.L ? lut[2 * (h * a.R + line)] * 2 : 0);
  auto next = [&]() {
    return walk.next(lane, [&](int lo, int hi, int bits, int hf, bool &full, bool &pad) { return rules.look(lo, hi, bits, hf, full, pad); });
  };
  Halves halves = next_halves<PAIRS>(group, next);
  if (halves.more) {
    held_t<T, D> xq;
    hold_operand<T, D>(xq, reinterpret_cast<const T *>(a.q) + z * a.q_sz + h * a.q_sh + row_in * a.q_ld, half, dead);
    const float slope = BIAS ? as_floats(a.slopes)[h] * kLog2e : 0.f, factor = apart(logit_factor<T, CAP>(a.out)), shift = CAP ? apart(logit_shift<T, CAP>(a.out)) : 0.f, in = apart(a.in);
    const i32x4r pk = rows_buffer<T, D>(reinterpret_cast<const T *>(a.k) + z * a.k_sz + hk * a.k_sh, a.k_ld, a.L);
    const i32x4r pv = rows_buffer<T, D>(reinterpret_cast<const T *>(a.v) + z * a.v_sz + hk * a.v_sh, a.v_ld, a.L);
    const i32x4r docs = buffer_of(DOCS ? a.docs + z * a.docs_sz : nullptr, (int64_t)a.L * 4);
    const uint32_t k_row = apart((uint32_t)a.k_ld * Q::ESZ), v_row = apart((uint32_t)a.v_ld * Q::ESZ);
    RowsLoad<T, D, sizeof(T) == 4> gk, gv;
    gk.init(a.k_ld, lane);
    gv.init(a.v_ld, lane);
    // each wavefront loads one of the two groups of sixteen rows of each piece
    auto issue = [&](int stage_no, const Half &x) {
      const uint32_t st = lds_address(smem) + stage_no * Q::STAGE + wave * (16 * Q::RB);
      const int pos = wave ? x.hi : x.lo;
      gk.issue(pk, pos, k_row, st);
      gv.issue(pv, pos, v_row, st + Q::PIECE);
      if (DOCS && wave == 0) load_documents(docs, x.lo, x.hi, lane, lds_address(extra) + stage_no * Q::EXTRA);
    };
    if (PAIRS == 1 || halves.own.n >= 0) issue(0, halves.own);
    PieceReads<T, D, false> reads;
    reads.init(smem, lane);

    // one half of a tile; false: it was the last
    auto step = [&](auto stage_no) {
      constexpr int S = decltype(stage_no)::value;
      const Halves all = halves, nxt = next_halves<PAIRS>(group, next);
      const Half &cur = all.own;
      quad_barrier();
      const int32_t *kd = reinterpret_cast<const int32_t *>(extra + S * Q::EXTRA);
      if (DOCS && all.pads) {
        if (PAIRS == 1 || cur.pad) {
          clear_rows<T, D>(smem + S * Q::STAGE, 16 * wave, kd, lane);
          clear_rows<T, D>(smem + S * Q::STAGE + Q::PIECE, 16 * wave, kd, lane);
        }
        lds_barrier();
      }
      if (nxt.own.n >= 0) issue(1 - S, nxt.own);
      uint32_t seen = 0xffffu;                          // bit i: the lane's row sees its key i
      bool some = true, whole = true;
      if (!cur.full) {
        const int mine = cur.bits >> (2 * (cur.n & 1) + 8 * wave + 4 * ((lane >> 4) & 1));
        seen = (mine & 1 ? first_bits(rules.limit - cur.lo - 8 * half) : 0u) | (mine & 2 ? first_bits(rules.limit - cur.hi - 8 * half) << 8 : 0u);
        if constexpr (DOCS) seen = same_document(seen, kd + 8 * half, rules.doc);
        some = __builtin_amdgcn_ballot_w64(seen != 0) != 0;
        whole = __builtin_amdgcn_ballot_w64(seen != 0xffffu) == 0;
      }
      if (some) {
        f32x16 s = rows_times<T, D, S * Q::STAGE, false>(reads, xq, zeros16());
        if constexpr (CAP)
#pragma unroll
          for (int i = 0; i < 16; i++) s[i] = cap_score<T>(s[i], in);
        const Logits<BIAS> logits(row - cur.lo - 8 * half, row - cur.hi - 8 * half, slope);
        float e[16], sum;
        for (bool moved = false;; moved = true) {
          const float ms = m == -INFINITY ? 0.f : m;
          logits.get(e, s, factor, [&](int) { return ms - shift; });
          sum = 0.f;
#pragma unroll
          for (int i = 0; i < 16; i++) e[i] = __builtin_amdgcn_exp2f(e[i]);
          if (!whole)
            for_16<0>([&](auto ic) { e[decltype(ic)::value] = keep(e[decltype(ic)::value], bit_mask<decltype(ic)::value>(seen)); });
#pragma unroll
          for (int i = 0; i < 16; i++) sum += e[i];
          if (moved || !__builtin_amdgcn_ballot_w64(sum > 8192.f || (m == -INFINITY && seen != 0))) break;
          float y[16], top = -INFINITY;
          logits.get(y, s, factor, [&](int) { return -shift; });
#pragma unroll
          for (int i = 0; i < 16; i++) top = fmaxf(top, (seen >> i) & 1 ? y[i] : -INFINITY);
          const float mn = fmaxf(m, fmaxf(top, swap32(top)));
          const float f = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
          l *= f;
#pragma unroll
          for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[mt][i] *= f;
          m = mn;
        }
        l += sum;
        Shares<T> p;
        p.set(e);
        columns_times<T, D, S * Q::STAGE + Q::PIECE, false>(o, reads, p);
      }
      halves = nxt;
      return halves.more;
    };
    while (step(Const<0>{}) && step(Const<1>{})) {}
  }

  if constexpr (PAIRS == 2) {                           // the second pair's maxima, sums and accumulators to the first
    quad_barrier();
    float *sums = reinterpret_cast<float *>(all_smem + pair_lds<T, D, PAIRS>()) + wave * (64 * (16 * MT + 2)) + lane;
    if (group) {
      sums[0] = m;
      sums[64] = l;
#pragma unroll
      for (int i = 0; i < 16 * MT; i++) sums[64 * (2 + i)] = o[i >> 4][i & 15];
    }
    lds_barrier();
    if (group) return;
    const float m2 = sums[0], top = fmaxf(m, m2), to = top == -INFINITY ? 0.f : top, f1 = __builtin_amdgcn_exp2f(m - to), f2 = __builtin_amdgcn_exp2f(m2 - to);
    m = top;
    l = l * f1 + sums[64] * f2;
#pragma unroll
    for (int i = 0; i < 16 * MT; i++) o[i >> 4][i & 15] = o[i >> 4][i & 15] * f1 + sums[64 * (2 + i)] * f2;
  }
  l += swap32(l);
  const bool none = dead || l == 0.f;                   // a row that sees no key: zeros, and no share of anything in the backward pass
  const float inv = none ? 0.f : 1.f / l;
  if (a.ref != nullptr && half == 0) {
    const float ref = none ? INFINITY : m + __builtin_amdgcn_logf(l);
    float *to = a.ref + ((int64_t)z * a.H + h) * 2 * a.rows + row;
    *to = ref;
    to[a.rows] = !none && (sizeof(T) == 4 || fabsf(ref) >= kRestFrom) ? __builtin_amdgcn_exp2f(ref - m) * inv : 1.f;
  }
#pragma unroll
  for (int mt = 0; mt < MT; mt++)
#pragma unroll
    for (int i = 0; i < 16; i++) o[mt][i] = none ? 0.f : o[mt][i] * inv;
  quad_barrier();                                       // the ring is free
  T *po = reinterpret_cast<T *>(a.o) + z * a.o_sz + h * a.o_sh;
  const int first = line * 64 + 32 * wave;
  unsigned char *stage = smem + wave * (32 * (D + Q::VEC) * Q::ESZ);
  store_some_rows<T, D>(stage, po + (int64_t)first * a.o_ld, a.L - first, po + (int64_t)(first + 16) * a.o_ld, a.L - first - 16, a.o_ld, o, lane);
  if constexpr (sizeof(T) == 2)
    if (a.ref != nullptr) {                             // what the rounding left out, for the backward pass (attention_rules_bwd.hip)
#pragma unroll
      for (int mt = 0; mt < MT; mt++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[mt][i] -= to_float(from_float<T>(o[mt][i]));
      T *pr = reinterpret_cast<T *>(a.o_rest) + (((int64_t)z * a.H + h) * a.L + first) * D;
      store_some_rows<T, D>(stage, pr, a.L - first, pr + 16 * D, a.L - first - 16, D, o, lane);
    }
}

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

template <typename T, int D, bool CAP, bool BIAS, bool DOCS> int launch_rules_fwd(const RuleArgs &a, hipStream_t st) {
  static std::atomic<uint64_t> done{0}, done2{0};
  const int64_t grid = rules_grid((int64_t)a.Z * a.H, a.R);
  if (few_lines<T, D>(a)) return rules_launch(k_rules_fwd<T, D, CAP, BIAS, DOCS, 2>, grid, 256, 2 * pair_lds<T, D, 2>(), done2, a, st);
  return rules_launch(k_rules_fwd<T, D, CAP, BIAS, DOCS, 1>, grid, 128, rules_lds<T, D>(), done, a, st);
}
template <typename T, int D, bool CAP, bool BIAS> int launch_rules_fwd(const RuleArgs &a, hipStream_t st) {
  return a.docs ? launch_rules_fwd<T, D, CAP, BIAS, true>(a, st) : launch_rules_fwd<T, D, CAP, BIAS, false>(a, st);
}
template <typename T, int D> int launch_rules_fwd(const RuleArgs &a, hipStream_t st) {
  if (a.capped) return a.slopes ? launch_rules_fwd<T, D, true, true>(a, st) : launch_rules_fwd<T, D, true, false>(a, st);
  return a.slopes ? launch_rules_fwd<T, D, false, true>(a, st) : launch_rules_fwd<T, D, false, false>(a, st);
}
template <typename T> int launch_rules_fwd(const RuleArgs &a, int D, hipStream_t st) { return D == 64 ? launch_rules_fwd<T, 64>(a, st) : launch_rules_fwd<T, 128>(a, st); }

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

extern "C" int bsp_attention_rules_fwd(const bsp_attention_rules_call *call, const void *q, const void *k, const void *v, void *o, void *stream) {
  RuleArgs a;
  const int rc = rules_args(call, a);
  if (rc != BSP_OK) return rc;
  const int64_t *s = call->strides;
  if (!q || !k || !v || !o || off16(q) || off16(k) || off16(v) || off16(o) || !s[2] || !s[5] || !s[8] || !s[11]) return BSP_ERR_ARG;
  if (call->stats && call->dtype != BSP_F32 && (!call->o_rest || off16(call->o_rest))) return BSP_ERR_ARG;
  a.q = q; a.k = k; a.v = v; a.o = o;
  a.o_sz = s[9]; a.o_sh = s[10]; a.o_ld = s[11];
  const hipStream_t st = as_stream(stream);
  if (a.docs) hipLaunchKernelGGL(k_rules_ranges, dim3((unsigned)cdiv((int64_t)a.Z * a.groups, 256)), dim3(256), 0, st, a.docs, a.docs_sz, a.L, a.groups, a.Z, call->ranges);
  const int rl = call->dtype == BSP_F16 ? launch_rules_fwd<f16>(a, call->D, st) : call->dtype == BSP_BF16 ? launch_rules_fwd<bf16>(a, call->D, st) : launch_rules_fwd<float>(a, call->D, st);
  if (rl != BSP_OK) return rl;
  BSP_LAUNCH_CHECK();
  return BSP_OK;
}
