// Forward pass of attention with score rules (attention_rules.h): one sweep over a line's tiles with a running maximum and sum
// per row.  As in attention_fwd.hip the maximum moves only when a lane's exponentials of a step add up to more than 8192.
// Stores o and, for the backward pass, per row `ref` and `factor` with p = exp2(y - ref) * factor: ref = m + log2 l rounded to one
// float, factor what the rounding left out (1 in 16-bit types while |ref| < 64, where it is below 2^-18).  16-bit types keep what the rounding of o left out
// as well.
// Measured: a causal prompt of 8192 positions in 16 heads of 128 (8 key heads), bf16, capped scores: 396 us, 695 TFLOP/s, vector operations 53 % of the cycles, matrix
// units 29 %, which two wavefronts a SIMD overlap little (more do not fit the registers); fp16 8 x 16 x 4096 over blocks of 16 with stride 64 and a bias by distance: 153 us,
// 70 % and 21 %.
//
// With X > 0 the logits have the product with a key part that all key heads share beside that with the head's own (attention_shared_fwd.hip): a third piece of a stage.  Shares are in two terms there
// (in_two_terms).
#ifndef BSP_ATTENTION_RULES_FWD_H
#define BSP_ATTENTION_RULES_FWD_H
#include "attention_rules.h"

namespace bsp {
namespace {

// (four wavefronts a SIMD leave 128 registers, which a bias or documents overrun; with a shared part, 16-bit types, a bias and documents 8 to 36 bytes a lane are in scratch memory all the same)
template <typename T, int D, int X, bool BIAS, bool DOCS> constexpr int fwd_waves() { return sizeof(T) == 4 ? (D == 64 ? 2 : 1) : D == 64 ? (BIAS || DOCS || X ? 3 : 4) : 2; }

template <typename T, int D, int X, bool CAP, bool BIAS, bool DOCS, int PAIRS>
__global__ void __launch_bounds__(128 * PAIRS, (fwd_waves<T, D, X, BIAS, DOCS>())) k_rules_fwd(RuleArgs a) {
  typedef Geo<T, D> Q;
  typedef RuleRing<T, D, X> Ring;
  constexpr int SX = X ? X : D;                         // (of types that are not used without X)
  constexpr int MT = D / 32;
  extern __shared__ __attribute__((aligned(1024))) unsigned char all_smem[];
  const int group = PAIRS == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 7);
  unsigned char *smem = all_smem + group * pair_lds<T, D, X, PAIRS>(), *extra = smem + Ring::RING;                // per stage: the documents of its 32 keys, twice
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
    held_t<T, SX> xqx;
    if constexpr (X) hold_operand<T, SX>(xqx, reinterpret_cast<const T *>(a.qx) + z * a.qx_sz + h * a.qx_sh + row_in * a.qx_ld, half, dead);
    const float slope = BIAS ? as_floats(a.slopes)[h] * kLog2e : 0.f, factor = apart(logit_factor<T, CAP>(a.out)), shift = CAP ? apart(logit_shift<T, CAP>(a.out)) : 0.f, in = apart(a.in);
    const i32x4r pk = rows_buffer<T, D>(reinterpret_cast<const T *>(a.k) + z * a.k_sz + hk * a.k_sh, a.k_ld, a.L);
    const i32x4r pv = rows_buffer<T, D>(reinterpret_cast<const T *>(a.v) + z * a.v_sz + hk * a.v_sh, a.v_ld, a.L);
    const i32x4r docs = buffer_of(DOCS ? a.docs + z * a.docs_sz : nullptr, (int64_t)a.L * 4);
    const uint32_t k_row = apart((uint32_t)a.k_ld * Q::ESZ), v_row = apart((uint32_t)a.v_ld * Q::ESZ);
    RowsLoad<T, D, sizeof(T) == 4> gk, gv;
    gk.init(a.k_ld, lane);
    gv.init(a.v_ld, lane);
    i32x4r pkx;
    uint32_t kx_row = 0;
    RowsLoad<T, SX, sizeof(T) == 4> gkx;
    if constexpr (X) {
      pkx = rows_buffer<T, SX>(reinterpret_cast<const T *>(a.kx) + z * a.kx_sz, a.kx_ld, a.L);
      kx_row = apart((uint32_t)a.kx_ld * Q::ESZ);
      gkx.init(a.kx_ld, lane);
    }
    // each wavefront loads one of the two groups of sixteen rows of each piece
    auto issue = [&](int stage_no, const Half &x) {
      const uint32_t st = lds_address(smem) + stage_no * Ring::STAGE + wave * (16 * Q::RB);
      const int pos = wave ? x.hi : x.lo;
      gk.issue(pk, pos, k_row, st);
      gv.issue(pv, pos, v_row, st + Q::PIECE);
      if constexpr (X) gkx.issue(pkx, pos, kx_row, lds_address(smem) + stage_no * Ring::STAGE + Ring::THIRD + wave * (16 * Geo<T, SX>::RB));
      if (DOCS && wave == 0) load_documents(docs, x.lo, x.hi, lane, lds_address(extra) + stage_no * Q::EXTRA);
    };
    if (PAIRS == 1 || halves.own.n >= 0) issue(0, halves.own);
    PieceReads<T, D, false> reads;
    reads.init(smem, lane);
    PieceReads<T, SX, false> readsx;
    if constexpr (X) readsx.init(smem, lane);

    // one half of a tile; false: it was the last
    auto step = [&](auto stage_no) {
      constexpr int S = decltype(stage_no)::value;
      const Halves all = halves, nxt = next_halves<PAIRS>(group, next);
      const Half &cur = all.own;
      quad_barrier();
      const int32_t *kd = reinterpret_cast<const int32_t *>(extra + S * Q::EXTRA);
      if (DOCS && all.pads) {
        if (PAIRS == 1 || cur.pad) {
          clear_rows<T, D>(smem + S * Ring::STAGE, 16 * wave, kd, lane);
          clear_rows<T, D>(smem + S * Ring::STAGE + Q::PIECE, 16 * wave, kd, lane);
          if constexpr (X) clear_rows<T, SX>(smem + S * Ring::STAGE + Ring::THIRD, 16 * wave, kd, lane);
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
        constexpr int NF = Q::NF, NX = X ? Geo<T, SX>::NF : 0, K0 = S * Ring::STAGE, V0 = K0 + Q::PIECE, X0 = K0 + Ring::THIRD;
        constexpr bool AHEAD = reads_ahead<T, D, X>();
        typedef typename RuleOperand<T>::type frag;
        f32x16 s = zeros16();
        Ahead<frag, 2 * MT, 3> columns;
        auto column = [&](int i) {
          if constexpr (AHEAD) return column_fragment<T, D, V0, false>(reads, i);
          else return frag();
        };
        if constexpr (AHEAD) {
          Ahead<frag, NF + NX, 5> rows;
          auto fragment = [&](int i) { return i < NF ? row_fragment<T, D, K0, false>(reads, i) : row_fragment<T, SX, X0, false>(readsx, i - NF); };
          rows.begin(fragment);
          rows.run(fragment, [&](int i, const frag &f) { s = fragment_times<T>(f, i < NF ? xq[i] : xqx[i - NF], s); });
          columns.begin(column);
        } else {
          s = rows_times<T, D, K0, false>(reads, xq, s);
          if constexpr (X) s = rows_times<T, SX, X0, false>(readsx, xqx, s);
        }
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
        if constexpr (in_two_terms<T, X>()) {
          Shares<T> rest;
          two_terms<T>(e, p, rest);
          if constexpr (AHEAD) {
            columns.run(column, [&](int i, const frag &f) {
              o[i % MT] = Mma<T, 32>::run(f, p.f[i / MT], o[i % MT]);
              o[i % MT] = Mma<T, 32>::run(f, rest.f[i / MT], o[i % MT]);
            });
          } else {
            columns_times_exact<T, D, V0, false>(o, reads, p, rest);
          }
        } else {
          p.set(e);
          columns_times<T, D, V0, false>(o, reads, p);
        }
      }
      halves = nxt;
      return halves.more;
    };
    while (step(Const<0>{}) && step(Const<1>{})) {}
  }

  if constexpr (PAIRS == 2) {                           // the second pair's maxima, sums and accumulators to the first
    quad_barrier();
    float *sums = reinterpret_cast<float *>(all_smem + pair_lds<T, D, X, PAIRS>()) + wave * (64 * (16 * MT + 2)) + lane;
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

template <typename T, int D, int X, bool CAP, bool BIAS, bool DOCS> int launch_rules_fwd(const RuleArgs &a, hipStream_t st) {
  static std::atomic<uint64_t> done{0}, done2{0};
  const int64_t grid = rules_grid((int64_t)a.Z * a.H, a.R);
  if constexpr (2 * pair_lds<T, D, X, 2>() <= kLdsBytes)
    if (few_lines<T, D, X>(a)) return rules_launch(k_rules_fwd<T, D, X, CAP, BIAS, DOCS, 2>, grid, 256, 2 * pair_lds<T, D, X, 2>(), done2, a, st);
  return rules_launch(k_rules_fwd<T, D, X, CAP, BIAS, DOCS, 1>, grid, 128, rules_lds<T, D, X>(), done, a, st);
}
template <typename T, int D, int X, bool CAP, bool BIAS> int launch_rules_fwd(const RuleArgs &a, hipStream_t st) {
  return a.docs ? launch_rules_fwd<T, D, X, CAP, BIAS, true>(a, st) : launch_rules_fwd<T, D, X, CAP, BIAS, false>(a, st);
}
template <typename T, int D, int X> int launch_rules_fwd(const RuleArgs &a, hipStream_t st) {
  if (a.capped) return a.slopes ? launch_rules_fwd<T, D, X, true, true>(a, st) : launch_rules_fwd<T, D, X, true, false>(a, st);
  return a.slopes ? launch_rules_fwd<T, D, X, false, true>(a, st) : launch_rules_fwd<T, D, X, false, false>(a, st);
}
template <typename T, int X> int launch_rules_fwd(const RuleArgs &a, int D, hipStream_t st) { return D == 64 ? launch_rules_fwd<T, 64, X>(a, st) : launch_rules_fwd<T, 128, X>(a, st); }
template <int X> int launch_rules_fwd(int dtype, int D, const RuleArgs &a, hipStream_t st) {
  return dtype == BSP_F16 ? launch_rules_fwd<f16, X>(a, D, st) : dtype == BSP_BF16 ? launch_rules_fwd<bf16, X>(a, D, st) : launch_rules_fwd<float, X>(a, D, st);
}

}  // namespace
}  // namespace bsp
#endif
