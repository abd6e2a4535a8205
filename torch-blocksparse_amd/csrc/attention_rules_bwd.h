// Backward pass of attention with score rules (attention_rules.h), p = exp2(y - ref) * factor computed again:
//     dv = p^T . do,   e = p * (dp - delta) * (1 - t^2)  (t the tanh of a capped score),   dq = scale * e . k,   dk = scale * e^T . q
// with dp = do . v^T and delta = sum_d do_d o_d, for which 16-bit types keep what the rounding of o left out as a second tensor: delta goes into every
// gradient of its row, and with o alone the gradients are off by 1.8 times what the roundings of p, of e and of the result make them.  16-bit types
// also take e in two terms for dq, and for dk a delta that the row kernel has corrected: errors against 64 bits (relative 2-norm) of dq 2.5e-3 -> 1.9e-3 in bf16, 3.0e-4 -> 2.2e-4 in
// fp16, of dk 2.5e-3 -> 2.35e-3, 3.0e-4 -> 2.95e-4, where rounding the results alone is 1.66e-3 and 2.07e-4.
//   row kernel    : a line of tiles per workgroup -> dq and -delta
//   column kernel : a column of tiles (or a part of a long one) of a key head per workgroup -> dk and dv; the column's tiles are
//                   those of all the query heads that share the key head, one after the other, so their sum needs no memory
// Measured: fp16 8 x 16 x 4096 over blocks of 16 with stride 64 and a bias by distance: rows 196 us (vector operations 64 % of the cycles, matrix units 34 %; 176 with e in one term), columns 255 (42 %,
// 26 %), sums of their parts 16; bf16 2 x 16 (4 key heads) x 4001 x 128, six documents, capped scores: 153 (132 with e in one term), 204 and 14, where the longest document's lines and columns are what takes so
// long; fp32 2 x 8 x 2023, two documents: 71, 97 and 7.
//
// With X > 0 (attention_shared_bwd.hip) a key part that all key heads share has part in the logits: its gradient is scale * e^T . qx summed over the heads, kept for each
// key head in fp32 and added by a last kernel; that of qx is scale * e . kx.  p and e are in two terms there, in all their products (in_two_terms).
#ifndef BSP_ATTENTION_RULES_BWD_H
#define BSP_ATTENTION_RULES_BWD_H
#include "attention_rules.h"

namespace bsp {
namespace {

// wavefronts a SIMD that the registers are for (with a shared part one fewer, or they spill: the rows of 16-bit types and 128 elements 90 to 250 bytes a lane.  What does so with a shared part as it is: the columns of fp32 and 128
// elements, at one wavefront a SIMD, 16 to 24 bytes, with a cap or documents 88 to 172; those of 16-bit types and 64 elements with all rules 12)
template <typename T, int D, int X, bool CAP> constexpr int row_waves() { return sizeof(T) == 4 ? (D == 64 && !X ? 2 : 1) : D == 64 ? (CAP || X ? 2 : 3) : X ? 1 : 2; }
template <typename T, int D, int X, bool CAP> constexpr int col_waves() { return D == 64 && !(X && sizeof(T) == 4) ? 2 : 1; }

template <typename T, int D, int X, bool CAP, bool BIAS, bool DOCS, int PAIRS>
__global__ void __launch_bounds__(128 * PAIRS, (row_waves<T, D, X, CAP>())) k_rules_bwd_rows(RuleArgs a) {
  typedef Geo<T, D> Q;
  typedef RuleRing<T, D, X> Ring;
  constexpr int MT = D / 32, SX = X ? X : D, XT = X / 32;   // (SX: of types that are not used without X)
  extern __shared__ __attribute__((aligned(1024))) unsigned char all_smem[];
  const int group = PAIRS == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 7);
  unsigned char *smem = all_smem + group * pair_lds<T, D, X, PAIRS>(), *extra = smem + Ring::RING;
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
  f32x16 dq[MT];
#pragma unroll
  for (int mt = 0; mt < MT; mt++) dq[mt] = zeros16();
  f32x16 dqx[SX / 32];
  if constexpr (X)
#pragma unroll
    for (int mt = 0; mt < XT; mt++) dqx[mt] = zeros16();

  held_t<T, D> xo;
  hold_operand<T, D>(xo, reinterpret_cast<const T *>(a.d_o) + z * a.do_sz + h * a.do_sh + row_in * a.do_ld, half, dead);
  float delta = 0.f;
  {
    held_t<T, D> of;
    hold_operand<T, D>(of, reinterpret_cast<const T *>(a.o_in) + z * a.oin_sz + h * a.oin_sh + row_in * a.oin_ld, half, dead);
#pragma unroll
    for (int s = 0; s < Q::NF; s++)
#pragma unroll
      for (int i = 0; i < Q::VEC; i++) delta = fmaf(to_float(xo[s][i]), to_float(of[s][i]), delta);
    if constexpr (sizeof(T) == 2) {                      // ... and with what the rounding of o left out
      hold_operand<T, D>(of, reinterpret_cast<const T *>(a.o_rest) + (((int64_t)z * a.H + h) * a.L + row_in) * D, half, dead);
#pragma unroll
      for (int s = 0; s < Q::NF; s++)
#pragma unroll
        for (int i = 0; i < Q::VEC; i++) delta = fmaf(to_float(xo[s][i]), to_float(of[s][i]), delta);
    }
    delta += swap32(delta);
  }
  // delta is also sum_j p_j dp_j.  The two differ by what the rounding of the forward pass's shares made of o, in 16-bit types enough to see in the gradients: what the
  // row's sum of p (dp - delta) is off zero by is added for the column kernel.
  constexpr bool FINE = sizeof(T) == 2;
  float off = 0.f;

  Walk<DOCS> walk;
  walk.init(a.lut + lut[2 * (h * a.R + line) + 1], line * 64 < a.L ? lut[2 * (h * a.R + line)] * 2 : 0);
  auto next = [&]() {
    return walk.next(lane, [&](int lo, int hi, int bits, int hf, bool &full, bool &pad) { return rules.look(lo, hi, bits, hf, full, pad); });
  };
  const float *stats = a.ref + ((int64_t)z * a.H + h) * 2 * a.rows + row;
  const float ref = stats[0], factor = stats[a.rows];
  Halves halves = next_halves<PAIRS>(group, next);
  if (halves.more) {
    held_t<T, D> xq;
    hold_operand<T, D>(xq, reinterpret_cast<const T *>(a.q) + z * a.q_sz + h * a.q_sh + row_in * a.q_ld, half, dead);
    held_t<T, SX> xqx;
    if constexpr (X) hold_operand<T, SX>(xqx, reinterpret_cast<const T *>(a.qx) + z * a.qx_sz + h * a.qx_sh + row_in * a.qx_ld, half, dead);
    const float slope = BIAS ? as_floats(a.slopes)[h] * kLog2e : 0.f, out = apart(logit_factor<T, CAP>(a.out)), in = apart(a.in), minus = ref - logit_shift<T, CAP>(a.out) - (CAP && sizeof(T) != 4 ? 2.f : 0.f);   // (e^y times four: see cap_through)
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
    PieceReads<T, D, false> reads;                      // the same for the k and the v piece
    reads.init(smem, lane);
    PieceReads<T, SX, false> readsx;
    if constexpr (X) readsx.init(smem, lane);

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
      uint32_t seen = 0xffffu;                          // as in the forward kernel
      bool some = true, whole = true;
      if (!cur.full) {
        const int mine = cur.bits >> (2 * (cur.n & 1) + 8 * wave + 4 * ((lane >> 4) & 1));
        seen = (mine & 1 ? first_bits(rules.limit - cur.lo - 8 * half) : 0u) | (mine & 2 ? first_bits(rules.limit - cur.hi - 8 * half) << 8 : 0u);
        if constexpr (DOCS) seen = same_document(seen, kd + 8 * half, rules.doc);
        some = __builtin_amdgcn_ballot_w64(seen != 0) != 0;
        whole = __builtin_amdgcn_ballot_w64(seen != 0xffffu) == 0;
      }
      if (some) {
        constexpr bool AHEAD = reads_ahead<T, D, X>();
        constexpr int NF = Q::NF, NX = X ? Geo<T, SX>::NF : 0, K0 = S * Ring::STAGE, V0 = K0 + Q::PIECE, X0 = K0 + Ring::THIRD;
        typedef typename RuleOperand<T>::type frag;
        f32x16 s = zeros16(), dp = zeros16();
        Ahead<frag, 2 * (MT + XT), 6> columns;
        auto column = [&](int i) {
          if constexpr (AHEAD) return i < 2 * MT ? column_fragment<T, D, K0, false>(reads, i) : column_fragment<T, SX, X0, false>(readsx, i - 2 * MT);
          else return frag();
        };
        if constexpr (AHEAD) {
          Ahead<frag, 2 * NF + NX, 6> rows;
          auto fragment = [&](int i) {
            return i < NF ? row_fragment<T, D, K0, false>(reads, i) : i < NF + NX ? row_fragment<T, SX, X0, false>(readsx, i - NF) : row_fragment<T, D, V0, false>(reads, i - NF - NX);
          };
          rows.begin(fragment);
          rows.run(fragment, [&](int i, const frag &f) {
            if (i < NF) s = fragment_times<T>(f, xq[i], s);
            else if (i < NF + NX) s = fragment_times<T>(f, xqx[i - NF], s);
            else dp = fragment_times<T>(f, xo[i - NF - NX], dp);
          });
          columns.begin(column);
        } else {
          s = rows_times<T, D, K0, false>(reads, xq, s);
          if constexpr (X) s = rows_times<T, SX, X0, false>(readsx, xqx, s);
          dp = rows_times<T, D, V0, false>(reads, xo, dp);
        }
        const Logits<BIAS> logits(row - cur.lo - 8 * half, row - cur.hi - 8 * half, slope);
        if constexpr (CAP)
#pragma unroll
          for (int i = 0; i < 16; i++) s[i] = cap_score<T>(s[i], in);
        float e[16];
        logits.get(e, s, out, [&](int) { return minus; });
#pragma unroll
        for (int i = 0; i < 16; i++) e[i] = __builtin_amdgcn_exp2f(e[i]) * (dp[i] - delta);
        auto keep_seen = [&]() {
          if (!whole)
            for_16<0>([&](auto ic) { e[decltype(ic)::value] = keep(e[decltype(ic)::value], bit_mask<decltype(ic)::value>(seen)); });
        };
        if constexpr (FINE) {
          keep_seen();
          float sums[4];
#pragma unroll
          for (int i = 0; i < 4; i++) sums[i] = (e[i] + e[4 + i]) + (e[8 + i] + e[12 + i]);
          off += (sums[0] + sums[1]) + (sums[2] + sums[3]);
        }
        if constexpr (CAP)
#pragma unroll
          for (int i = 0; i < 16; i++) e[i] *= cap_through<T, true>(s[i]);
        if constexpr (CAP || !FINE) keep_seen();
        if constexpr (FINE) {
          Shares<T> most, rest;
          two_terms<T>(e, most, rest);
          if constexpr (AHEAD) {
            columns.run(column, [&](int i, const frag &f) {
              const int ks = i < 2 * MT ? i / MT : (i - 2 * MT) / XT;
              f32x16 &to = i < 2 * MT ? dq[i % MT] : dqx[(i - 2 * MT) % XT];
              to = Mma<T, 32>::run(f, most.f[ks], to);
              to = Mma<T, 32>::run(f, rest.f[ks], to);
            });
          } else {
            columns_times_exact<T, D, K0, false>(dq, reads, most, rest);
            if constexpr (X) columns_times_exact<T, SX, X0, false>(dqx, readsx, most, rest);
          }
        } else {
          Shares<T> ds;
          ds.set(e);
          columns_times<T, D, K0, false>(dq, reads, ds);
          if constexpr (X) columns_times<T, SX, X0, false>(dqx, readsx, ds);
        }
      }
      halves = nxt;
      return halves.more;
    };
    while (step(Const<0>{}) && step(Const<1>{})) {}
  }
  if constexpr (PAIRS == 2) {                           // the second pair's sums to the first
    quad_barrier();
    float *sums = reinterpret_cast<float *>(all_smem + pair_lds<T, D, X, PAIRS>()) + wave * (64 * (16 * (MT + XT) + 2)) + lane;
    if (group) {
      sums[0] = off;
#pragma unroll
      for (int i = 0; i < 16 * MT; i++) sums[64 * (1 + i)] = dq[i >> 4][i & 15];
      if constexpr (X)
#pragma unroll
        for (int i = 0; i < 16 * XT; i++) sums[64 * (1 + 16 * MT + i)] = dqx[i >> 4][i & 15];
    }
    lds_barrier();
    if (group) return;
    off += sums[0];
#pragma unroll
    for (int i = 0; i < 16 * MT; i++) dq[i >> 4][i & 15] += sums[64 * (1 + i)];
    if constexpr (X)
#pragma unroll
      for (int i = 0; i < 16 * XT; i++) dqx[i >> 4][i & 15] += sums[64 * (1 + 16 * MT + i)];
  }
  if constexpr (FINE) delta += (off + swap32(off)) * factor * (CAP ? 0.25f : 1.f);
  if (half == 0) a.delta[((int64_t)z * a.H + h) * a.rows + row] = -delta;   // (its negative: where the column kernel's dp starts from)
  const float last = a.scale * factor;
#pragma unroll
  for (int mt = 0; mt < MT; mt++)
#pragma unroll
    for (int i = 0; i < 16; i++) dq[mt][i] *= last;
  quad_barrier();                                       // the ring is free
  T *po = reinterpret_cast<T *>(a.o) + z * a.o_sz + h * a.o_sh;
  const int first = line * 64 + 32 * wave;
  store_some_rows<T, D>(smem + wave * (32 * (D + Q::VEC) * Q::ESZ), po + (int64_t)first * a.o_ld, a.L - first, po + (int64_t)(first + 16) * a.o_ld, a.L - first - 16, a.o_ld, dq, lane);
  if constexpr (X) {
#pragma unroll
    for (int mt = 0; mt < XT; mt++)
#pragma unroll
      for (int i = 0; i < 16; i++) dqx[mt][i] *= last;
    T *px = reinterpret_cast<T *>(a.ox) + z * a.ox_sz + h * a.ox_sh;
    store_some_rows<T, SX>(smem + wave * (32 * (D + Q::VEC) * Q::ESZ), px + (int64_t)first * a.ox_ld, a.L - first, px + (int64_t)(first + 16) * a.ox_ld, a.L - first - 16, a.ox_ld, dqx, lane);
  }
}

// Columns.  A work item is a column of tiles (64 keys: four groups of sixteen) of a key head or a part of a long one: twelve
// ints (tiles, offset of their entries, key head, column or -1: nothing to do, slot of its partial sums or -1, ., ., ., the positions of the four groups
// of keys); an entry names the four groups of rows, each by its query head among those of the key head, times 2^24, plus its
// position.  A wavefront owns 32 of the keys; its k and v rows stay in registers.
constexpr int kHeadShift = 24, kPosition = (1 << kHeadShift) - 1;

template <typename T, int D, int X, bool CAP, bool BIAS, bool DOCS>
__global__ void __launch_bounds__(128, (col_waves<T, D, X, CAP>())) k_rules_bwd_cols(RuleArgs a) {
  typedef Geo<T, D> Q;
  typedef RuleRing<T, D, X> Ring;
  constexpr int MT = D / 32, SX = X ? X : D, XT = X / 32;   // (SX: of types that are not used without X)
  // dk, dv, k and v alone take 192 registers at head dimension 128; at 64 what this saves is the third wavefront a SIMD, where no rule needs the registers
  // (BigBird 12 x 16384: 76 -> 67 us; with a bias, which has two wavefronts either way: 312 -> 322)
  constexpr bool LEAN = D == 128 || sizeof(T) == 4 || X || !(CAP || BIAS || DOCS);
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  unsigned char *extra = smem + Ring::RING;                // per stage: ref of its 32 rows, their factors, their -delta (twice), their documents (twice)
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, half = lane >> 5;
  const int kv_heads = (int)Quotient(a.H, a.G).q;
  const Place place = rules_place(blockIdx.x, a.Z * kv_heads, a.R);
  if (place.unit < 0) return;
  const HeadOf of(place.unit, a.Z, 1);
  const int z = of.z, hk = of.hk;
  const table_ptr head = as_table(a.lut) + 12 * (hk * a.R + place.item);
  if (head[3] < 0) return;                              // (the key heads' lists are filled up to one length)
  const int slot = head[4];
  const int key_lo = head[8 + 2 * wave], key_hi = head[8 + 2 * wave + 1];
  const int key = (l32 < 16 ? key_lo : key_hi) + (l32 & 15), key_in = key < a.L ? key : a.L - 1;
  const int doc = DOCS ? a.docs[z * a.docs_sz + key_in] : 0;
  const bool dead = key >= a.L || doc < 0;
  const int prefix = a.causal && a.prefix ? as_table(a.prefix)[z] : 0;
  // the lane's key is seen by the rows from this one on
  const int from = dead ? kPosition : a.causal && key >= prefix ? key : 0;
  int key_min = head[8], key_max = head[8];
#pragma unroll
  for (int g = 1; g < 4; g++) {
    const int p = head[8 + g];
    key_min = p < key_min ? p : key_min;
    key_max = p > key_max ? p : key_max;
  }
  key_max += 15;
  const int L = apart(a.L), most = apart(a.causal && key_max >= prefix ? key_max : 0), least = apart(a.causal && key_min >= prefix ? key_min : 0);   // rows from `most` on see all of the column's keys, those below `least` none
  Range range{0, 0};
  Ranges ranges;
  if constexpr (DOCS) {
    ranges.init(a, z);
    range = ranges.at(head[8]);
#pragma unroll
    for (int g = 1; g < 4; g++) {
      const Range r = ranges.at(head[8 + g]);
      range.lo = r.lo < range.lo ? r.lo : range.lo;
      range.hi = r.hi > range.hi ? r.hi : range.hi;
    }
  }
  f32x16 dk[MT], dv[MT];
#pragma unroll
  for (int mt = 0; mt < MT; mt++) dk[mt] = dv[mt] = zeros16();
  f32x16 dkx[SX / 32];
  if constexpr (X)
#pragma unroll
    for (int mt = 0; mt < XT; mt++) dkx[mt] = zeros16();

  Walk<DOCS> walk;
  walk.init(a.lut + head[1], key_min < a.L ? head[0] * 2 : 0);
  auto next = [&]() {
    return walk.next(lane, [&](int lo, int hi, int bits, int hf, bool &full, bool &pad) {
      bits >>= 8 * hf;
      lo &= kPosition;
      hi &= kPosition;
      bool see_lo = (bits & 0x0f) && lo < L && lo + 15 >= least, see_hi = (bits & 0xf0) && hi < L && hi + 15 >= least;
      full = (bits & 0xff) == 0xff && lo >= most && hi >= most;
      if constexpr (DOCS) {
        const Range x = ranges.at(lo), y = ranges.at(hi);
        const int low = range.lo < 0 ? 0 : range.lo;
        see_lo = see_lo && x.hi >= low && x.lo <= range.hi;
        see_hi = see_hi && y.hi >= low && y.lo <= range.hi;
        full = full && range.lo == range.hi && x.lo == range.lo && x.hi == range.lo && y.lo == range.lo && y.hi == range.lo;
        pad = x.lo < 0 || y.lo < 0;
      }
      return see_lo || see_hi;
    });
  };
  Half cur = next();
  if (cur.n >= 0) {
    held_t<T, D> xk, xv;
    hold_operand<T, D>(xk, reinterpret_cast<const T *>(a.k) + z * a.k_sz + hk * a.k_sh + key_in * a.k_ld, half, dead);
    hold_operand<T, D>(xv, reinterpret_cast<const T *>(a.v) + z * a.v_sz + hk * a.v_sh + key_in * a.v_ld, half, dead);
    held_t<T, SX> xkx;
    if constexpr (X) hold_operand<T, SX>(xkx, reinterpret_cast<const T *>(a.kx) + z * a.kx_sz + key_in * a.kx_ld, half, dead);
    const int first_head = hk * a.G;
    const char *pq = reinterpret_cast<const char *>(reinterpret_cast<const T *>(a.q) + z * a.q_sz + first_head * a.q_sh);
    const char *pdo = reinterpret_cast<const char *>(reinterpret_cast<const T *>(a.d_o) + z * a.do_sz + first_head * a.do_sh);
    const int64_t q_head = apart(a.q_sh * Q::ESZ), do_head = apart(a.do_sh * Q::ESZ);
    const uint32_t q_row = apart((uint32_t)a.q_ld * Q::ESZ), do_row = apart((uint32_t)a.do_ld * Q::ESZ);
    i32x4r q_rows = rows_buffer<T, D>(reinterpret_cast<const T *>(pq), a.q_ld, a.L), do_rows = rows_buffer<T, D>(reinterpret_cast<const T *>(pdo), a.do_ld, a.L);
    const i32x4r docs = buffer_of(DOCS ? a.docs + z * a.docs_sz : nullptr, (int64_t)a.L * 4);
    const i32x4r stats = wave == 0 ? buffer_of(a.ref + ((int64_t)z * a.H + first_head) * 2 * a.rows, a.G * a.rows * 8) : buffer_of(a.delta + ((int64_t)z * a.H + first_head) * a.rows, a.G * a.rows * 4);
    const int per = apart((int)a.rows << (1 - wave)), lane_stat = (lane & 15) + (wave == 0 && half ? (int)a.rows : 0);
    const float in = apart(a.in), out = apart(logit_factor<T, CAP>(a.out)), shift = CAP ? apart(logit_shift<T, CAP>(a.out)) : 0.f;
    const float *slopes = BIAS ? apart(a.slopes + first_head) : nullptr;
    RowsLoad<T, D, LEAN> gq, gdo;
    gq.init(a.q_ld, lane);
    gdo.init(a.do_ld, lane);
    const char *pqx = nullptr;
    int64_t qx_head = 0;
    uint32_t qx_row = 0;
    i32x4r qx_rows;
    RowsLoad<T, SX, LEAN> gqx;
    if constexpr (X) {
      pqx = reinterpret_cast<const char *>(reinterpret_cast<const T *>(a.qx) + z * a.qx_sz + first_head * a.qx_sh);
      qx_head = apart(a.qx_sh * Q::ESZ);
      qx_row = apart((uint32_t)a.qx_ld * Q::ESZ);
      qx_rows = rows_buffer<T, SX>(reinterpret_cast<const T *>(pqx), a.qx_ld, a.L);
      gqx.init(a.qx_ld, lane);
    }
    int head_now = 0;                                   // the query head that q_rows and do_rows are of
    auto issue = [&](int stage_no, const Half &x) {
      const uint32_t st = lds_address(smem) + stage_no * Ring::STAGE + wave * (16 * Q::RB), ex = lds_address(extra) + stage_no * Q::EXTRA;
      const int pos = wave ? x.hi : x.lo, hq = pos >> kHeadShift, lo = x.lo & kPosition, hi = x.hi & kPosition;
      if (hq != head_now) {
        head_now = hq;
        q_rows = move_buffer(q_rows, pq + hq * q_head);
        do_rows = move_buffer(do_rows, pdo + hq * do_head);
        if constexpr (X) qx_rows = move_buffer(qx_rows, pqx + hq * qx_head);
      }
      gq.issue(q_rows, pos & kPosition, q_row, st);
      gdo.issue(do_rows, pos & kPosition, do_row, st + Q::PIECE);
      if constexpr (X) gqx.issue(qx_rows, pos & kPosition, qx_row, lds_address(smem) + stage_no * Ring::STAGE + Ring::THIRD + wave * (16 * Geo<T, SX>::RB));
      const int at_lo = (x.lo >> kHeadShift) * per + lo, at_hi = (x.hi >> kHeadShift) * per + hi;
      buffer_to_lds<4>(stats, (uint32_t)((lane & 16 ? at_hi : at_lo) + lane_stat) * 4u, 0, ex + wave * 256);
      if (DOCS && wave == 1) load_documents(docs, lo, hi, lane, ex + 512);
    };
    issue(0, cur);
    PieceReads<T, D, LEAN> reads;                       // the same for the q and the do piece
    reads.init(smem, lane);
    PieceReads<T, SX, LEAN> readsx;
    if constexpr (X) readsx.init(smem, lane);

    auto step = [&](auto stage_no) {
      constexpr int S = decltype(stage_no)::value, Q0 = S * Ring::STAGE, O0 = Q0 + Q::PIECE, X0 = Q0 + Ring::THIRD;
      const Half nxt = next();
      quad_barrier();
      const int lo = cur.lo & kPosition, hi = cur.hi & kPosition;
      const float *stat = reinterpret_cast<const float *>(extra + S * Q::EXTRA);
      const int32_t *rd = reinterpret_cast<const int32_t *>(extra + S * Q::EXTRA + 512);
      if (DOCS && cur.pad) {
        clear_rows<T, D>(smem + Q0, 16 * wave, rd, lane);
        clear_rows<T, D>(smem + O0, 16 * wave, rd, lane);
        if constexpr (X) clear_rows<T, SX>(smem + X0, 16 * wave, rd, lane);
        lds_barrier();
      }
      if (nxt.n >= 0) issue(1 - S, nxt);
      uint32_t seen = 0xffffu;                          // bit i: the lane's key is seen by row i of the lane's sixteen
      bool some = true, whole = true;
      if (!cur.full) {
        const int mine = cur.bits >> (8 * (cur.n & 1) + 2 * wave + ((lane >> 4) & 1));
        seen = (mine & 1 ? 0xffu & ~first_bits(from - lo - 8 * half) : 0u) | (mine & 16 ? (0xffu & ~first_bits(from - hi - 8 * half)) << 8 : 0u);
        if constexpr (DOCS) seen = same_document(seen, rd + 8 * half, doc);
        some = __builtin_amdgcn_ballot_w64(seen != 0) != 0;
        whole = __builtin_amdgcn_ballot_w64(seen != 0xffffu) == 0;
      }
      if (some) {
        const bool factors = __builtin_amdgcn_ballot_w64(stat[32 + l32] != 1.f) != 0;
        constexpr bool AHEAD = reads_ahead<T, D, X>();
        constexpr int NF = Q::NF, NX = X ? Geo<T, SX>::NF : 0;
        typedef typename RuleOperand<T>::type frag;
        f32x16 s = zeros16();
        // of the products p^T . do and do . v^T, then of e^T . q
        Ahead<frag, 2 * MT + NF, 6> of_do;
        Ahead<frag, 2 * (MT + XT), 6> of_q;
        auto do_fragment = [&](int i) {
          if constexpr (AHEAD) return i < 2 * MT ? column_fragment<T, D, O0, LEAN>(reads, i) : row_fragment<T, D, O0, LEAN>(reads, i - 2 * MT);
          else return frag();
        };
        auto q_fragment = [&](int i) {
          if constexpr (AHEAD) return i < 2 * MT ? column_fragment<T, D, Q0, LEAN>(reads, i) : column_fragment<T, SX, X0, LEAN>(readsx, i - 2 * MT);
          else return frag();
        };
        if constexpr (AHEAD) {
          Ahead<frag, NF + NX, 6> rows;
          auto fragment = [&](int i) { return i < NF ? row_fragment<T, D, Q0, LEAN>(reads, i) : row_fragment<T, SX, X0, LEAN>(readsx, i - NF); };
          rows.begin(fragment);
          rows.run(fragment, [&](int i, const frag &f) { s = fragment_times<T>(f, i < NF ? xk[i] : xkx[i - NF], s); });
          of_do.begin(do_fragment);
        } else {
          s = rows_times<T, D, Q0, LEAN>(reads, xk, s);
          if constexpr (X) s = rows_times<T, SX, X0, LEAN>(readsx, xkx, s);
        }
        float slope_lo = 0.f, slope_hi = 0.f;
        if constexpr (BIAS) {
          slope_lo = as_floats(slopes)[cur.lo >> kHeadShift] * kLog2e;
          slope_hi = as_floats(slopes)[cur.hi >> kHeadShift] * kLog2e;
        }
        const Logits<BIAS> logits(key - lo - 8 * half, key - hi - 8 * half, slope_lo, slope_hi);
        if constexpr (CAP)
#pragma unroll
          for (int i = 0; i < 16; i++) s[i] = cap_score<T>(s[i], in);
        // the rows' values, in the lane's order: 8 half .., 16 + 8 half ..
        const float *st = stat + 8 * half;
        float p[16], e[16];
        {
          f32x4 ref[4];
#pragma unroll
          for (int g = 0; g < 4; g++) ref[g] = *reinterpret_cast<const f32x4 *>(st + 16 * (g >> 1) + 4 * (g & 1));
          logits.get(p, s, out, [&](int i) { return ref[i >> 2][i & 3] - shift; });
        }
#pragma unroll
        for (int i = 0; i < 16; i++) p[i] = __builtin_amdgcn_exp2f(p[i]);
        if (factors)
#pragma unroll
          for (int g = 0; g < 4; g++) {
            const f32x4 f = *reinterpret_cast<const f32x4 *>(st + 32 + 16 * (g >> 1) + 4 * (g & 1));
#pragma unroll
            for (int j = 0; j < 4; j++) p[4 * g + j] *= f[j];
          }
        if (!whole)
          for_16<0>([&](auto ic) { p[decltype(ic)::value] = keep(p[decltype(ic)::value], bit_mask<decltype(ic)::value>(seen)); });
        constexpr bool TWO = in_two_terms<T, X>();
        Shares<T> share, rest;
        if constexpr (TWO) {
          float left[16];
#pragma unroll
          for (int i = 0; i < 16; i++) left[i] = p[i];
          two_terms<T>(left, share, rest);
        } else {
          share.set(p);
        }
        if constexpr (TWO && !AHEAD) columns_times_exact<T, D, O0, LEAN>(dv, reads, share, rest);
        else if constexpr (!AHEAD) columns_times<T, D, O0, LEAN>(dv, reads, share);
        f32x16 dp;
#pragma unroll
        for (int g = 0; g < 4; g++) {
          const f32x4 nd = *reinterpret_cast<const f32x4 *>(st + 64 + 16 * (g >> 1) + 4 * (g & 1));
#pragma unroll
          for (int j = 0; j < 4; j++) dp[4 * g + j] = nd[j];
        }
        if constexpr (AHEAD) {
          of_do.run(do_fragment, [&](int i, const frag &f) {
            if (i < 2 * MT) {
              dv[i % MT] = Mma<T, 32>::run(f, share.f[i / MT], dv[i % MT]);
              dv[i % MT] = Mma<T, 32>::run(f, rest.f[i / MT], dv[i % MT]);
            }
            else dp = fragment_times<T>(f, xv[i - 2 * MT], dp);
          });
          of_q.begin(q_fragment);
        } else {
          dp = rows_times<T, D, O0, LEAN>(reads, xv, dp);
        }
#pragma unroll
        for (int i = 0; i < 16; i++) {
          e[i] = p[i] * dp[i];
          if constexpr (CAP) e[i] *= cap_through<T, __is_same(T, bf16)>(s[i]);   // (fp16 keeps the factor: what is rounded next should be no smaller than it is)
        }
        if (!whole)
          for_16<0>([&](auto ic) { e[decltype(ic)::value] = keep(e[decltype(ic)::value], bit_mask<decltype(ic)::value>(seen)); });
        if constexpr (TWO) two_terms<T>(e, share, rest);
        else share.set(e);
        if constexpr (AHEAD) {
          of_q.run(q_fragment, [&](int i, const frag &f) {
            f32x16 &to = i < 2 * MT ? dk[i % MT] : dkx[(i - 2 * MT) % XT];
            const int ks = i < 2 * MT ? i / MT : (i - 2 * MT) / XT;
            to = Mma<T, 32>::run(f, share.f[ks], to);
            to = Mma<T, 32>::run(f, rest.f[ks], to);
          });
        } else if constexpr (TWO) {
          columns_times_exact<T, D, Q0, LEAN>(dk, reads, share, rest);
          columns_times_exact<T, SX, X0, LEAN>(dkx, readsx, share, rest);
        } else {
          columns_times<T, D, Q0, LEAN>(dk, reads, share);
          if constexpr (X) columns_times<T, SX, X0, LEAN>(dkx, readsx, share);
        }
      }
      cur = nxt;
      return cur.n >= 0;
    };
    while (step(Const<0>{}) && step(Const<1>{})) {}
  }
#pragma unroll
  for (int mt = 0; mt < MT; mt++)
#pragma unroll
    for (int i = 0; i < 16; i++) dk[mt][i] *= a.scale * (CAP && __is_same(T, bf16) ? 4.f : 1.f);
  if constexpr (X)
#pragma unroll
    for (int mt = 0; mt < XT; mt++)
#pragma unroll
      for (int i = 0; i < 16; i++) dkx[mt][i] *= a.scale * (CAP && __is_same(T, bf16) ? 4.f : 1.f);
  constexpr int SLOT = 64 * (2 * D + X);
  auto store_x = [&](float *to) {                       // the lane's key's
#pragma unroll
    for (int j = 0; j < XT; j++)
#pragma unroll
      for (int g = 0; g < 4; g++) *reinterpret_cast<f32x4 *>(to + 4 * half + 32 * j + 8 * g) = f32x4{dkx[j][4 * g], dkx[j][4 * g + 1], dkx[j][4 * g + 2], dkx[j][4 * g + 3]};
  };
  if (slot >= 0) {                                      // a part of a long column: fp32 sums to its slot [dk, dv][64 keys][D]
    float *ws = a.partial + ((int64_t)z * a.n_slots + slot) * SLOT + (32 * wave + l32) * D + 4 * half;
#pragma unroll
    for (int j = 0; j < MT; j++)
#pragma unroll
      for (int g = 0; g < 4; g++) {
        *reinterpret_cast<f32x4 *>(ws + 32 * j + 8 * g) = f32x4{dk[j][4 * g], dk[j][4 * g + 1], dk[j][4 * g + 2], dk[j][4 * g + 3]};
        *reinterpret_cast<f32x4 *>(ws + 64 * D + 32 * j + 8 * g) = f32x4{dv[j][4 * g], dv[j][4 * g + 1], dv[j][4 * g + 2], dv[j][4 * g + 3]};
      }
    if constexpr (X) store_x(a.partial + ((int64_t)z * a.n_slots + slot) * SLOT + 2 * 64 * D + (32 * wave + l32) * X);
    return;
  }
  if constexpr (X)
    if (key < a.L) store_x(a.kx_heads + (((int64_t)z * kv_heads + hk) * a.L + key) * X);
  quad_barrier();                                       // the ring is free
  unsigned char *stage = smem + wave * (32 * (D + Q::VEC) * Q::ESZ);
  T *pdk = reinterpret_cast<T *>(a.o) + z * a.o_sz + hk * a.o_sh, *pdv = reinterpret_cast<T *>(a.o2) + z * a.o2_sz + hk * a.o2_sh;
  store_some_rows<T, D>(stage, pdk + (int64_t)key_lo * a.o_ld, a.L - key_lo, pdk + (int64_t)key_hi * a.o_ld, a.L - key_hi, a.o_ld, dk, lane);
  store_some_rows<T, D>(stage, pdv + (int64_t)key_lo * a.o2_ld, a.L - key_lo, pdv + (int64_t)key_hi * a.o2_ld, a.L - key_hi, a.o2_ld, dv, lane);
}

// dk and dv of the columns computed in parts: the sum of the parts' slots in order.  split_lut: per such column eight ints
// (key head, column, first slot, parts, the positions of its four groups of keys).
template <typename T, int D, int X> __global__ void __launch_bounds__(256) k_rules_bwd_cols_sum(RuleArgs a) {
  constexpr int PER = 64 * D / 4, SLOT = 64 * (2 * D + X), WGS = SLOT / 4 / 256;   // four values a thread
  const int piece = blockIdx.x % WGS, col = (blockIdx.x / WGS) % a.n_split, z = (blockIdx.x / WGS) / a.n_split;
  const table_ptr lut = as_table(a.split_lut) + 8 * col;
  const int hk = lut[0], first = lut[2], parts = lut[3];
  const float *ws = a.partial + ((int64_t)z * a.n_slots + first) * SLOT;
  const int g = piece * 256 + threadIdx.x, which = g / PER, rem = g % PER, shared = which == 2;
  const int key = shared ? rem / (X / 4 + !X) : rem / (D / 4), d4 = shared ? rem % (X / 4 + !X) : rem % (D / 4);
  const int pos = (key < 32 ? (key < 16 ? lut[4] : lut[5]) : (key < 48 ? lut[6] : lut[7])) + (key & 15);
  if (pos >= a.L) return;
  f32x4 sum = *reinterpret_cast<const f32x4 *>(ws + 4 * g);
  for (int part = 1; part < parts; part++) {
    const f32x4 v = *reinterpret_cast<const f32x4 *>(ws + (int64_t)part * SLOT + 4 * g);
#pragma unroll
    for (int e = 0; e < 4; e++) sum[e] += v[e];
  }
  if constexpr (X)
    if (shared) {
      *reinterpret_cast<f32x4 *>(a.kx_heads + (((int64_t)z * (int)Quotient(a.H, a.G).q + hk) * a.L + pos) * X + 4 * d4) = sum;
      return;
    }
  T *dst = (which ? reinterpret_cast<T *>(a.o2) + z * a.o2_sz + hk * a.o2_sh + (int64_t)pos * a.o2_ld
                  : reinterpret_cast<T *>(a.o) + z * a.o_sz + hk * a.o_sh + (int64_t)pos * a.o_ld) + 4 * d4;
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<f32x4 *>(dst) = sum;
  } else {
    union { u32x2 raw; T e[4]; } pk;
#pragma unroll
    for (int e = 0; e < 4; e++) pk.e[e] = from_float<T>(sum[e]);
    *reinterpret_cast<u32x2 *>(dst) = pk.raw;
  }
}

template <typename T, int D, int X, bool CAP, bool BIAS, bool DOCS> int launch_rules_bwd(const RuleArgs &a, bool cols, hipStream_t st) {
  if (!cols) {
    static std::atomic<uint64_t> done{0}, done2{0};
    const int64_t grid = rules_grid((int64_t)a.Z * a.H, a.R);
    if constexpr (2 * pair_lds<T, D, X, 2>() <= kLdsBytes)
      if (few_lines<T, D, X>(a)) return rules_launch(k_rules_bwd_rows<T, D, X, CAP, BIAS, DOCS, 2>, grid, 256, 2 * pair_lds<T, D, X, 2>(), done2, a, st);
    return rules_launch(k_rules_bwd_rows<T, D, X, CAP, BIAS, DOCS, 1>, grid, 128, rules_lds<T, D, X>(), done, a, st);
  }
  static std::atomic<uint64_t> done{0};
  const int rc = rules_launch(k_rules_bwd_cols<T, D, X, CAP, BIAS, DOCS>, rules_grid((int64_t)a.Z * (a.H / a.G), a.R), 128, rules_lds<T, D, X>(), done, a, st);
  if (rc != BSP_OK) return rc;
  if (a.n_split > 0)
    hipLaunchKernelGGL((k_rules_bwd_cols_sum<T, D, X>), dim3((unsigned)((int64_t)a.Z * a.n_split * (64 * (2 * D + X) / 4 / 256))), dim3(256), 0, st, a);
  return BSP_OK;
}
template <typename T, int D, int X, bool CAP, bool BIAS> int launch_rules_bwd(const RuleArgs &a, bool cols, hipStream_t st) {
  return a.docs ? launch_rules_bwd<T, D, X, CAP, BIAS, true>(a, cols, st) : launch_rules_bwd<T, D, X, CAP, BIAS, false>(a, cols, st);
}
template <typename T, int D, int X> int launch_rules_bwd(const RuleArgs &a, bool cols, hipStream_t st) {
  if (a.capped) return a.slopes ? launch_rules_bwd<T, D, X, true, true>(a, cols, st) : launch_rules_bwd<T, D, X, true, false>(a, cols, st);
  return a.slopes ? launch_rules_bwd<T, D, X, false, true>(a, cols, st) : launch_rules_bwd<T, D, X, false, false>(a, cols, st);
}
template <int X> int launch_rules_bwd(int dtype, int D, const RuleArgs &a, bool cols, hipStream_t st) {
  if (dtype == BSP_F16) return D == 64 ? launch_rules_bwd<f16, 64, X>(a, cols, st) : launch_rules_bwd<f16, 128, X>(a, cols, st);
  if (dtype == BSP_BF16) return D == 64 ? launch_rules_bwd<bf16, 64, X>(a, cols, st) : launch_rules_bwd<bf16, 128, X>(a, cols, st);
  return D == 64 ? launch_rules_bwd<float, 64, X>(a, cols, st) : launch_rules_bwd<float, 128, X>(a, cols, st);
}

}  // namespace
}  // namespace bsp
#endif
