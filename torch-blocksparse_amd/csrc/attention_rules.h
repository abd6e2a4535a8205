// Shared pieces of the attention kernels with score rules (attention_rules_fwd.hip, attention_rules_bwd.hip): block-sparse
// attention whose logits are
//     y_ij = cap * tanh(scale * q_i . k_j / cap) - slope_h * |i - j|        (no cap: scale * q_i . k_j - ...)
// over the keys j that row i sees: block (h, i / block, j / block) is in the layout, both positions carry the same document
// number and it is not negative, and without `causal` any j, with it j <= i or j < prefix of the batch.  q has G heads for each
// head of k and v.  The length need not fill the last block.  A row that sees no key gets zeros, in the result and as gradient.
//
// The tiles, the work split and the LDS ring are those of attention_quad.h: a workgroup of two wavefronts has the 64 rows of a line
// (keys of a column) and walks the line's (column's) tiles in halves of 32 columns (rows).  What the rules add:
//   * a walk (Walk): 64 halves at a time, one a lane, are held against the rules by their positions and the range of document numbers
//     in each group of sixteen positions; three lane masks say which halves any row sees, which every row sees whole, and
//     which hold positions without document.  The loop visits the first kind only, and looks at single scores
//     in those of them that are not of the second.
//   * a score is seen or not by a bit of a sixteen-bit word per lane.  What the position rules leave of a lane's two runs of
//     eight consecutive keys is a run itself, so the word is two shifts; documents are compared one by one.
//   * positions without document (padding) may hold anything, NaN included: their rows of a stage are set to zero before the
//     products (0 * NaN would reach every row of the tile).  Positions past the end are loaded as zeros: operands are fetched
//     through buffer descriptors that end with the head's last row.
// fp32: the same kernels on the fp32 matrix units (32x32x2), which take their operands as they lie in a row: no transposing reads.
#ifndef BSP_ATTENTION_RULES_H
#define BSP_ATTENTION_RULES_H
#include "attention_quad.h"

namespace bsp {

struct RuleArgs {
  const void *q, *k, *v;
  const void *d_o, *o_in;          // backward: do, and the forward result (row kernel)
  void *o, *o2;                    // forward: o; row kernel: dq; column kernel: dk and dv
  void *o_rest;                    // [Z][H][L][D]: what the rounding of o to a 16-bit type left out
  float *ref, *delta;              // ref: [Z][H][2][rows]: p = exp2(y - ref) * factor, y in the log2 domain; delta: [Z][H][rows], -sum_d do . o
  int64_t rows;                    // 64 * lines
  int64_t q_sz, q_sh, q_ld, k_sz, k_sh, k_ld, v_sz, v_sh, v_ld, do_sz, do_sh, do_ld, oin_sz, oin_sh, oin_ld;
  int64_t o_sz, o_sh, o_ld, o2_sz, o2_sh, o2_ld;
  float in, out;                   // y = out * tanh(in * s / 2) with a cap, s * out without
  float scale;                     // of the sums dq and dk
  const float *slopes;
  const int32_t *docs; int64_t docs_sz;
  const int32_t *prefix;
  const int32_t *ranges; int groups;   // per batch and group of sixteen positions the least and the greatest document number (least: -1 if any is negative)
  int causal, capped;
  const int32_t *lut;
  float *partial;                  // column kernel: slots of the parts of long columns, [Z][n_slots][dk, dv][64][D]
  const int32_t *split_lut;
  int n_slots, n_split;
  int Z, H, G, R, L;               // G: query heads a key head; R: lines of the table per head, 64 R >= L (column kernel: work items of a key head)
};

namespace {

template <typename T, int D> struct Geo {
  static constexpr int ESZ = sizeof(T), RB = D * ESZ, CPR = RB / 16, NF = RB / 32, VEC = 16 / ESZ;   // bytes and 16-byte chunks of a row; operand fragments; elements a chunk
  static constexpr int PIECE = 32 * RB, STAGE = 2 * PIECE, RING = 2 * STAGE;
  static constexpr int EXTRA = 768;                      // bytes behind each stage's pieces: documents, statistics
};
template <typename T> struct RuleOperand { typedef typename Mma<T, 32>::frag_t type; };
template <> struct RuleOperand<float> { typedef f32x4 type; };
template <typename T, int D> using held_t = typename RuleOperand<T>::type[Geo<T, D>::NF];

template <typename T, int D> __device__ __forceinline__ int rule_swz(int r) {
  if constexpr (sizeof(T) == 4) return r & 15;
  else return quad_swz<D>(r);
}

// The lane's row of an operand that stays in registers: chunk 2 s + lane / 32 of it, or zeros
template <typename T, int D> __device__ __forceinline__ void hold_operand(held_t<T, D> &f, const T *row, int half, bool dead) {
#pragma unroll
  for (int s = 0; s < Geo<T, D>::NF; s++) {
    const u32x4 raw = *reinterpret_cast<const u32x4 *>(row + Geo<T, D>::VEC * (2 * s + half));
    f[s] = __builtin_bit_cast(typename RuleOperand<T>::type, dead ? u32x4{0, 0, 0, 0} : raw);
  }
}

// `bytes` bytes from p on as a buffer: loads from behind it give zeros
typedef int i32x4r __attribute__((ext_vector_type(4)));
__device__ __forceinline__ i32x4r buffer_of(const void *p, int64_t bytes) {
  const uint64_t at = reinterpret_cast<uint64_t>(p);
  return i32x4r{(int)(uint32_t)at, (int)(uint32_t)(at >> 32) & 0xffff, (int)(uint32_t)bytes, 0x00020000};
}
// the rows of a head: row stride ld and `length` rows of D elements
template <typename T, int D> __device__ __forceinline__ i32x4r rows_buffer(const T *p, int64_t ld, int length) { return buffer_of(p, ((length - 1) * ld + D) * (int64_t)sizeof(T)); }
// the same length from another place
__device__ __forceinline__ i32x4r move_buffer(const i32x4r &b, const char *p) { return i32x4r{(int)(uint32_t)reinterpret_cast<uint64_t>(p), (int)(uint32_t)(reinterpret_cast<uint64_t>(p) >> 32) & 0xffff, b[2], b[3]}; }
// load_to_lds from a buffer
template <int BYTES> __device__ __forceinline__ void buffer_to_lds(const i32x4r &rsrc, uint32_t off, uint32_t add, uint32_t dst) {
  uint32_t at;                                            // (the addition also is the instruction that must lie between m0 and its use)
  if constexpr (BYTES == 16) asm volatile("s_mov_b32 m0, %4\n\tv_add_u32 %0, %2, %1\n\tbuffer_load_dwordx4 %0, %3, 0 offen lds" : "=&v"(at) : "v"(off), "s"(add), "s"(rsrc), "s"(dst) : "m0", "memory");
  else asm volatile("s_mov_b32 m0, %4\n\tv_add_u32 %0, %2, %1\n\tbuffer_load_dword %0, %3, 0 offen lds" : "=&v"(at) : "v"(off), "s"(add), "s"(rsrc), "s"(dst) : "m0", "memory");
}

// Sixteen consecutive rows, global -> LDS.  Rows behind the last one come as zeros.
template <typename T, int D, bool LEAN> struct RowsLoad {
  typedef Geo<T, D> Q;
  static constexpr int RPL = 64 / Q::CPR, LW = 16 / RPL;
  uint32_t off[LEAN ? 1 : LW];
  uint32_t chunk;
  __device__ __forceinline__ void init(int64_t ld, int lane) {
    chunk = (uint32_t)((lane % Q::CPR) ^ rule_swz<T, D>(lane / Q::CPR));
#pragma unroll
    for (int i = 0; i < (LEAN ? 1 : LW); i++)
      off[i] = (uint32_t)((i * RPL + lane / Q::CPR) * ld) * Q::ESZ + (LEAN ? 0u : (chunk ^ (uint32_t)rule_swz<T, D>(i * RPL)) << 4);
  }
  __device__ __forceinline__ void issue(const i32x4r &rows, int pos, uint32_t row_bytes, uint32_t lds) const {
    uint32_t c = chunk;
    if constexpr (LEAN) asm volatile("" : "+v"(c));
#pragma unroll
    for (int i = 0; i < LW; i++)
      if constexpr (LEAN) buffer_to_lds<16>(rows, off[0] + ((c ^ (uint32_t)rule_swz<T, D>(i * RPL)) << 4), (uint32_t)(pos + i * RPL) * row_bytes, lds + i * 1024);
      else buffer_to_lds<16>(rows, off[i], (uint32_t)pos * row_bytes, lds + i * 1024);
  }
};

// Those of sixteen rows (from row0 on) of a piece whose positions carry no document: zeros
template <typename T, int D> __device__ __forceinline__ void clear_rows(unsigned char *piece, int row0, const int32_t *docs_of_stage, int lane) {
  typedef Geo<T, D> Q;
  constexpr int RPL = 64 / Q::CPR;
#pragma unroll 1
  for (int i = 0; i < 16 / RPL; i++) {
    const int r = row0 + i * RPL + lane / Q::CPR;
    if (docs_of_stage[r] < 0) *reinterpret_cast<u32x4 *>(piece + r * Q::RB + (lane % Q::CPR) * 16) = u32x4{0, 0, 0, 0};
  }
}

// The operand reads of a piece, along its rows and transposed: LDS addresses in the piece at offset 0.  (Reads go through pointers to LDS made of them, so
// that a stage's offset is a constant of the instruction; from a generic pointer each read costs an addition.)
template <typename T, int D, bool LEAN> struct PieceReads {
  RowReads<D, LEAN> rows;
  TrReads<D, LEAN> tr;
  __device__ __forceinline__ void init(const unsigned char *smem, int lane) {
    rows.init(0, lane);
#pragma unroll
    for (int s = 0; s < (LEAN ? 1 : D / 16); s++) rows.a[s] += lds_address(smem);
    tr.init(lds_address(smem), 0, lane);
  }
};
template <int D, bool LEAN> struct PieceReads<float, D, LEAN> {
  uint32_t row, tr;                // the others are an exclusive-or of constants away
  __device__ __forceinline__ void init(const unsigned char *smem, int lane) {
    const int half = lane >> 5, l32 = lane & 31, r = deal_row(l32);
    row = lds_address(smem) + (uint32_t)(r * Geo<float, D>::RB + ((half ^ rule_swz<float, D>(r)) << 4));
    tr = lds_address(smem) + (uint32_t)(8 * half * Geo<float, D>::RB + (((l32 >> 2) ^ (8 * half)) << 4) + ((l32 & 3) << 2));
  }
};
template <typename V> __device__ __forceinline__ V lds_read(uint32_t at) { return *(const V __attribute__((address_space(3))) *)(uintptr_t)at; }

// The operand fragment of chunk s of the lane's row, and the product with it
template <typename T, int D, int OFF, bool LEAN>
__device__ __forceinline__ typename RuleOperand<T>::type row_fragment(const PieceReads<T, D, LEAN> &reads, int s) {
  uint32_t at;
  if constexpr (sizeof(T) == 4) at = reads.row ^ (uint32_t)(s << 5);
  else if constexpr (LEAN) at = reads.rows.a[0] ^ (uint32_t)(s << 5);
  else at = reads.rows.a[s];
  return lds_read<typename RuleOperand<T>::type>(at + OFF);
}
template <typename T> __device__ __forceinline__ f32x16 fragment_times(const typename RuleOperand<T>::type &f, const typename RuleOperand<T>::type &b, f32x16 acc) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 4; j++) acc = Mma<float, 32>::run(f[j], b[j], acc);
    return acc;
  } else {
    return Mma<T, 32>::run(f, b, acc);
  }
}
// acc + (32 rows of a piece, dealt by deal_row) . b: value i = row 16 (i / 8) + 8 (lane / 32) + i % 8 of the piece, column lane % 32
template <typename T, int D, int OFF, bool LEAN>
__device__ __forceinline__ f32x16 rows_times(PieceReads<T, D, LEAN> reads, const held_t<T, D> &b, f32x16 acc) {
  if constexpr (LEAN && sizeof(T) == 2) asm volatile("" : "+v"(reads.rows.a[0]));   // (the others are made when they are wanted, not held)
  typename RuleOperand<T>::type f[Geo<T, D>::NF];
#pragma unroll
  for (int s = 0; s < Geo<T, D>::NF; s++) f[s] = row_fragment<T, D, OFF, LEAN>(reads, s);
#pragma unroll
  for (int s = 0; s < Geo<T, D>::NF; s++) acc = fragment_times<T>(f[s], b[s], acc);
  return acc;
}
__device__ __forceinline__ f32x16 zeros16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; i++) z[i] = 0.f;
  return z;
}

// Sixteen values a lane, one per row of a piece as rows_times deals them, as the operand of columns_times: rounded to the
// operands' type (the products take no other; the two-term form that loses nothing is twice the products), in fp32 as they are.  The forward pass has its shares
// relative to the running maximum, the backward pass normalised ones: in fp16 those below 2^-14 are off by up to 2^-25, as every fp16 number.
template <typename T> struct Shares {
  typename Mma<T, 32>::frag_t f[2];
  __device__ __forceinline__ void set(const float (&e)[16]) {
#pragma unroll
    for (int ks = 0; ks < 2; ks++) f[ks] = pack8<T>(reinterpret_cast<const float (&)[8]>(e[8 * ks]));
  }
};
template <> struct Shares<float> {
  float e[16];
  __device__ __forceinline__ void set(const float (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 16; i++) e[i] = v[i];
  }
};

// acc[mt] += (32 rows of a piece, transposed)[column 32 mt ..][row] . b[row]
template <typename T, int D, int OFF, bool LEAN>
__device__ __forceinline__ void columns_times(f32x16 (&acc)[D / 32], const PieceReads<T, D, LEAN> &reads, const Shares<T> &b) {
  if constexpr (sizeof(T) == 4) {
    constexpr int RB = Geo<T, D>::RB;
#pragma unroll
    for (int i = 0; i < 16; i++)
#pragma unroll
      for (int mt = 0; mt < D / 32; mt++) {
        const float x = lds_read<float>((reads.tr ^ (uint32_t)((8 * mt ^ (i & 7)) << 4)) + OFF + (16 * (i / 8) + i % 8) * RB);
        acc[mt] = Mma<float, 32>::run(x, b.e[i], acc[mt]);
      }
  } else {
    tr_product<T, D, OFF, LEAN>(acc, reads.tr, b.f);
  }
}

// ... + (32 rows of a piece, transposed) . e for sixteen values a lane in two operands, what they are rounded to and what that leaves out: as exact as
// products of fp32 numbers, for half as many products again
template <typename T, int D, int OFF, bool LEAN>
__device__ __forceinline__ void columns_times_exact(f32x16 (&acc)[D / 32], const PieceReads<T, D, LEAN> &reads, float (&e)[16]) {
  typedef Mma<T, 32> M;
  Shares<T> most, rest;
  most.set(e);
#pragma unroll
  for (int i = 0; i < 16; i++) e[i] -= to_float(most.f[i >> 3][i & 7]);
  rest.set(e);
  uint32_t lo[D / 32], hi[D / 32];
  reads.tr.get(lo, hi);
#pragma unroll
  for (int mt = 0; mt < D / 32; mt += 2) {
    constexpr int HI = LEAN ? 4 * 2 * D : 0;
    typename M::frag_t f[4];
#pragma unroll
    for (int i = 0; i < 4; i++) f[i] = tr_fragment<T>(lo[mt + (i & 1)] + OFF + (i >> 1) * (16 * 2 * D), hi[mt + (i & 1)] + OFF + HI + (i >> 1) * (16 * 2 * D));
#pragma unroll
    for (int i = 0; i < 4; i++) acc[mt + (i & 1)] = M::run(f[i], most.f[i >> 1], acc[mt + (i & 1)]);
#pragma unroll
    for (int i = 0; i < 4; i++) acc[mt + (i & 1)] = M::run(f[i], rest.f[i >> 1], acc[mt + (i & 1)]);
  }
}

// Capped scores.  With x = scale * s / cap, tanh(x) = 1 - 2 r and 1 - tanh(x)^2 = 4 (r - r^2), r = 1 / (exp(2 x) + 1): the kernels for 16-bit
// types keep r, whose error of 2^-24 cap * log2 e takes to the logit: little beside what the operands' rounding leaves of it.  In fp32 they keep
// the tanh, from its series where x is small (in trained models nearly everywhere) with its relative precision: up to x = 0.45 the
// next term is below 2^-27 of the sum.
template <typename T> __device__ __forceinline__ float cap_score(float s, float in) {
  const float r = __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(s * (in * kLog2e)) + 1.f);
  if constexpr (sizeof(T) == 4) {
    const float x = 0.5f * in * s, z = x * x;
    float p = fmaf(z, 21844.f / 6081075.f, -1382.f / 155925.f);
    p = fmaf(z, p, 62.f / 2835.f);
    p = fmaf(z, p, -17.f / 315.f);
    p = fmaf(z, p, 2.f / 15.f);
    p = fmaf(z, p, -1.f / 3.f);
    return z < 0.2025f ? fmaf(x * z, p, x) : fmaf(-2.f, r, 1.f);
  }
  return r;
}
// 1 - tanh^2 of what cap_score gives, or (QUARTER, 16-bit types) a quarter of it, which is one operation less
template <typename T, bool QUARTER> __device__ __forceinline__ float cap_through(float c) {
  if constexpr (sizeof(T) == 4) return fmaf(-c, c, 1.f);
  else if constexpr (QUARTER) return fmaf(-c, c, c);
  else return fmaf(-4.f * c, c, 4.f * c);
}
// the logit of a score s (or of what cap_score gives) is s * factor + shift
template <typename T, bool CAP> __device__ __forceinline__ float logit_factor(float out) { return CAP && sizeof(T) != 4 ? -2.f * out : out; }
template <typename T, bool CAP> __device__ __forceinline__ float logit_shift(float out) { return CAP && sizeof(T) != 4 ? out : 0.f; }
inline void logit_args(RuleArgs &a, float scale, float cap) {
  a.scale = scale;
  a.capped = cap > 0.f;
  a.in = cap > 0.f ? 2.f * scale / cap : 0.f;
  a.out = (cap > 0.f ? cap : scale) * kLog2e;
}

// A value that is the same in all lanes, in scalar registers of its own.  Arguments are loaded sixteen dwords at a time, and as long as one
// of them is used in a loop all sixteen are kept, spilled to lanes of vector registers and read back there: thirty of the instructions of a step.
template <typename V> __device__ __forceinline__ V apart(V v) {
  constexpr int N = sizeof(V) / 4;
  struct Words { int w[N]; };
  Words x = __builtin_bit_cast(Words, v);
#pragma unroll
  for (int i = 0; i < N; i++) {
    int w;
    // (the unit waits for neither side by itself: the lane's value may have been written by the instruction before, and any unit may read
    // the scalar register next)
    asm volatile("s_nop 1\n\tv_readfirstlane_b32 %0, %1\n\ts_nop 4" : "=s"(w) : "v"(x.w[i]));
    x.w[i] = w;
  }
  return __builtin_bit_cast(V, x);
}

// The least and greatest document number of a group of sixteen positions
struct Range { int lo, hi; };
struct Ranges {
  const int32_t *of_batch;
  int last;
  __device__ __forceinline__ void init(const RuleArgs &a, int z) {
    of_batch = apart(a.ranges + 2 * (int64_t)z * a.groups);
    last = apart(a.groups - 1);
  }
  __device__ __forceinline__ Range at(int pos) const {
    const int g = pos >> 4;
    const int32_t *r = of_batch + 2 * (g < last ? g : last);
    return Range{r[0], r[1]};
  }
};

// The halves of a line's (column's) tiles that are worth a visit, 64 looked at together, one a lane.  From the last to the first: in a
// causal layout the nearest keys come first then, whose logits a bias by distance makes the largest, so that the running maximum is found at
// once (from the first on it moves in two steps of three: 221 us for the forward pass of fp16 8 x 16 x 4096 over the layout of blocks of
// 16 with stride 64).
struct Half { int n, lo, hi, bits; bool full, pad; };
template <bool DOCS> struct Walk {
  const int32_t *core;
  int base;
  uint64_t live, full, pad;
  int v_lo, v_hi, v_bits;
  __device__ __forceinline__ void init(const int32_t *entries, int halves) {
    core = entries;
    base = halves;                 // halves at and above it are done
    live = 0;
  }
  // look(lo, hi, bits of the half's pieces, which half of its tile, &full, &pad) -> does any row see anything of it
  template <class F> __device__ __forceinline__ Half next(int lane, F &&look) {
    while (live == 0) {
      if (base <= 0) return Half{-1, 0, 0, 0, false, false};
      const int end = base;
      base = base > 64 ? base - 64 : 0;
      const int n = base + lane, at = n < end ? n : end - 1;
      const int32_t *e = core + kEntry * (at >> 1);
      v_lo = e[2 * (at & 1)];
      v_hi = e[2 * (at & 1) + 1];
      v_bits = e[4];
      bool f = false, p = false;
      const bool l = look(v_lo, v_hi, v_bits, at & 1, f, p);
      live = __builtin_amdgcn_ballot_w64(l && n < end);
      full = __builtin_amdgcn_ballot_w64(f);
      if constexpr (DOCS) pad = __builtin_amdgcn_ballot_w64(p);
    }
    const int j = 63 - __builtin_clzll(live);
    live &= ~((uint64_t)1 << j);
    return Half{base + j, __builtin_amdgcn_readlane(v_lo, j), __builtin_amdgcn_readlane(v_hi, j), __builtin_amdgcn_readlane(v_bits, j),
                (bool)((full >> j) & 1), DOCS && (bool)((pad >> j) & 1)};
  }
};

// The rules as the row kernels (a line of 64 rows; the lane has row `row`) apply them
template <bool DOCS> struct LineRules {
  int most, least;                 // the keys below `most` are seen by a row of the line, those below `least` by all, as far as positions go
  int limit;                       // ... the keys below it by the lane's row
  int doc;                         // the lane's document
  Range range;                     // of the line
  Ranges ranges;
  __device__ __forceinline__ void init(const RuleArgs &a, int z, int line, int row, bool &dead) {
    const int prefix = a.causal && a.prefix ? as_table(a.prefix)[z] : 0, first = line * 64;
    doc = 0;
    if constexpr (DOCS) {
      ranges.init(a, z);
      doc = a.docs[z * a.docs_sz + (row < a.L ? row : a.L - 1)];
      const int lane = threadIdx.x & 3;
      const Range g = ranges.at(first + 16 * lane < a.L ? first + 16 * lane : first);
      int lo = g.lo, hi = g.hi;
#pragma unroll
      for (int d = 1; d < 4; d <<= 1) {
        const int ol = __shfl_xor(lo, d), oh = __shfl_xor(hi, d);
        lo = ol < lo ? ol : lo;
        hi = oh > hi ? oh : hi;
      }
      range = Range{__builtin_amdgcn_readfirstlane(lo), __builtin_amdgcn_readfirstlane(hi)};
    }
    dead = row >= a.L || doc < 0;
    auto below = [&](int i) { const int n = a.causal ? (i + 1 > prefix ? i + 1 : prefix) : a.L; return n < a.L ? n : a.L; };
    most = apart(below(first + 63));
    least = apart(below(first));
    limit = dead ? 0 : below(row);
  }
  __device__ __forceinline__ bool look(int lo, int hi, int bits, int half, bool &full, bool &pad) const {
    bits >>= 2 * half;
    bool see_lo = (bits & 0x1111) && lo < most, see_hi = (bits & 0x2222) && hi < most;
    full = (bits & 0x3333) == 0x3333 && lo + 15 < least && hi + 15 < least;
    if constexpr (DOCS) {
      const Range x = ranges.at(lo), y = ranges.at(hi);
      const int from = range.lo < 0 ? 0 : range.lo;
      see_lo = see_lo && x.hi >= from && x.lo <= range.hi;
      see_hi = see_hi && y.hi >= from && y.lo <= range.hi;
      full = full && range.lo == range.hi && x.lo == range.lo && x.hi == range.lo && y.lo == range.lo && y.hi == range.lo;
      pad = x.lo < 0 || y.lo < 0;
    }
    return see_lo || see_hi;
  }
};

// floats that are the same in all lanes, read as table_ptr reads tables
typedef const float __attribute__((address_space(4))) *floats_ptr;
__device__ __forceinline__ floats_ptr as_floats(const float *p) { return (floats_ptr)p; }

// Logits of the lane's sixteen scores less `minus`: s * out - slope * distance - minus, the scores of run g at distances |at_g - i|, i = 0 .. 7.
// Where a wavefront's scores all lie on one side of the diagonal (nearly everywhere) the distances are at_g - i or its negative, and
// one multiply-add more than without a bias is enough.
template <bool BIAS> struct Logits {
  float base[2], slope[2];
  bool straight;
  __device__ __forceinline__ Logits(int at_lo, int at_hi, float s) : Logits(at_lo, at_hi, s, s) {}
  __device__ __forceinline__ Logits(int at_lo, int at_hi, float s_lo, float s_hi) {
    if constexpr (BIAS) {
      const int least = at_lo < at_hi ? at_lo : at_hi, most = at_lo < at_hi ? at_hi : at_lo;
      const bool past = __builtin_amdgcn_ballot_w64(least < 7) == 0;        // every distance is at - i
      straight = past || __builtin_amdgcn_ballot_w64(most > 0) == 0;
      base[0] = (float)at_lo;
      base[1] = (float)at_hi;
      slope[0] = s_lo;
      slope[1] = s_hi;
      if (straight) {
        const float sign = past ? 1.f : -1.f;
#pragma unroll
        for (int g = 0; g < 2; g++) slope[g] *= sign, base[g] *= -slope[g];
      }
    }
  }
  // y(i) for i = 0 .. 15, minus(i) a value per score (a constant, usually)
  template <class S, class M> __device__ __forceinline__ void get(float (&y)[16], const S &s, float out, M &&minus) const {
    if constexpr (!BIAS) {
#pragma unroll
      for (int i = 0; i < 16; i++) y[i] = fmaf(s[i], out, -minus(i));
    } else if (straight) {
#pragma unroll
      for (int i = 0; i < 16; i++) y[i] = fmaf(s[i], out, fmaf(slope[i >> 3], (float)(i & 7), base[i >> 3] - minus(i)));
    } else {
#pragma unroll
      for (int i = 0; i < 16; i++) y[i] = fmaf(s[i], out, fmaf(-slope[i >> 3], fabsf(base[i >> 3] - (float)(i & 7)), -minus(i)));
    }
  }
};

// the lowest n of eight bits, n any number
__device__ __forceinline__ uint32_t first_bits(int n) { return (1u << (n < 0 ? 0 : n > 8 ? 8 : n)) - 1u; }
// all ones where bit i of the word is set, else zero; what is `and`ed with it is kept or becomes zero, whatever it is, NaN too.  (As assembly: the
// compiler makes a test and a selection of it, three operations and a wait.)
template <int I> __device__ __forceinline__ uint32_t bit_mask(uint32_t word) {
  uint32_t m;
  asm("v_bfe_i32 %0, %1, %2, 1" : "=v"(m) : "v"(word), "n"(I));
  return m;
}
__device__ __forceinline__ float keep(float v, uint32_t mask) { return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, v) & mask); }
// the bits of the word whose documents (eight and eight consecutive ones) are not the lane's taken out
__device__ __forceinline__ uint32_t same_document(uint32_t word, const int32_t *docs, int doc) {
  typedef int i32x4v __attribute__((ext_vector_type(4)));
#pragma unroll
  for (int g = 0; g < 4; g++) {
    const i32x4v d = *reinterpret_cast<const i32x4v *>(docs + 16 * (g >> 1) + 4 * (g & 1));
#pragma unroll
    for (int i = 0; i < 4; i++) word &= d[i] == doc ? ~0u : ~(1u << (4 * g + i));
  }
  return word;
}

// the documents of a half's 32 positions to LDS, twice (64 lanes)
__device__ __forceinline__ void load_documents(const i32x4r &docs, int lo, int hi, int lane, uint32_t dst) {
  buffer_to_lds<4>(docs, (uint32_t)((lane & 16 ? hi : lo) + (lane & 15)) * 4u, 0, dst);
}

// acc[mt][4g + e] = out[row][32 mt + 8 g + 4 (lane / 32) + e], row = lane % 32 of 32 rows: those of lo (16, of which the first n_lo
// exist) and hi, through the wavefront's piece of LDS to stores of whole rows
template <typename T, int D> __device__ __forceinline__ void store_some_rows(unsigned char *piece, T *lo, int n_lo, T *hi, int n_hi, int64_t ld, const f32x16 (&acc)[D / 32], int lane) {
  typedef Geo<T, D> Q;
  T *stage = reinterpret_cast<T *>(piece);
  constexpr int LDS = D + Q::VEC;
#pragma unroll
  for (int mt = 0; mt < D / 32; mt++)
#pragma unroll
    for (int g = 0; g < 4; g++) {
      T *at = stage + (lane & 31) * LDS + 32 * mt + 8 * g + 4 * (lane >> 5);
      if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<f32x4 *>(at) = f32x4{acc[mt][4 * g], acc[mt][4 * g + 1], acc[mt][4 * g + 2], acc[mt][4 * g + 3]};
      } else {
        union { u32x2 raw; T e[4]; } pk;
#pragma unroll
        for (int e = 0; e < 4; e++) pk.e[e] = from_float<T>(acc[mt][4 * g + e]);
        *reinterpret_cast<u32x2 *>(at) = pk.raw;
      }
    }
  __builtin_amdgcn_wave_barrier();   // LDS operations of one wavefront complete in order; this only pins the code order
  constexpr int RPS = 64 / Q::CPR;   // rows per store
#pragma unroll
  for (int i = 0; i < 32 / RPS; i++) {
    const int r = i * RPS + lane / Q::CPR, ch = lane % Q::CPR;
    const bool low = i * RPS < 16;
    if ((low ? r < n_lo : r - 16 < n_hi)) {
      T *dst = (low ? lo + (int64_t)r * ld : hi + (int64_t)(r - 16) * ld) + Q::VEC * ch;
      __builtin_nontemporal_store(*reinterpret_cast<const u32x4 *>(stage + r * LDS + Q::VEC * ch), reinterpret_cast<u32x4 *>(dst));
    }
  }
  __builtin_amdgcn_wave_barrier();
}
template <typename T, int D> constexpr int rules_lds() {
  constexpr int ring = Geo<T, D>::RING + 2 * Geo<T, D>::EXTRA, out = 64 * (D + Geo<T, D>::VEC) * Geo<T, D>::ESZ;
  return ring > out ? ring : out;
}

// A launch of few lines has two pairs of wavefronts to a line, each of which takes every other half of a tile, with a ring of its own; at the end the second
// pair's sums are added to the first's through its ring.
template <typename T, int D, int PAIRS> constexpr int pair_lds() {
  constexpr int sums = 2 * 64 * 4 * (D / 2 + 2);        // two wavefronts' accumulators, maxima and sums
  return PAIRS == 1 || rules_lds<T, D>() > sums ? rules_lds<T, D>() : sums;
}
// The halves of the pair of wavefronts `group`; more: some pair has one; pads: one of them has padding
struct Halves { Half own; bool more, pads; };
template <int PAIRS, class F> __device__ __forceinline__ Halves next_halves(int group, F &&next) {
  const Half a = next();
  if constexpr (PAIRS == 1) return Halves{a, a.n >= 0, a.pad};
  const Half b = a.n >= 0 ? next() : a;
  return Halves{group ? b : a, a.n >= 0, a.pad || b.pad};
}

// Which of n work items of which of `units` heads (all of equal cost, item 0 the longest) a workgroup does.  Workgroups go round the eight
// XCDs, each with an L2 of its own: the heads are dealt to the XCDs whole, so that a head's k and v are fetched into one L2, four heads at a
// time, their longest items first.  Heads past a multiple of eight go first, an item here, an item there: every XCD gets the same
// share of the long ones.  (One run of heads and lines cut in eight pieces gives the XCDs unequal work: the first half of a causal head's lines is three
// times the second.  Full causal attention over 8192 positions in 16 heads of 128: 595 us that way.)
struct Place { int unit, item; };
__host__ __device__ __forceinline__ int64_t rules_grid(int64_t units, int64_t n) { return (units % 8 * n + 7) / 8 * 8 + units / 8 * 8 * n; }
__device__ __forceinline__ Place rules_place(uint32_t wg, int units, int n) {
  const uint32_t rest = units & 7, spread = (rest * n + 7) & ~7u;
  if (wg < spread) {
    const Quotient p(wg, rest);
    return Place{__builtin_amdgcn_readfirstlane(p.q < (uint32_t)n ? (int)((units & ~7) + p.r) : -1), __builtin_amdgcn_readfirstlane((int)p.q)};
  }
  wg -= spread;
  const uint32_t per = units >> 3, x = wg & 7, i = wg >> 3;      // heads per XCD
  const Quotient g(i, kHeadsTogether * n);
  const uint32_t first = g.q * kHeadsTogether, heads = per - first < kHeadsTogether ? per - first : kHeadsTogether;
  const Quotient p(g.r, heads);
  return Place{__builtin_amdgcn_readfirstlane((int)(x * per + first + p.r)), __builtin_amdgcn_readfirstlane((int)p.q)};
}

// The query head and batch of a unit: the heads that share a key head next to each other, then the batches (their documents, and with them
// the cost of a head, may differ: an XCD gets some of each)
struct HeadOf {
  int h, hk, z;
  __device__ __forceinline__ HeadOf(int unit, int Z, int G) {
    const Quotient g(unit, G), b(g.q, Z);
    z = __builtin_amdgcn_readfirstlane(b.r);            // (a division's result is in a vector register, and what follows from it would be)
    hk = __builtin_amdgcn_readfirstlane(b.q);
    h = __builtin_amdgcn_readfirstlane(hk * G + g.r);
  }
};

// everybody's LDS operations are done
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Two pairs of wavefronts a line in launches of few lines, whose wavefronts would leave SIMDs idle or with nobody to change places with.  The rule knows the number
// of lines, not of their tiles (which documents and a prefix change from call to call).  Causal layouts without holes, forward pass, one pair -> two: 512 lines of 1024 positions fp32 104 -> 61 us (128 elements: 148 -> 102), bf16 24 -> 18 (34 -> 25); 1024 lines of 4096 positions
// 456 -> 318 (578 -> 642), 82 -> 63 (126 -> 104); 2048 of them 693 -> 577 (1130 -> 1261), 124 -> 116 (198 -> 217); twelve heads of 256 lines of BigBird fp16 51 -> 59.
// Short lines, of 7 tiles (BigBird): fp16 768 lines 18.0 -> 17.3, 1536 29.7 -> 31.9; bf16 of 128 elements 512 lines 22.9 -> 19.2, 1024 30.6 -> 35.6; fp32 512 lines 68.6 -> 43.3, 1024 76.8 ->
// 78.7, of 128 elements 256 74.3 -> 45.3, 512 80.2 -> 91.6; of one tile: fp16 768 lines 7.1 -> 8.1, bf16 of 128 elements 1024 14.5 -> 19.4, fp32 512 12.6 -> 11.8, of 128 elements 21.8 -> 29.0.
template <typename T, int D> inline bool few_lines(const RuleArgs &a) {
  return a.R >= 4 && (int64_t)a.Z * a.H * a.R <= (D == 64 ? 2048 : sizeof(T) == 4 ? 512 : 1024);
}
template <typename K> int rules_launch(K kernel, int64_t n_wg, int threads, int lds, std::atomic<uint64_t> &done, const RuleArgs &a, hipStream_t st) {
  if (lds > 65536 && !raise_lds_limit(reinterpret_cast<const void *>(kernel), lds, done)) return BSP_ERR_HIP;
  hipLaunchKernelGGL(kernel, dim3((unsigned)n_wg), dim3((unsigned)threads), lds, st, a);
  return BSP_OK;
}

}  // namespace

// call -> kernel arguments, checked (attention_rules_fwd.hip)
int rules_args(const bsp_attention_rules_call *c, RuleArgs &a);
}  // namespace bsp
#endif
