// Attention of one new position a sequence over a cache of latent vectors (latent.h), the absorbed form: every head's key of position j is the latent vector c_j and the
// shared part r_j, its value is c_j:
//     y_j = cap * tanh(scale * (q . c_j + q_r . r_j) / cap) - slope_h * (n - 1 - j),   o = sum_j softmax_j(y) c_j        (no cap: scale * (q . c_j + q_r . r_j) - ...)
// over the positions j < n whose page the sequence holds and, with a layout, whose block is in row (n - 1) / block of head h.
//
// Each byte of the pages is read once for all heads of a workgroup (up to 64; more are several workgroups', which read the pages again) and is key and value at once, so it goes to LDS, straight
// from global memory. A wavefront has sixteen heads.  Both products are taken transposed on the matrix units (16 x 16 x 32): scores as positions x heads, results as elements x heads.  A lane then has one head, so
// maximum, sum and rescaling are single registers, and the shares a lane has computed are the operand of the second product as they are: its other operand, positions across, comes from
// LDS by transposing reads in the same order of positions.
//
// A step of a workgroup is 64 positions: four groups of sixteen, each wavefront loads one.  With at most sixteen heads (HW = 1) each wavefront goes through groups of its own and
// needs no barrier; with up to 32 (HW = 2) two wavefronts, with more all four share their groups.
//
// All steps of all sequences are one row of work that is cut into equal pieces, one a workgroup, so that uneven lengths leave no compute unit idle: a workgroup finds its piece by
// a sum over the lengths.  A sequence that lies in several pieces is joined by a second kernel.
//
// Measured, latent vectors of 512, bf16: 16 sequences of up to 16384 positions (151 MB of pages) with 16 heads 52 us (3.8 TB/s; the join among them), 32 59, 64 72, 128 heads 109, 9.6 of them the join (47
// GFLOP; 435 TFLOP/s).  16 heads are bound by the loads of a workgroup that has one step's on its way.  64 and more: of 240000 cycles a workgroup the products' reads from LDS (17.5 MB a compute
// unit, 137000 cycles at 128 bytes a clock) and products (66000) overlap in part, the rest is a step's exponentials between them and a piece's ends: queries, sums written (33 MB, read back by the
// join), the search for the piece.  Shorter: 16 x 16 heads over up to 4096 positions with a layout, fp16, 15 and 4 us; one sequence of 33 positions 10.8.
//
// Latent vectors of 512 take all of a wavefront's 512 registers, and 16 to 48 bytes a lane are in scratch memory (smaller ones none).
//
// Wavefronts of 32 heads, two for the same heads, on 32 x 32 x 16 products take half of the reads from LDS, but exchange shares and wait for each other in every step: 128 heads 117 us, 64 85 where this
// takes 98 and 66, all of it with shares in one term.
#include "attention_common.h"
#include "latent.h"

namespace bsp {

struct LatentArgs {
  const void *q, *qr; void *o;     // [B, H, latent], [B, H, 64], [B, H, latent]
  int64_t q_sb, q_sh, qr_sb, qr_sh, o_sb, o_sh;
  const void *pages; int64_t n_pages;
  const int32_t *table; int64_t table_sb; int width;     // pages of a sequence
  const int32_t *lengths;
  const int32_t *rows;             // NULL, or per unit and block-row (first entry, then one past the last row's end), then entries of three ints: block-column, a bit for each of the unit's heads that sees it
  int n_rows;
  const float *slopes;
  float scale, cap;
  float *partial;                  // two slots a workgroup: [heads a unit][latent] sums; behind all of them [heads a unit][2] maxima and sums of shares
  int32_t *meta;                   // per item (sequence and unit) two ints: the workgroup that begins it, how many have a part (0, 1: nothing to join)
  int B, H, block, shift;          // shift: log2 of the groups of sixteen positions a block
  int most_groups;                 // the most groups of 16 positions that a sequence goes through
  int units, per, pieces;          // workgroups' heads a sequence: units of `per`; pieces of the work
};

namespace {

template <typename T> struct LatentMma;
template <> struct LatentMma<f16> {
  typedef f16x8 frag8; typedef f16x4 frag4;
  static __device__ __forceinline__ f32x4 run(frag8 a, frag8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ f32x4 run(frag4 a, frag4 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x16f16(a, b, c, 0, 0, 0); }
};
template <> struct LatentMma<bf16> {
  typedef bf16x8 frag8; typedef bf16x4 frag4;
  static __device__ __forceinline__ f32x4 run(frag8 a, frag8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ f32x4 run(frag4 a, frag4 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, a), __builtin_bit_cast(s16x4, b), c, 0, 0, 0); }
};

template <int LAT> struct LatentGeo {
  static constexpr int ROW = 2 * (LAT + kRope), LROW = 2 * LAT;               // bytes of a position, of its latent vector
  static constexpr int GROUP = 16 * ROW, STAGE = 4 * GROUP, RING = 2 * STAGE;   // sixteen positions: their latent vectors, then their shared parts
  static constexpr int JOIN = LAT + 4;                                         // floats of a head's sums when wavefronts are joined
  static constexpr int CPR = LROW / 16, RPI = 64 / CPR, LOADS = 16 / RPI + 2;   // 16-byte chunks of a latent vector, rows of a load, loads of a group
  static constexpr int STATS = RING, FACTORS = RING + 512, LDS = FACTORS + 1024;   // behind the stages: maxima and sums of 64 rows, and what each's sums are multiplied by
  static_assert(64 * JOIN * 4 <= RING && LDS <= 160 * 1024, "");
};

typedef int i32x4b __attribute__((ext_vector_type(4)));
// 16 bytes a lane from `rows` (a buffer: zeros from behind its end) to 1 KB of LDS
__device__ __forceinline__ void rows_to_lds(const i32x4b &rows, uint32_t off, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(off), "s"(rows), "s"(dst) : "m0", "memory");
}
template <typename V> __device__ __forceinline__ V latent_read(uint32_t at) { return *(const V __attribute__((address_space(3))) *)(uintptr_t)at; }
__device__ __forceinline__ s16x4 latent_read_tr(uint32_t at) {
  typedef s16x4 __attribute__((address_space(3))) * lds_ptr;
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(uintptr_t)at);
}
typedef short s16x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ s16x8 latent_read_tr2(uint32_t at, uint32_t then) { return __builtin_shufflevector(latent_read_tr(at), latent_read_tr(then), 0, 1, 2, 3, 4, 5, 6, 7); }
// a value that the compiler does not look into
__device__ __forceinline__ uint32_t own(uint32_t v) {
  asm volatile("" : "+v"(v));
  return v;
}
// sums times f, left where the matrix units have them (all at once in the other registers, they would take the place of what the loop keeps there)
template <typename V> __device__ __forceinline__ V scaled_by(V v, float f) {
  v *= f;
  asm volatile("" : "+a"(v));
  return v;
}
// shared parts in LDS: two rows fill the 256 bytes of the 64 banks
__device__ __forceinline__ uint32_t rope_chunk(uint32_t chunk, uint32_t r) { return chunk ^ (r >> 1); }

// sixteen positions as a step sees them: the first one's number in the sequence, how many count, the heads (bits, the wavefront's own) that see them
struct LatentGroup { int pos, n, mask; };
// what a score is made of
struct LatentScores { float factor, cap; bool capped, sloped; int last; };   // last: the new position
// N logits, in the log2 domain, less `minus`: one multiply-add each where there is neither a cap nor a bias.  pos(i): the position of score i
template <int N, class S, class P> __device__ __forceinline__ void latent_logits(float (&y)[N], S &&score, const LatentScores &c, float slope, float minus, P &&pos) {
  if (!c.capped && !c.sloped) {
#pragma unroll
    for (int i = 0; i < N; i++) y[i] = fmaf(score(i), c.factor, -minus);
    return;
  }
#pragma unroll
  for (int i = 0; i < N; i++) y[i] = score(i) * c.factor;
  if (c.capped)
#pragma unroll
    for (int i = 0; i < N; i++) y[i] = c.cap * fmaf(-2.f, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(y[i]) + 1.f), 1.f);
#pragma unroll
  for (int i = 0; i < N; i++) y[i] = fmaf(-slope, (float)(c.last - pos(i)), y[i]) - minus;
}
// the lowest n of four bits, n any number
__device__ __forceinline__ uint32_t first_of_four(int n) { return (1u << (n < 0 ? 0 : n > 4 ? 4 : n)) - 1u; }

// The operands of both products come from LDS a batch of four reads at a time while the products of batches before are taken; left alone, the compiler reads one and waits for it, to save registers.  Every
// batch also issues its part of the next step's loads (load(k)): all at once they would hold up the wavefront for the time that a compute unit takes for them, 64 bytes a clock.
//
// Sixteen heads a wavefront, each wavefront HW of a step's groups.  Shares go into the product in two terms, what they are rounded to and what that leaves out: with the first alone a sum is off by half a step
// of the type times the sum of its terms' sizes, which nothing bounds where latent vectors cancel (128 heads 98 us with the first alone, 109 with both, 64 65 and 72; errors against 64 bits 1.94 and 1.65 in 1000 in bf16, 2.3 and 2.1 in 10000 in fp16, where
// rounding the results alone is the second).  The chunks of a latent vector in LDS: every row
// begins in the first bank, so pairs of chunks of 256 bytes are exchanged by the row's number, which serves both reads without a conflict: a transposing read takes a pair from each of
// eight rows at a time, a read along the rows a chunk of eight rows and its neighbour of the eight others.
template <typename T, int LAT, int HW> struct Heads {
  typedef LatentGeo<LAT> G;
  typedef LatentMma<T> M;
  typedef typename M::frag8 frag8;
  typedef typename std::conditional<HW == 1, typename M::frag4, frag8>::type frag;
  static constexpr int GROUPS = HW, SOURCES = 4 / HW, NS = LAT / 32, NR = kRope / 32, NT = LAT / 16;
  static constexpr int EXTRA = 4;                       // steps that going over to another item takes as long as
  static constexpr bool BARRIER = HW > 1;
  static __device__ __forceinline__ uint32_t chunk(uint32_t c, uint32_t r) { return c ^ (r & 7) << 1; }
  static __device__ __forceinline__ int first_group(int wave) { return wave / HW * HW; }
  static __device__ __forceinline__ int head_of(int wave, int lane) { return 16 * (wave % HW) + (lane & 15); }
  static __device__ __forceinline__ int mask(int wave, int lo, int hi) { return (HW == 4 && wave & 2 ? hi : lo) >> (HW > 1 ? 16 * (wave & 1) : 0); }
  // the rows that have what wavefronts found of head h
  static __device__ __forceinline__ int source(int h, int p) { return 16 * (p * HW + h / 16) + h % 16; }

  frag8 q[NS + NR];
  f32x4 o[NT];
  float m, l, slope, scaled;
  uint32_t row_at, rope_at, tr_at;                      // in a group: the lane's row (positions across the matrix rows), and of the transposing reads
  int key, c;
  bool here;

  __device__ __forceinline__ void init(const T *pq, const T *pr, bool here_, float slope_, int lane) {
    key = lane & 15; c = lane >> 4; here = here_; slope = slope_;
#pragma unroll
    for (int s = 0; s < NS + NR; s++) {
      const T *from = s < NS ? pq + 32 * s : pr + 32 * (s - NS);
      q[s] = __builtin_bit_cast(frag8, here ? *reinterpret_cast<const u32x4 *>(from + 8 * c) : u32x4{0, 0, 0, 0});
    }
    row_at = key * G::LROW + (chunk(c, key) << 4);
    rope_at = 16 * G::LROW + key * (2 * kRope) + (rope_chunk(c, key) << 4);
    const uint32_t r = 4 * c + (key >> 2);
    tr_at = r * G::LROW + (chunk((key & 3) >> 1, r) << 4) + 8 * (key & 1);
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int n = 0; n < NT; n++) o[n] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // the queries are here (looked at in the loop, the compiler would wait there for all loads of the next step)
  __device__ __forceinline__ void arrived() {
#pragma unroll
    for (int s = 0; s < NS + NR; s++) asm volatile("" : "+v"(q[s]));
  }

  // false: the sums are to be scaled first, then the step taken again
  template <class F> __device__ __forceinline__ bool step(uint32_t stage_of_all, const LatentGroup (&now)[GROUPS], const LatentScores &scores, bool again, int wave, F &&load) {
    // the step's addresses; all others are constants away (as values of their own, or the compiler keeps hundreds of sums with those constants)
    const uint32_t stage = stage_of_all + first_group(wave) * G::GROUP;
    uint32_t at_row[4], at_rope[NR], at_col[8];
#pragma unroll
    for (int i = 0; i < 4; i++) at_row[i] = own(stage + (own(row_at) ^ (i << 6)));
#pragma unroll
    for (int i = 0; i < NR; i++) at_rope[i] = own(stage + (own(rope_at) ^ (i << 6)));
    // scores: value 4 k + i is that of position 4 c + i of group k
    constexpr int ALL = NS + NR, TB = 4 / HW, BATCHES = (ALL + TB - 1) / TB, AHEAD = 3;
    constexpr int CHAINS = 4 / HW;                        // four products that do not wait for each other
    f32x4 acc[HW][CHAINS];
#pragma unroll
    for (int k = 0; k < HW; k++)
#pragma unroll
      for (int x = 0; x < CHAINS; x++) acc[k][x] = f32x4{0.f, 0.f, 0.f, 0.f};
    frag8 rows[AHEAD + 1][4];
    auto read_rows = [&](int b) {
#pragma unroll
      for (int j = 0; j < TB; j++)
#pragma unroll
        for (int k = 0; k < HW; k++) {
          const int t = b * TB + j;
          if (t < ALL) rows[b % (AHEAD + 1)][j * HW + k] = latent_read<frag8>((t < NS ? at_row[t & 3] + (t >> 2) * 256 : at_rope[t < NS ? 0 : t - NS]) + k * G::GROUP);
        }
    };
#pragma unroll
    for (int b = 0; b < AHEAD; b++) read_rows(b);
#pragma unroll
    for (int b = 0; b < BATCHES; b++) {
      if (b + AHEAD < BATCHES) read_rows(b + AHEAD);
#pragma unroll
      for (int k = b * G::LOADS / BATCHES; k < (b + 1) * G::LOADS / BATCHES; k++) load(k);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < TB; j++)
#pragma unroll
        for (int k = 0; k < HW; k++) {
          const int t = b * TB + j;
          if (t < ALL) acc[k][t % CHAINS] = M::run(rows[b % (AHEAD + 1)][j * HW + k], q[t], acc[k][t % CHAINS]);
        }
      __builtin_amdgcn_sched_barrier(0);
    }
    constexpr int PAIRS = HW == 1 ? 1 : HW / 2, NB = NT / 4, PER = HW == 1 ? 4 : 8;
    frag cols[3][4];
#pragma unroll
    for (int i = 0; i < 8; i++) at_col[i] = own(stage + (own(tr_at) ^ (i << 5)));
    auto read_cols = [&](int b) {
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int n = b % NB * 4 + j;
        const uint32_t from = at_col[n & 7] + b / NB * 2 * G::GROUP + (n >> 3) * 256;
        if constexpr (HW == 1) cols[b % 3][j] = __builtin_bit_cast(frag, latent_read_tr(from));
        else cols[b % 3][j] = __builtin_bit_cast(frag, latent_read_tr2(from, from + G::GROUP));
      }
    };
    read_cols(0);
    read_cols(1);
    __builtin_amdgcn_sched_barrier(0);
    uint32_t seen = (1u << (4 * HW)) - 1u;
    bool all = true;
#pragma unroll
    for (int k = 0; k < HW; k++) all = all && now[k].n == 16 && (now[k].mask & 0xffff) == 0xffff;
    if (!all) {
      seen = 0;
#pragma unroll
      for (int k = 0; k < HW; k++) seen |= (here && (now[k].mask >> key & 1) ? first_of_four(now[k].n - 4 * c) : 0u) << (4 * k);
    }
    float sc[4 * HW];
#pragma unroll
    for (int i = 0; i < 4 * HW; i++) {
      sc[i] = acc[i >> 2][0][i & 3];
#pragma unroll
      for (int x = 1; x < CHAINS; x++) sc[i] += acc[i >> 2][x][i & 3];
    }
    auto logits = [&](float (&y)[4 * HW], float minus) {
      latent_logits(y, [&](int i) { return sc[i]; }, scores, slope, minus, [&](int i) { return now[i >> 2].pos + 4 * c + (i & 3); });
    };
    // shares relative to the running maximum, which moves when they grow past 8192
    float e[4 * HW], sum;
    auto exponentials = [&]() {
      logits(e, m == -INFINITY ? 0.f : m);
#pragma unroll
      for (int i = 0; i < 4 * HW; i++) e[i] = __builtin_amdgcn_exp2f(e[i]);
      if (!all)
#pragma unroll
        for (int i = 0; i < 4 * HW; i++) e[i] = seen >> i & 1 ? e[i] : 0.f;
      sum = 0.f;
#pragma unroll
      for (int i = 0; i < 4 * HW; i++) sum += e[i];
    };
    exponentials();
    auto top_of = [&]() {
      float y[4 * HW], top = -INFINITY;
      logits(y, 0.f);
#pragma unroll
      for (int i = 0; i < 4 * HW; i++) top = fmaxf(top, seen >> i & 1 ? y[i] : -INFINITY);
      top = fmaxf(top, __shfl_xor(top, 16));
      return fmaxf(top, __shfl_xor(top, 32));
    };
    if (__builtin_amdgcn_ballot_w64(m == -INFINITY && seen != 0)) {            // the first that a head sees: its sums are zeros
      const float top = top_of();
      m = m == -INFINITY ? top : m;
      exponentials();
    }
    if (!again && __builtin_amdgcn_ballot_w64(sum > 8192.f)) {
      const float mn = fmaxf(m, top_of());
      scaled = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
      l *= scaled;
      m = mn;
      return false;
    }
    l += sum;
    frag most[PAIRS], rest[PAIRS];
#pragma unroll
    for (int i = 0; i < 4 * HW; i++) {
      most[i / PER][i % PER] = from_float<T>(e[i]);
      rest[i / PER][i % PER] = from_float<T>(e[i] - to_float(most[i / PER][i % PER]));
    }
#pragma unroll
    for (int b = 0; b < PAIRS * NB; b++) {
      if (b + 2 < PAIRS * NB) read_cols(b + 2);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < 4; j++) o[b % NB * 4 + j] = M::run(cols[b % 3][j], most[b / NB], o[b % NB * 4 + j]);
#pragma unroll
      for (int j = 0; j < 4; j++) o[b % NB * 4 + j] = M::run(cols[b % 3][j], rest[b / NB], o[b % NB * 4 + j]);
      __builtin_amdgcn_sched_barrier(0);
    }
    return true;
  }
  __device__ __forceinline__ void scale() {
#pragma unroll
    for (int n = 0; n < NT; n++) o[n] = scaled_by(o[n], scaled);
  }
  // maximum, sum and sums to their row
  __device__ __forceinline__ void put(float *join, float *stats, int wave) {
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    const int r = 16 * wave + key;
    if (c == 0) stats[2 * r] = m, stats[2 * r + 1] = l;
#pragma unroll
    for (int n = 0; n < NT; n++) *reinterpret_cast<f32x4 *>(join + r * G::JOIN + 16 * n + 4 * c) = o[n];
  }
};

// An item is a sequence and a unit of its heads; its groups of sixteen positions
struct LatentItem {
  int b, unit, len, groups, entry;
  LatentItem() = default;
  __device__ __forceinline__ LatentItem(const LatentArgs &a, uint32_t item) {
    const Quotient i(item, a.units);
    b = (int)i.q;
    unit = (int)i.r;
    const int64_t held = (int64_t)a.width * a.block, seen = (int64_t)a.n_rows * a.block, most = a.rows && seen < held ? seen : held;
    len = a.lengths[b];
    len = len < most ? len : (int)most;
    groups = entry = 0;
    if (len > 0) {
      groups = (len + 15) >> 4;
      if (a.rows) {
        const int32_t *t = a.rows + (int64_t)unit * (a.n_rows + 1) + (len - 1) / a.block;
        entry = t[0];
        groups = (t[1] - t[0]) << a.shift;
      }
      groups = groups < a.most_groups ? groups : a.most_groups;   // (or parts would be written past the workspace, where a caller has most_blocks wrong)
    }
  }
  __device__ __forceinline__ int steps() const { return (groups + 3) >> 2; }
};

template <typename T, int LAT, int HW>
__global__ void __launch_bounds__(256, 1) k_latent_attention(LatentArgs a) {
  typedef LatentGeo<LAT> G;
  typedef Heads<T, LAT, HW> H;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int mine = H::first_group(wave);            // the first of the step's groups that the wavefront goes through
  const uint32_t items = (uint32_t)(a.B * a.units), ring = (uint32_t)(uintptr_t)BSP_LDS_PTR(smem);

  // The workgroup's piece [lo, hi) of all steps, and the item that it begins in.  Where there are more steps than pieces, an item counts `extra` steps more ahead of its own: what a
  // workgroup that goes over to another item spends on the queries and on the sums of the last (16 x 64 heads over up to 16384 positions: 81 us without, 72 with; 128 x 128 heads over up to 500:
  // 87 and 65; 300 x 16 over up to 600: 61 and 46; two or eight steps instead of four: 76 and 72, 67 and 62).  With a step or less a piece they would only leave pieces empty: 4 x 128 heads over up to 300,
  // 25 us with them, 21 without.
  int64_t total = 0, lo, hi, begin = 0;
  uint32_t item = 0;
  LatentItem found{}, looked{};                         // that item; what the thread has looked at last
  int pieces, extra;
  {
    int *sums = reinterpret_cast<int *>(smem + G::STATS);                     // (where no tile goes)
    // of 256 items: the thread's steps, the steps and (2^40 each) the number of those before it in the chunk that have any; returns the chunk's
    auto chunk_sum = [&](uint32_t base, int &own, uint64_t &before) {
      const uint32_t i = base + tid;
      own = 0;
      if (i < items) {
        looked = LatentItem(a, i);
        own = looked.steps();
      }
      const uint64_t mine_of = (uint64_t)own | (own > 0 ? (uint64_t)1 << 40 : 0);
      uint64_t x = mine_of;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const uint64_t y = __shfl_up((unsigned long long)x, d);
        if (lane >= d) x += y;
      }
      __syncthreads();
      if (lane == 63) reinterpret_cast<uint64_t *>(sums)[wave] = x;
      __syncthreads();
      uint64_t all = 0;
      before = x - mine_of;
#pragma unroll
      for (int w = 0; w < 4; w++) {
        const uint64_t y = reinterpret_cast<uint64_t *>(sums)[w];
        before += w < wave ? y : 0;
        all += y;
      }
      return all;
    };
    constexpr uint64_t kSteps = ((uint64_t)1 << 40) - 1;
    int own = 0;
    uint64_t before = 0, every = 0;
    for (uint32_t base = 0; base < items; base += 256) {
      every += chunk_sum(base, own, before);
      const uint32_t i = base + tid;
      if (i < items && own == 0) {                                            // nothing is seen: zeros
        if (blockIdx.x == 0) a.meta[2 * (int64_t)i + 1] = 0;
      }
      uint64_t none = __builtin_amdgcn_ballot_w64(i < items && own == 0 && i % gridDim.x == blockIdx.x);
      while (none) {
        const int j = __builtin_ctzll(none);
        none &= none - 1;
        const Quotient z(base + 64 * wave + j, a.units);
        const int first = (int)z.r * a.per, n = a.H - first < a.per ? a.H - first : a.per;
        for (int k = lane; k < n * (LAT / 8); k += 64)
          *reinterpret_cast<u32x4 *>(reinterpret_cast<T *>(a.o) + z.q * a.o_sb + (first + k / (LAT / 8)) * a.o_sh + 8 * (k % (LAT / 8))) = u32x4{0, 0, 0, 0};
      }
    }
    total = (int64_t)(every & kSteps);
    pieces = total < a.pieces ? (int)total : a.pieces;    // (none is empty)
    if ((int)blockIdx.x >= pieces) return;
    extra = total > a.pieces ? H::EXTRA : 0;
    auto steps_of = [&](uint64_t x) { return (int64_t)(x & kSteps) + extra * (int64_t)(x >> 40); };
    total = steps_of(every);
    lo = total * blockIdx.x / pieces;
    hi = total * (blockIdx.x + 1) / pieces;
    int64_t done = 0;
    for (uint32_t base = 0; base < items; base += 256) {
      if (items > 256 || base > 0) {
        const int64_t all = steps_of(chunk_sum(base, own, before));
        if (done + all <= lo) {
          done += all;
          continue;
        }
      }
      const int64_t from = done + steps_of(before);
      __syncthreads();
      if (own > 0 && from <= lo && lo < from + own + extra) {
        sums[4] = (int)base + tid;
        sums[5] = (int)(from - done);
        sums[6] = looked.len;
        sums[7] = looked.groups;
        sums[8] = looked.entry;
      }
      __syncthreads();
      item = (uint32_t)__builtin_amdgcn_readfirstlane(sums[4]);
      begin = done + __builtin_amdgcn_readfirstlane(sums[5]);
      const Quotient of(item, a.units);
      found.b = (int)of.q;
      found.unit = (int)of.r;
      found.len = sums[6];
      found.groups = sums[7];
      found.entry = sums[8];
      break;
    }
  }

  LatentScores scores;
  scores.capped = a.cap > 0.f;
  scores.sloped = a.slopes != nullptr;
  scores.factor = scores.capped ? 2.f * kLog2e * a.scale / a.cap : a.scale * kLog2e;
  scores.cap = a.cap * kLog2e;

  bool looked_up = true;
  for (; begin < hi && item < items; item++) {
    const LatentItem it = looked_up ? found : LatentItem(a, item);
    looked_up = false;
    const int steps = __builtin_amdgcn_readfirstlane(it.steps());
    if (steps == 0) continue;
    // the item's steps that are the workgroup's
    const int64_t first_step = begin + extra;
    begin = first_step + steps;
    const int s0 = lo > first_step ? (int)(lo - first_step) : 0, s1 = begin < hi ? steps : (int)(hi - first_step);
    if (s1 <= s0) continue;
    const int b = __builtin_amdgcn_readfirstlane(it.b), unit = __builtin_amdgcn_readfirstlane(it.unit), len = __builtin_amdgcn_readfirstlane(it.len);
    const int groups = __builtin_amdgcn_readfirstlane(it.groups), entry = __builtin_amdgcn_readfirstlane(it.entry);
    const int first = unit * a.per, heads = a.H - first < a.per ? a.H - first : a.per;
    scores.last = len - 1;

    // 64 groups at a time, one a lane
    int base = s0, v_page = 0, v_pos = 0, v_n = 0, v_sub = 0, v_lo = 0, v_hi = 0;
    auto look = [&]() {
      const int g = 4 * base + lane;
      const bool in = g < groups;
      int col = g >> a.shift;
      v_lo = v_hi = -1;
      if (a.rows) {
        const int32_t *e = a.rows + (int64_t)a.units * (a.n_rows + 1) + 3 * (int64_t)(in ? entry + col : entry);
        col = e[0];
        v_lo = e[1];
        v_hi = e[2];
      }
      v_sub = g & ((1 << a.shift) - 1);
      v_pos = col * a.block + 16 * v_sub;
      int n = in ? len - v_pos : 0, page = 0;
      if (n > 0) page = a.table[b * a.table_sb + col];    // (col * block < len, so within the row of the table)
      if (page < 0 || page >= a.n_pages) n = 0;
      v_n = n < 0 ? 0 : n > 16 ? 16 : n;
      v_page = v_n > 0 ? page : 0;
    };
    auto group_of = [&](int i) {
      return LatentGroup{__builtin_amdgcn_readlane(v_pos, i), __builtin_amdgcn_readlane(v_n, i), H::mask(wave, __builtin_amdgcn_readlane(v_lo, i), __builtin_amdgcn_readlane(v_hi, i))};
    };
    // the wavefront's group of a step on its way to its place in one of the stages: load k of the group
    i32x4b rows;
    uint32_t dst = 0;
    auto aim = [&](int s) {
      const int i = 4 * (s - base) + wave;
      const int page = __builtin_amdgcn_readlane(v_page, i), sub = __builtin_amdgcn_readlane(v_sub, i), n = s < s1 ? __builtin_amdgcn_readlane(v_n, i) : 0;
      const uint64_t from = reinterpret_cast<uint64_t>(a.pages) + ((int64_t)page * a.block + 16 * sub) * (int64_t)G::ROW;
      rows = i32x4b{(int)(uint32_t)from, (int)(uint32_t)(from >> 32) & 0xffff, n * G::ROW, 0x00020000};
      dst = __builtin_amdgcn_readfirstlane(ring + (s & 1) * G::STAGE + wave * G::GROUP);
    };
    // (a row's number is that of the load's first and the lane's, in bits of their own, and the exchange of chunks goes by bits)
    const uint32_t lane_chunk = H::chunk(lane % G::CPR, lane / G::CPR) << 4, lane_row = lane / G::CPR * G::ROW;
    const uint32_t lane_rope = rope_chunk(lane % 8, lane / 8) << 4, lane_rope_row = lane / 8 * G::ROW + G::LROW;
    auto load = [&](int k) {
      const int j = k - (G::LOADS - 2);
      if (j < 0) rows_to_lds(rows, (own(lane_chunk) ^ H::chunk(0, k * G::RPI) << 4) + (lane_row + k * G::RPI * G::ROW), dst + k * 1024);
      else rows_to_lds(rows, (own(lane_rope) ^ rope_chunk(0, 8 * j) << 4) + (lane_rope_row + 8 * j * G::ROW), dst + 16 * G::LROW + j * 1024);
    };

    look();
    aim(s0);
#pragma unroll
    for (int k = 0; k < G::LOADS; k++) load(k);
    H x;
    {
      const int head = H::head_of(wave, lane);        // the lane's head among the unit's
      const bool here = head < heads;
      const int64_t h = first + (here ? head : 0);
      x.init(reinterpret_cast<const T *>(a.q) + b * a.q_sb + h * a.q_sh, reinterpret_cast<const T *>(a.qr) + b * a.qr_sb + h * a.qr_sh, here,
             a.slopes ? a.slopes[h] * kLog2e : 0.f, lane);
    }
    LatentGroup now[H::GROUPS], next[H::GROUPS];
#pragma unroll
    for (int k = 0; k < H::GROUPS; k++) now[k] = next[k] = group_of(mine + k);

    // A step whose shares grow past 8192 leaves the loop for the sums to be scaled and is taken again: with that in it, the compiler moves all sums out of the matrix
    // units' registers and back in every step.
    x.arrived();
    int s = s0;
    bool again = false;
    while (true) {
      for (; s < s1; s++) {
        if (!again) {
          BSP_WAIT_VM(0);
          asm volatile("" ::: "memory");
          if constexpr (H::BARRIER) {
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
          }
          if (s + 1 - base == 16 && s + 1 < s1) {
            base = s + 1;
            look();
          }
          aim(s + 1);                                     // (behind the last step: loads of nothing; a step that is taken again loads the same again)
          if (s + 1 < s1) {
#pragma unroll
            for (int k = 0; k < H::GROUPS; k++) next[k] = group_of(4 * (s + 1 - base) + mine + k);
          }
        }
        again = !x.step(ring + (s & 1) * G::STAGE, now, scores, again, wave, load);
        if (again) break;
#pragma unroll
        for (int k = 0; k < H::GROUPS; k++) now[k] = next[k];
      }
      if (s >= s1) break;
      x.scale();
    }

    // the wavefronts' results: per head the maximum, the sum, LAT sums
    BSP_WAIT_VM(0);
    __syncthreads();
    float *join = reinterpret_cast<float *>(smem), *stats = reinterpret_cast<float *>(smem + G::STATS);
    x.put(join, stats, wave);
    __syncthreads();
    const bool whole = s0 == 0 && s1 == steps;
    const int slot = 2 * blockIdx.x + (s0 == 0 ? 1 : 0);  // (of a piece's parts one at most begins its item and one at most does not)
    if (tid == 0 && s0 == 0) {
      int parts = 1;
      if (!whole) {                                       // up to the piece that the item's last step is in
        const int64_t last = (begin * pieces - 1) / total;
        parts = (int)(last - blockIdx.x) + 1;
      }
      int32_t *to = a.meta + 2 * (int64_t)item;
      to[0] = blockIdx.x;
      to[1] = parts;
    }
    // what each source's sums are multiplied by, a head a thread; then four elements a thread, four of them on their way
    float *by = reinterpret_cast<float *>(smem + G::FACTORS);
    float *parts_of = a.partial + (int64_t)slot * a.per * LAT, *stats_of = a.partial + (int64_t)2 * a.pieces * a.per * LAT + (int64_t)slot * a.per * 2;
    if (tid < heads) {
      float top = -INFINITY, sum = 0.f, f[H::SOURCES];
#pragma unroll
      for (int p = 0; p < H::SOURCES; p++) top = fmaxf(top, stats[2 * H::source(tid, p)]);
#pragma unroll
      for (int p = 0; p < H::SOURCES; p++) {
        const int r = H::source(tid, p);
        f[p] = stats[2 * r] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(stats[2 * r] - top);
        sum = fmaf(f[p], stats[2 * r + 1], sum);
      }
      const float last = !whole ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
      for (int p = 0; p < H::SOURCES; p++) by[64 * p + tid] = f[p] * last;
      if (!whole) stats_of[2 * tid] = top, stats_of[2 * tid + 1] = sum;
    }
    __syncthreads();
    constexpr int LANES = LAT / 4, U = 4, TERMS = H::SOURCES;   // LANES: threads of a head
    const int all = heads * LANES;
    for (int i0 = tid; i0 < all; i0 += 256 * U) {
      f32x4 v[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int i = i0 + 256 * u < all ? i0 + 256 * u : i0, h = i / LANES, d = i % LANES * 4;
        v[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int p = 0; p < TERMS; p++) {
          const float f = by[64 * p + h];
          const f32x4 w = *reinterpret_cast<const f32x4 *>(join + H::source(h, p) * G::JOIN + d);
#pragma unroll
          for (int e = 0; e < 4; e++) v[u][e] = f == 0.f ? v[u][e] : fmaf(f, w[e], v[u][e]);
        }
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int i = i0 + 256 * u, h = i / LANES, d = i % LANES * 4;
        if (i >= all) continue;
        if (whole) {
          union { u32x2 raw; T e[4]; } out;
#pragma unroll
          for (int e = 0; e < 4; e++) out.e[e] = from_float<T>(v[u][e]);
          *reinterpret_cast<u32x2 *>(reinterpret_cast<T *>(a.o) + b * a.o_sb + (first + h) * a.o_sh + d) = out.raw;
        } else {
          *reinterpret_cast<f32x4 *>(parts_of + h * LAT + d) = v[u];
        }
      }
    }
    __syncthreads();
  }
}

// The parts of a sequence's head joined: a workgroup a head (or SPAN of its elements), a part's maximum and sum a lane at a time, then the parts among its W wavefronts.  Parts that saw nothing have
// a factor of 0.
template <typename T, int LAT, int SPAN, int W> __global__ void __launch_bounds__(64 * W) k_latent_join(LatentArgs a) {
  constexpr int N = SPAN / 64;
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  __shared__ float sums[W][SPAN + 2], tops[W];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Quotient at(blockIdx.x, a.H);
  const int from_element = blockIdx.y * SPAN;
  const int b = (int)at.q, h = (int)at.r, unit = h / a.per, r = h % a.per;
  const int32_t *meta = a.meta + 2 * ((int64_t)b * a.units + unit);
  const int parts = meta[1];
  if (parts <= 1) return;
  const int from = meta[0];
  const float *stats = a.partial + (int64_t)2 * a.pieces * a.per * LAT;
  auto part = [&](int p) { return (int64_t)(2 * (from + p) + (p == 0 ? 1 : 0)) * a.per + r; };
  float top = -INFINITY;
  for (int p = tid; p < parts; p += 64 * W) top = fmaxf(top, stats[2 * part(p)]);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
  if (lane == 0) tops[wave] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < W; w++) top = fmaxf(top, tops[w]);
  float sum = 0.f, x[N] = {};
  for (int p0 = wave; p0 < parts; p0 += 4 * W) {             // four of the wavefront's parts on their way
    f32x2 own[4];
    float v[4][N];
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const int64_t p = part(p0 + W * u < parts ? p0 + W * u : p0);
      own[u] = *reinterpret_cast<const f32x2 *>(stats + 2 * p);
#pragma unroll
      for (int e = 0; e < N; e += 2) {
        const f32x2 w = *reinterpret_cast<const f32x2 *>(a.partial + p * LAT + from_element + 64 * e + 2 * lane);
        v[u][e] = w[0];
        v[u][e + 1] = w[1];
      }
    }
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const float f = p0 + W * u >= parts || own[u][0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(own[u][0] - top);
      sum = fmaf(f, own[u][1], sum);
#pragma unroll
      for (int e = 0; e < N; e++) x[e] = fmaf(f, v[u][e], x[e]);
    }
  }
  if (lane == 0) sums[wave][SPAN] = sum;
#pragma unroll
  for (int e = 0; e < N; e += 2) *reinterpret_cast<f32x2 *>(&sums[wave][0] + 64 * e + 2 * lane) = f32x2{x[e], x[e + 1]};
  __syncthreads();
  sum = 0.f;
#pragma unroll
  for (int w = 0; w < W; w++) sum += sums[w][SPAN];
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  for (int d = tid; d < SPAN; d += 64 * W) {
    float y = 0.f;
#pragma unroll
    for (int w = 0; w < W; w++) y += sums[w][d];
    reinterpret_cast<T *>(a.o)[b * a.o_sb + h * a.o_sh + from_element + d] = from_float<T>(sum == 0.f ? 0.f : y * inv);
  }
}

template <typename T, int LAT, int HW> int launch_latent_heads(const LatentArgs &a, hipStream_t st) {
  static std::atomic<uint64_t> done{0};
  if (LatentGeo<LAT>::LDS > 65536 && !raise_lds_limit(reinterpret_cast<const void *>(k_latent_attention<T, LAT, HW>), LatentGeo<LAT>::LDS, done)) return BSP_ERR_HIP;
  hipLaunchKernelGGL((k_latent_attention<T, LAT, HW>), dim3((unsigned)a.pieces), dim3(256), LatentGeo<LAT>::LDS, st, a);
  return BSP_OK;
}
template <typename T, int LAT> int launch_latent(const LatentArgs &a, bool joined, hipStream_t st) {
  // (as few wavefronts to a group as have heads: the others would read the same from LDS for nothing.  16 sequences of up to 16384 positions, 16 heads: 52.0 us by one and 52.6 by two, with latent
  // vectors of 128 22.2 and 24.2)
  const int rc = a.per <= 16 ? launch_latent_heads<T, LAT, 1>(a, st) : a.per <= 32 ? launch_latent_heads<T, LAT, 2>(a, st) : launch_latent_heads<T, LAT, 4>(a, st);
  if (rc != BSP_OK) return rc;
  // a head's elements among several workgroups, of more wavefronts, where there are few heads: with one a head one sequence of up to 16384 positions takes 11.7 us for 16 heads (256 parts of
  // each) and 9.2 for 128, like this 6.2 and 8.4; 4 x 32 heads 6.9 and 6.1
  if (joined && (int64_t)a.B * a.H <= 128) hipLaunchKernelGGL((k_latent_join<T, LAT, 128, 16>), dim3((unsigned)((int64_t)a.B * a.H), LAT / 128), dim3(1024), 0, st, a);
  else if (joined) hipLaunchKernelGGL((k_latent_join<T, LAT, LAT, 4>), dim3((unsigned)((int64_t)a.B * a.H)), dim3(256), 0, st, a);
  BSP_LAUNCH_CHECK();
  return BSP_OK;
}
template <typename T> int launch_latent(const LatentArgs &a, int latent, bool joined, hipStream_t st) {
  return latent == 512 ? launch_latent<T, 512>(a, joined, st) : latent == 256 ? launch_latent<T, 256>(a, joined, st) : launch_latent<T, 128>(a, joined, st);
}

constexpr int kMostHeads = 64;     // of a workgroup

int latent_units(int H) { return (H + kMostHeads - 1) / kMostHeads; }
// Workgroups of a launch over B sequences of at most `blocks` blocks: one a compute unit, of as many as there are steps
int latent_pieces(int B, int H, int block, int64_t blocks) {
  const double steps = (double)B * latent_units(H) * (double)((blocks * block + 63) / 64);
  return steps < 256. ? (int)steps : 256;
}

}  // namespace
}  // namespace bsp

using namespace bsp;

extern "C" int bsp_latent_attention_heads(int H) {
  if (H <= 0) return BSP_ERR_ARG;
  return (H + latent_units(H) - 1) / latent_units(H);
}

extern "C" int64_t bsp_latent_attention_workspace_bytes(int B, int H, int latent, int block, int64_t most_blocks) {
  if (B <= 0 || H <= 0 || !latent_ok(latent, block) || most_blocks <= 0) return BSP_ERR_ARG;
  const int64_t meta = ((int64_t)B * latent_units(H) * 8 + 15) / 16 * 16;
  return meta + (most_blocks * block <= 64 ? 0 : (int64_t)latent_pieces(B, H, block, most_blocks) * 2 * bsp_latent_attention_heads(H) * (latent + 2) * 4);
}

extern "C" int bsp_latent_attention(int dtype, const void *q, int64_t q_stride_b, int64_t q_stride_h, const void *q_r, int64_t qr_stride_b, int64_t qr_stride_h, void *o,
                                    int64_t o_stride_b, int64_t o_stride_h, int B, int H, const void *pages, int n_pages, int block, int latent, const int32_t *table,
                                    int64_t table_stride, int width, const int32_t *lengths, const int32_t *rows, int n_rows, int64_t most_blocks, float scale, float softcap,
                                    const float *slopes, void *workspace, int64_t workspace_bytes, void *stream) {
  if (!q || !q_r || !o || !pages || !table || !lengths || B <= 0 || H <= 0 || n_pages <= 0 || width <= 0 || most_blocks <= 0) return BSP_ERR_ARG;
  if ((dtype != BSP_F16 && dtype != BSP_BF16) || !latent_ok(latent, block)) return BSP_ERR_UNSUPPORTED;
  const void *ptrs[] = {q, q_r, o, pages, workspace};
  for (const void *p : ptrs)
    if (reinterpret_cast<uintptr_t>(p) & 15) return BSP_ERR_ARG;
  if (q_stride_b % 8 || q_stride_h % 8 || qr_stride_b % 8 || qr_stride_h % 8 || o_stride_b % 8 || o_stride_h % 8) return BSP_ERR_ARG;
  if (!scores_ok(scale, softcap) || (rows && n_rows <= 0)) return BSP_ERR_ARG;
  if ((int64_t)width * block >= ((int64_t)1 << 24) || (int64_t)n_pages * block >= ((int64_t)1 << 31) || (rows && n_rows > 65536)) return BSP_ERR_UNSUPPORTED;
  if ((int64_t)B * H >= ((int64_t)1 << 24)) return BSP_ERR_UNSUPPORTED;       // (a grid has fewer than 2^32 threads)
  if (!workspace || workspace_bytes < bsp_latent_attention_workspace_bytes(B, H, latent, block, most_blocks)) return BSP_ERR_CAPACITY;
  LatentArgs a{};
  a.q = q; a.q_sb = q_stride_b; a.q_sh = q_stride_h; a.qr = q_r; a.qr_sb = qr_stride_b; a.qr_sh = qr_stride_h;
  a.o = o; a.o_sb = o_stride_b; a.o_sh = o_stride_h;
  a.pages = pages; a.n_pages = n_pages; a.table = table; a.table_sb = table_stride; a.width = width; a.lengths = lengths;
  a.rows = rows; a.n_rows = n_rows; a.slopes = slopes; a.scale = scale; a.cap = softcap;
  a.B = B; a.H = H; a.block = block; a.shift = __builtin_ctz(block) - 4;
  a.most_groups = (int)(most_blocks < (1 << 24) ? most_blocks << a.shift : 1 << 30);
  a.units = latent_units(H); a.per = bsp_latent_attention_heads(H); a.pieces = latent_pieces(B, H, block, most_blocks);
  a.meta = reinterpret_cast<int32_t *>(workspace);
  a.partial = reinterpret_cast<float *>(reinterpret_cast<unsigned char *>(workspace) + ((int64_t)B * a.units * 8 + 15) / 16 * 16);
  const bool joined = most_blocks * block > 64;           // (else no sequence has more than one step)
  return dtype == BSP_F16 ? launch_latent<f16>(a, latent, joined, as_stream(stream)) : launch_latent<bf16>(a, latent, joined, as_stream(stream));
}
