// Attention of one new position a sequence over a quantised cache (cache.h): for sequence b of length n and query head h
//     y_j = cap * tanh(scale * q . k_j / cap) - slope_h * (n - 1 - j),   o = softmax(y) . v
// over the positions j < n whose page the sequence holds and, with a layout, whose block is in row (n - 1) / block of head h.
//
// What bounds it is the cache: every byte of the pages that are seen is read once for all the query heads that share a key head (up
// to 16 a workgroup).  Each of a workgroup's four wavefronts goes through its own pairs of tiles of sixteen positions, a pair's
// codes and steps on their way while the one before is computed, and the wavefronts' results are joined in LDS.  Where sequences and
// key heads do not fill the chip the positions are split among workgroups, and a second kernel joins what those leave.
//
// The codes are operands as they are, bit patterns of fp16 numbers below the normal ones, so a score is the sum over the groups of step * (q . codes) +
// least * (sum of the group's q), the products on the matrix units (16 x 16 x 32: a group each).  q is scaled by a power of two per head to the
// range of fp16, which loses nothing that 2^-35 of its largest element would not.  Values are v = least + code * step rounded to fp16
// (2^-12 of it; 65504 at most) through LDS, where the product with the shares reads them transposed.
//
// Measured: sixteen sequences of up to 16384 positions, 32 query heads of 128 on 8 key heads, 4 bits (218 MB of pages): 52 us with the join, 4.2 TB/s
// (all of 16384 positions: 61 us, 5.5 TB/s); loading the same bytes and nothing else takes 40.  What is left is that compute units get unequal shares of ragged
// sequences, and the vector units: taking the codes out of their words for keys and values was 240 of 390 operations a pair of tiles and is 140 of 270 with keys as
// they lie (63 us before).  Looking for values past fp16's range (see `large`) is 1.3 of the 52.
//
// Scores lie with a position per lane and the query heads along the sixteen result rows of the matrix unit, dealt so that a head takes one
// value in a quarter of the lanes: with at most four heads a key head (V = 1) a tile costs one exponential a lane, with up to eight two.
#include "attention_common.h"
#include "cache.h"

namespace bsp {

struct DecodeArgs {
  const void *q; void *o;          // [B, H, D]
  int64_t q_sb, q_sh, o_sb, o_sh;
  const unsigned char *pages; int64_t n_pages;
  const int32_t *table; int64_t table_sb; int width;     // pages of a sequence
  const int32_t *lengths;
  const int32_t *rows;             // NULL, or per unit and block-row (first entry, then one past the last row's end), then entries: block-column << 16 | heads of the unit that see it
  int n_rows;
  const float *slopes;
  float scale, cap;
  float *partial;                  // [B][units][splits][heads a unit][D + 2]
  int B, H, kv_heads, block, tile_shift;                  // tile_shift: log2 of the tiles of sixteen positions a page
  int G, per, units, splits, chunk;   // query heads a key head; heads of a unit (a workgroup's), units; workgroups a unit, pairs of tiles a wavefront of them
};

namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

template <int BITS, int D> struct RawTile {
  static constexpr int QB = D * BITS / 32 / 4;            // 32-bit words of a quarter row
  static constexpr int GROUPS = D / 32;
  uint32_t kc[QB], vc[QB], km[GROUPS], vm[GROUPS];
};
// (each byte is read once: streamed past the L2, 54.5 -> 52 us)
template <int N> __device__ __forceinline__ void load_words(uint32_t (&w)[N], const unsigned char *p) {
  if constexpr (N == 2) {
    const u32x2 x = __builtin_nontemporal_load(reinterpret_cast<const u32x2 *>(p));
    w[0] = x[0], w[1] = x[1];
  } else {
#pragma unroll
    for (int i = 0; i < N / 4; i++) {
      const u32x4 x = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p + 16 * i));
#pragma unroll
      for (int j = 0; j < 4; j++) w[4 * i + j] = x[j];
    }
  }
}
__device__ __forceinline__ float step_of(uint32_t meta) { return (float)__builtin_bit_cast(f16, (uint16_t)meta); }
__device__ __forceinline__ float least_of(uint32_t meta) { return (float)__builtin_bit_cast(f16, (uint16_t)(meta >> 16)); }
template <int BITS, int D> struct DecodeLds {
  static constexpr int VROW = 2 * D + 16, PROW = 80;      // bytes of a position's values, of a head's 32 shares
  static constexpr int join(int V) { return 4 * 4 * V * (D + 2) * 4; }
  static constexpr int wave(bool fine) { return 32 * VROW + (fine ? 2 : 1) * 16 * PROW; }
  static constexpr int bytes(int V, bool fine) { return 4 * wave(fine) > join(V) ? 4 * wave(fine) : join(V); }
};

// FINE: float16, whose results have eleven bits: the shares in two terms, what they are rounded to and what that leaves out.  (In bfloat16 their rounding is nothing beside
// the result's.)
template <int BITS, int D, int V, bool FINE>
__global__ void __launch_bounds__(256, 3) k_cache_attention(DecodeArgs a) {
  typedef Page<BITS, D> P;
  typedef DecodeLds<BITS, D> L;
  constexpr int GR = D / 32, NT = D / 16;
  __shared__ __attribute__((aligned(16))) unsigned char smem[L::bytes(V, FINE)];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), key = lane & 15, c = lane >> 4;
  // the first pieces of all sequences and heads, then the second ones: the workgroups that find nothing to do come last, and every XCD (they take workgroups
  // in turn) gets the same share of the long sequences
  const uint32_t groups = (uint32_t)(a.B * a.units), split = blockIdx.x / groups, group = blockIdx.x % groups;
  const int unit = (int)(group % (uint32_t)a.units), b = (int)(group / (uint32_t)a.units);
  const int per_key = (a.G + a.per - 1) / a.per, hk = unit / per_key, first = hk * a.G + unit % per_key * a.per;
  const int heads = hk * a.G + a.G - first < a.per ? hk * a.G + a.G - first : a.per;     // the unit's query heads: first ..
  const int held = a.width * a.block, most = a.rows && a.n_rows * a.block < held ? a.n_rows * a.block : held;
  int len = as_table(a.lengths)[b];
  len = len < most ? len : most;

  int tiles = 0, entry = 0;
  if (len > 0) {
    tiles = (len + 15) >> 4;
    if (a.rows) {
      const table_ptr t = as_table(a.rows) + unit * (a.n_rows + 1) + (len - 1) / a.block;
      entry = t[0];
      tiles = (t[1] - t[0]) << a.tile_shift;
    }
  }
  // this wavefront's pairs of tiles: the same number for all, whatever the sequences' lengths, so that no workgroup has much more to do than another
  const int pairs = (tiles + 1) >> 1, part = split * 4 + wave;
  const int p_end = pairs < (part + 1) * a.chunk ? pairs : (part + 1) * a.chunk;
  int pair = part * a.chunk;

  // row m of a product's first operand belongs to the unit's head (m / 4) * V + m % 4
  const int row = (key >> 2) * V + (key & 3);
  const bool row_here = (key & 3) < V && row < heads;
  union { u32x4 raw; f16 h[8]; bf16 f[8]; } q[GR];
#pragma unroll
  for (int g = 0; g < GR; g++)
    q[g].raw = *reinterpret_cast<const u32x4 *>(reinterpret_cast<const uint16_t *>(a.q) + b * a.q_sb + (first + (row_here ? row : 0)) * a.q_sh + 8 * c + 32 * g);

  unsigned char *values = smem + wave * L::wave(FINE), *shares = values + 32 * L::VROW;
  const int64_t page_bytes = P::bytes(a.block) * a.kv_heads;
  const unsigned char *pages = a.pages + P::bytes(a.block) * hk;
  const int value = P::codes(a.block, 1), k_meta = P::meta(a.block, 0);       // where a page's values lie behind its keys, and the steps behind the codes
  const uint32_t own_codes = key * P::ROW + c * (P::ROW / 4), own_meta = key * P::META;

  // 32 pairs at a time, a tile a lane: its page, its first position, how many of its positions count, the heads that see it
  int base = pair, v_page = 0, v_pos = 0, v_info = 0;
  auto look = [&]() {
    const int t = 2 * base + lane;
    int col = t >> a.tile_shift, mask = 0xffff;
    const bool in = t < tiles && (t >> 1) < p_end;
    if (a.rows) {
      const uint32_t e = in ? (uint32_t)a.rows[entry + col] : 0u;
      col = (int)(e >> 16);
      mask = (int)(e & 0xffffu);
    }
    const int sub = t & ((1 << a.tile_shift) - 1);
    v_pos = col * a.block + 16 * sub;
    int n = in ? len - v_pos : 0, page = 0;
    if (n > 0) page = a.table[b * a.table_sb + col];   // (col * block < len, so within the row of the table)
    if (page < 0 || page >= a.n_pages) n = 0;
    n = n < 0 ? 0 : n > 16 ? 16 : n;
    v_page = n > 0 ? page : 0;
    v_info = sub | n << 8 | mask << 16;
  };
  struct Tile { int pos, n, mask; };
  auto fetch = [&](RawTile<BITS, D> &x, int at) {       // tile `at` of the lanes' 64
    const int page = __builtin_amdgcn_readlane(v_page, at), info = __builtin_amdgcn_readlane(v_info, at);
    const int sub = info & 0xff, n = (info >> 8) & 0xff;
    // (addresses of the wavefront, and 32-bit ones of the lane from there)
    const unsigned char *codes = pages + page * page_bytes + 16 * sub * P::ROW, *meta = pages + page * page_bytes + 16 * sub * P::META;
    load_words(x.kc, codes + own_codes);
    load_words(x.vc, codes + value + own_codes);
    load_words(x.km, meta + k_meta + own_meta);
    load_words(x.vm, meta + k_meta + value + own_meta);
    return Tile{__builtin_amdgcn_readlane(v_pos, at), n, (info >> 16) & 0xffff};
  };
  RawTile<BITS, D> raw[2];
  Tile tile[2];
  if (pair < p_end) {                                     // (before q is looked at: loads of which each waits for the last)
    look();
#pragma unroll
    for (int u = 0; u < 2; u++) tile[u] = fetch(raw[u], u);
  }

  // the lane's heads: value j of the lane belongs to the unit's head c * V + j
  const bool capped = a.cap > 0.f;
  float m[V], l[V], factor[V], slope[V], qsum[V][GR];
  h8 qf[GR];
  {
    float x[GR][8], top = 0.f;
#pragma unroll
    for (int g = 0; g < GR; g++) {
#pragma unroll
      for (int i = 0; i < 8; i++) {
        x[g][i] = row_here ? (FINE ? to_float(q[g].h[i]) : to_float(q[g].f[i])) : 0.f;
        top = fmaxf(top, fabsf(x[g][i]));
      }
    }
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    // 2^e so that the largest element is in [2^14, 2^15)
    const int e = top > 0.f && top < INFINITY ? 14 - ilogbf(top) : 0;
#pragma unroll
    for (int g = 0; g < GR; g++) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        qf[g][i] = (_Float16)ldexpf(x[g][i], e - code_up<BITS>(i));
        sum += ldexpf((float)qf[g][i], code_up<BITS>(i) - 24);
      }
      sum += __shfl_xor(sum, 16);
      sum += __shfl_xor(sum, 32);
#pragma unroll
      for (int j = 0; j < V; j++) qsum[j][g] = __shfl(sum, 4 * c + j);
    }
#pragma unroll
    for (int j = 0; j < V; j++) {
      const int r2 = c * V + j, e2 = __shfl(e, 4 * c + j);
      // what a score is multiplied by: the power of two alone may be past fp32's range, and a product that is turns a score of zero into NaN
      factor[j] = fminf(fmaxf(ldexpf(capped ? 2.f * kLog2e * a.scale / a.cap : a.scale * kLog2e, 24 - e2), -__FLT_MAX__), __FLT_MAX__);
      m[j] = r2 < heads ? -INFINITY : 0.f;
      l[j] = 0.f;
      slope[j] = a.slopes && r2 < heads ? a.slopes[first + r2] * kLog2e : 0.f;
    }
  }
  f32x4 o[NT];
#pragma unroll
  for (int n = 0; n < NT; n++) o[n] = f32x4{0.f, 0.f, 0.f, 0.f};

  if (pair < p_end) {
    while (true) {
      // scores and values of the pair
      float y[2][V];
      uint32_t seen = 0;                                  // bit 4 u + j
      uint32_t most = 0;                                  // the greatest step and the greatest least value of the lane's groups, if above zero (or NaN)
#pragma unroll
      for (int u = 0; u < 2; u++) {
        const bool here = key < tile[u].n;                // what lies behind the sequence's end stands for zeros (looked at here and not where it is loaded, which would be waiting for it)
        float s[V];
#pragma unroll
        for (int j = 0; j < V; j++) s[j] = 0.f;
#pragma unroll
        for (int g = 0; g < GR; g++) {
          uint32_t p[4];
          chunk_bits<BITS>(raw[u].kc + g * (BITS / 4), p);
          const f32x4 dot = __builtin_amdgcn_mfma_f32_16x16x32_f16(qf[g], __builtin_bit_cast(h8, u32x4{p[0], p[1], p[2], p[3]}), f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
          const float step = step_of(raw[u].km[g]), least = least_of(raw[u].km[g]);
#pragma unroll
          for (int j = 0; j < V; j++) s[j] = fmaf(step, dot[j], fmaf(least, qsum[j][g], s[j]));
        }
        const float behind = (float)(len - 1 - tile[u].pos - key);
#pragma unroll
        for (int j = 0; j < V; j++) {
          float x = s[j] * factor[j];
          if (capped) {
            asm volatile("");                             // (a branch: not computed where there is no cap)
            x = a.cap * kLog2e * fmaf(-2.f, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x) + 1.f), 1.f);
          }
          y[u][j] = fmaf(-slope[j], behind, x);
          seen |= (here && (tile[u].mask >> (c * V + j) & 1)) ? 1u << (4 * u + j) : 0u;
        }
#pragma unroll
        for (int g = 0; g < GR; g++) {
          f16x2 p[4];
          chunk_codes<BITS>(raw[u].vc + g * (BITS / 4), p);
          const uint32_t meta = here ? raw[u].vm[g] : 0u;
          const f16 step = __builtin_bit_cast(f16, (uint16_t)meta), least = __builtin_bit_cast(f16, (uint16_t)(meta >> 16));
          union { u32x4 w; f16x2 h[4]; } v;
#pragma unroll
          for (int i = 0; i < 4; i++) v.h[i] = __builtin_elementwise_fma(p[i], f16x2{step, step}, f16x2{least, least});
          *reinterpret_cast<u32x4 *>(values + (16 * u + key) * L::VROW + 64 * g + 16 * c) = v.w;
        }
#pragma unroll
        for (int g = 0; g < GR; g += 2) asm("v_pk_maximum3_f16 %0, %0, %1, %2" : "+v"(most) : "v"(raw[u].vm[g]), "v"(raw[u].vm[g + 1]));
      }
      // A step that was rounded up takes the last codes of a group that reaches the end of fp16's range past it: 65504 then, not infinity, which would make
      // NaN of every share that is zero.  least + (2^BITS - 1) * step > 65504 takes a step or a least value of half of that.
      const bool large = __builtin_amdgcn_ballot_w64((most & 0xffffu) >= (BITS == 4 ? 0x6800u : 0x5800u) || most >= 0x78000000u) != 0;    // (2048, 128; 32768)
      // the next pair on its way (into the registers that the scores have come from)
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int j = 0; j < V; j++) asm volatile("" : "+v"(y[u][j]));
      pair++;
      const bool more = pair < p_end;
      if (more) {
        if (pair - base == 32) {
          base = pair;
          look();
        }
#pragma unroll
        for (int u = 0; u < 2; u++) tile[u] = fetch(raw[u], 2 * (pair - base) + u);
      }
      // shares relative to the running maximum, which moves when they grow past 8192
      float e[2][V], sum[V];
      auto exponentials = [&]() {
#pragma unroll
        for (int j = 0; j < V; j++) {
          const float ms = m[j] == -INFINITY ? 0.f : m[j];
          sum[j] = 0.f;
#pragma unroll
          for (int u = 0; u < 2; u++) {
            e[u][j] = seen >> (4 * u + j) & 1 ? __builtin_amdgcn_exp2f(y[u][j] - ms) : 0.f;
            sum[j] += FINE ? e[u][j] : (float)(f16)e[u][j];   // as the product below has them
          }
        }
      };
      exponentials();
      bool move = false;
#pragma unroll
      for (int j = 0; j < V; j++) move |= sum[j] > 8192.f || (m[j] == -INFINITY && (seen & (0x11u << j)));
      const uint64_t moves = __builtin_amdgcn_ballot_w64(move);
      if (large || moves) {                               // (one branch in the usual case)
        if (moves) {
#pragma unroll
          for (int j = 0; j < V; j++) {
            float top = fmaxf(seen >> j & 1 ? y[0][j] : -INFINITY, seen >> (4 + j) & 1 ? y[1][j] : -INFINITY);
#pragma unroll
            for (int d = 1; d < 16; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
            const float mn = fmaxf(m[j], top), f = __builtin_amdgcn_exp2f(m[j] - (mn == -INFINITY ? 0.f : mn));
            l[j] *= f;
#pragma unroll
            for (int n = 0; n < NT; n++) o[n][j] *= f;
            m[j] = mn;
          }
          exponentials();
        }
        if (large) {
#pragma unroll 1
          for (int n = 0; n < 2 * GR; n++) {
            union { u32x4 w; f16 h[8]; } v;
            u32x4 *at = reinterpret_cast<u32x4 *>(values + (16 * (n / GR) + key) * L::VROW + 64 * (n % GR) + 16 * c);
            v.w = *at;
#pragma unroll
            for (int i = 0; i < 8; i++) v.h[i] = v.h[i] > (f16)65504.f ? (f16)65504.f : v.h[i];
            *at = v.w;
          }
        }
      }
#pragma unroll
      for (int j = 0; j < V; j++) {
        l[j] += sum[j];
#pragma unroll
        for (int u = 0; u < 2; u++) *reinterpret_cast<f16 *>(shares + (4 * c + j) * L::PROW + 2 * (16 * u + key)) = (f16)e[u][j];
      }
      if constexpr (FINE)
#pragma unroll
        for (int j = 0; j < V; j++)
#pragma unroll
          for (int u = 0; u < 2; u++) *reinterpret_cast<f16 *>(shares + (16 + 4 * c + j) * L::PROW + 2 * (16 * u + key)) = (f16)(e[u][j] - (float)(f16)e[u][j]);
      asm volatile("" ::: "memory");
      __builtin_amdgcn_wave_barrier();                    // LDS operations of one wavefront complete in order; this only pins the code order
      // (rows of no head hold whatever was there: they come out as rows of no head)
      const h8 pf = *reinterpret_cast<const h8 *>(shares + key * L::PROW + 16 * c);
      const uint32_t vat = (uint32_t)(uintptr_t)BSP_LDS_PTR(values) + (8 * c + (key >> 2)) * L::VROW + 8 * (key & 3);
      auto value_operand = [&](int n) {
        typedef s16x4 __attribute__((address_space(3))) * lds_ptr;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(uintptr_t)(vat + 32 * n)), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(uintptr_t)(vat + 32 * n + 4 * L::VROW));
        typedef short s16x8 __attribute__((ext_vector_type(8)));
        return __builtin_bit_cast(h8, (s16x8)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
      };
      if constexpr (FINE) {
        const h8 pr = *reinterpret_cast<const h8 *>(shares + (16 + key) * L::PROW + 16 * c);
#pragma unroll
        for (int n = 0; n < NT; n++) {
          const h8 vf = value_operand(n);
          o[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pf, vf, o[n], 0, 0, 0);
          o[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pr, vf, o[n], 0, 0, 0);
        }
      } else {
#pragma unroll
        for (int n = 0; n < NT; n++) o[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pf, value_operand(n), o[n], 0, 0, 0);
      }
      asm volatile("" ::: "memory");
      __builtin_amdgcn_wave_barrier();
      if (!more) break;
    }
  }

  // the four wavefronts' results: per head the maximum, the sum, D values
  __syncthreads();
  float *join = reinterpret_cast<float *>(smem);
  constexpr int ROWS = 4 * V, ONE = D + 2;
#pragma unroll
  for (int j = 0; j < V; j++) {
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) l[j] += __shfl_xor(l[j], d);
    float *to = join + (wave * ROWS + c * V + j) * ONE;
    if (key == 0) to[0] = m[j], to[1] = l[j];
#pragma unroll
    for (int n = 0; n < NT; n++) to[2 + 16 * n + key] = o[n][j];
  }
  __syncthreads();
  for (int i = tid; i < heads * (D / 2); i += 256) {
    const int r = i / (D / 2), d = i % (D / 2) * 2;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; w++) top = fmaxf(top, join[(w * ROWS + r) * ONE]);
    float sum = 0.f, x0 = 0.f, x1 = 0.f;
#pragma unroll
    for (int w = 0; w < 4; w++) {
      const float *from = join + (w * ROWS + r) * ONE;
      const float f = from[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(from[0] - top);
      sum = fmaf(f, from[1], sum);
      x0 = fmaf(f, from[2 + d], x0);
      x1 = fmaf(f, from[3 + d], x1);
    }
    if (a.splits > 1) {
      float *to = a.partial + ((((int64_t)b * a.units + unit) * a.splits + split) * a.per + r) * ONE;
      if (d == 0) *reinterpret_cast<f32x2 *>(to) = f32x2{top, sum};
      *reinterpret_cast<f32x2 *>(to + 2 + d) = f32x2{x0, x1};
    } else {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      uint16_t *to = reinterpret_cast<uint16_t *>(a.o) + b * a.o_sb + (first + r) * a.o_sh + d;
      x0 = sum == 0.f ? 0.f : x0 * inv;
      x1 = sum == 0.f ? 0.f : x1 * inv;
      *reinterpret_cast<uint32_t *>(to) = FINE
          ? (uint32_t)__builtin_bit_cast(uint16_t, (f16)x0) | (uint32_t)__builtin_bit_cast(uint16_t, (f16)x1) << 16
          : (uint32_t)__builtin_bit_cast(uint16_t, (bf16)x0) | (uint32_t)__builtin_bit_cast(uint16_t, (bf16)x1) << 16;
    }
  }
}

// The splits of a head joined, a head a wavefront: a split's maximum and sum a lane (so at most 64 splits), then D / 64 elements a lane, the
// loads of eight splits under way at a time.  Splits that saw nothing left zeros and a factor of 0.
template <int D> __global__ void __launch_bounds__(256) k_cache_attention_join(DecodeArgs a, int dtype) {
  constexpr int ONE = D + 2, N = D / 64;
  const int lane = threadIdx.x & 63;
  const int64_t i = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (i >= (int64_t)a.B * a.H) return;
  const int h = (int)(i % a.H), b = (int)(i / a.H);
  const int per_key = (a.G + a.per - 1) / a.per, in_key = h % a.G, unit = h / a.G * per_key + in_key / a.per, r = in_key % a.per;
  const float *from = a.partial + (((int64_t)b * a.units + unit) * a.splits * a.per + r) * ONE;
  const int64_t next = (int64_t)a.per * ONE;
  f32x2 own = {-INFINITY, 0.f};
  if (lane < a.splits) own = *reinterpret_cast<const f32x2 *>(from + lane * next);
  float top = own[0];
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
  const float f = own[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(own[0] - top);
  float sum = f * own[1];
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
  float x[N] = {};
  for (int s = 0; s < a.splits; s += 8) {
    float v[8][N];
#pragma unroll
    for (int u = 0; u < 8; u++) {
      const float *p = from + (s + u < a.splits ? s + u : a.splits - 1) * next + 2 + N * lane;
      if constexpr (N == 2) {
        const f32x2 w = *reinterpret_cast<const f32x2 *>(p);
        v[u][0] = w[0], v[u][1] = w[1];
      } else {
        v[u][0] = *p;
      }
    }
#pragma unroll
    for (int u = 0; u < 8; u++) {
      const float g = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), s + u));    // (0 past the last split)
#pragma unroll
      for (int e = 0; e < N; e++) x[e] = fmaf(g, v[u][e], x[e]);
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  uint16_t *to = reinterpret_cast<uint16_t *>(a.o) + b * a.o_sb + h * a.o_sh + N * lane;
  uint32_t bits = 0;
#pragma unroll
  for (int e = 0; e < N; e++) {
    const float y = sum == 0.f ? 0.f : x[e] * inv;
    bits |= (uint32_t)(dtype == BSP_F16 ? __builtin_bit_cast(uint16_t, (f16)y) : __builtin_bit_cast(uint16_t, (bf16)y)) << (16 * e);
  }
  if constexpr (N == 2) *reinterpret_cast<uint32_t *>(to) = bits;
  else *to = (uint16_t)bits;
}

template <int BITS, int D, bool FINE> void launch_decode(const DecodeArgs &a, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)a.B * a.units * a.splits));
  if (a.per <= 4) hipLaunchKernelGGL((k_cache_attention<BITS, D, 1, FINE>), grid, dim3(256), 0, st, a);
  else if (a.per <= 8) hipLaunchKernelGGL((k_cache_attention<BITS, D, 2, FINE>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((k_cache_attention<BITS, D, 4, FINE>), grid, dim3(256), 0, st, a);
}
template <int BITS, int D> int launch_decode(const DecodeArgs &a, int dtype, hipStream_t st) {
  if (dtype == BSP_F16) launch_decode<BITS, D, true>(a, st);
  else launch_decode<BITS, D, false>(a, st);
  if (a.splits > 1) hipLaunchKernelGGL(k_cache_attention_join<D>, dim3((unsigned)cdiv((int64_t)a.B * a.H, 4)), dim3(256), 0, st, a, dtype);
  BSP_LAUNCH_CHECK();
  return BSP_OK;
}

// Sixteen heads to a workgroup at most, evenly where a key head has more
inline int heads_a_unit(int G) { return (G + (G + 15) / 16 - 1) / ((G + 15) / 16); }

}  // namespace
}  // namespace bsp

using namespace bsp;

// Workgroups to split a sequence's positions over, `blocks` blocks at most (lengths are on the device): enough for three a compute unit, each with at
// least eight pairs of tiles a wavefront.
extern "C" int bsp_cache_attention_splits(int B, int H, int kv_heads, int block, int64_t blocks) {
  if (B <= 0 || H <= 0 || kv_heads <= 0 || H % kv_heads || block <= 0 || blocks <= 0) return BSP_ERR_ARG;
  const int G = H / kv_heads, per = heads_a_unit(G);
  const int64_t groups = (int64_t)B * kv_heads * ((G + per - 1) / per), pairs = (blocks * block + 31) / 32;
  int64_t n = (768 + groups - 1) / groups;
  if (n > pairs / 32) n = pairs / 32;
  return (int)(n < 1 ? 1 : n > 64 ? 64 : n);
}

extern "C" int64_t bsp_cache_attention_workspace_bytes(int B, int H, int kv_heads, int D, int splits) {
  if (B <= 0 || H <= 0 || kv_heads <= 0 || H % kv_heads || splits <= 0) return BSP_ERR_ARG;
  const int G = H / kv_heads, per = heads_a_unit(G);
  return splits > 1 ? (int64_t)B * kv_heads * ((G + per - 1) / per) * per * splits * (D + 2) * 4 : 0;
}

extern "C" int bsp_cache_attention(int dtype, const void *q, int64_t q_stride_b, int64_t q_stride_h, void *o, int64_t o_stride_b, int64_t o_stride_h, int B, int H,
                                   const void *pages, int n_pages, int block, int kv_heads, int D, int bits, const int32_t *table, int64_t table_stride, int width,
                                   const int32_t *lengths, const int32_t *rows, int n_rows, int64_t most_blocks, float scale, float softcap, const float *slopes,
                                   void *workspace, int64_t workspace_bytes, int splits, void *stream) {
  if (!q || !o || !pages || !table || !lengths || B <= 0 || H <= 0 || kv_heads <= 0 || H % kv_heads || n_pages <= 0 || width <= 0 || splits < 1 || splits > 64) return BSP_ERR_ARG;
  if ((dtype != BSP_F16 && dtype != BSP_BF16) || bsp_cache_page_bytes(block, kv_heads, D, bits) <= 0) return BSP_ERR_UNSUPPORTED;
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(pages)) & 15) || (reinterpret_cast<uintptr_t>(o) & 3) || q_stride_b % 8 || q_stride_h % 8 || o_stride_b % 2 || o_stride_h % 2) return BSP_ERR_ARG;
  if (!scores_ok(scale, softcap) || (rows && n_rows <= 0) || most_blocks <= 0) return BSP_ERR_ARG;
  if ((int64_t)width * block >= ((int64_t)1 << 24) || (int64_t)n_pages * block >= ((int64_t)1 << 31) || (rows && n_rows > 65536)) return BSP_ERR_UNSUPPORTED;
  const int64_t need = bsp_cache_attention_workspace_bytes(B, H, kv_heads, D, splits);
  if (need > 0 && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) || workspace_bytes < need)) return BSP_ERR_CAPACITY;
  DecodeArgs a{};
  a.G = H / kv_heads;
  a.per = heads_a_unit(a.G);
  a.units = kv_heads * ((a.G + a.per - 1) / a.per);
  if ((int64_t)B * a.units * splits * 256 >= ((int64_t)1 << 32) || (int64_t)B * H * 64 + 256 >= ((int64_t)1 << 32)) return BSP_ERR_UNSUPPORTED;   // (a grid has fewer than 2^32 threads)
  a.q = q; a.q_sb = q_stride_b; a.q_sh = q_stride_h; a.o = o; a.o_sb = o_stride_b; a.o_sh = o_stride_h;
  a.pages = reinterpret_cast<const unsigned char *>(pages); a.n_pages = n_pages;
  a.table = table; a.table_sb = table_stride; a.width = width; a.lengths = lengths;
  a.rows = rows; a.n_rows = n_rows; a.slopes = slopes; a.scale = scale; a.cap = softcap;
  a.partial = reinterpret_cast<float *>(workspace);
  a.B = B; a.H = H; a.kv_heads = kv_heads; a.block = block; a.splits = splits;
  const int64_t pairs = (most_blocks * block + 31) / 32;
  a.chunk = (int)((pairs + 4 * splits - 1) / (4 * splits));
  a.tile_shift = block == 16 ? 0 : block == 32 ? 1 : block == 64 ? 2 : 3;
  const hipStream_t st = as_stream(stream);
  if (bits == 4) return D == 64 ? launch_decode<4, 64>(a, dtype, st) : launch_decode<4, 128>(a, dtype, st);
  return D == 64 ? launch_decode<8, 64>(a, dtype, st) : launch_decode<8, 128>(a, dtype, st);
}
