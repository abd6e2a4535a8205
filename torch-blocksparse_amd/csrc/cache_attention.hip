// Attention of one new position a sequence over a quantised cache (cache.h): for sequence b of length n and query head h
//     y_j = cap * tanh(scale * q . k_j / cap) - slope_h * (n - 1 - j),   o = softmax(y) . v
// over the positions j < n whose page the sequence holds and, with a layout, whose block is in row (n - 1) / block of head h.
//
// What bounds it is the cache: every byte of the pages that are seen is read once for all the query heads that share a key head (up
// to 16 a workgroup).  Each of a workgroup's four wavefronts goes through its own pairs of tiles of sixteen positions, a pair's
// codes and steps on their way while the one before is computed, and the wavefronts' results are joined in LDS.  Where sequences and
// key heads do not fill the chip the positions are split among workgroups, and a second kernel joins what those leave.
//
// The codes are operands as they are: small integers are exact in fp16, so a score is the sum over the groups of step * (q . codes) +
// least * (sum of the group's q), the products on the matrix units (16 x 16 x 32: a group each).  q is scaled by a power of two per head to the
// range of fp16, which loses nothing that 2^-35 of its largest element would not.  Values are v = least + code * step rounded to fp16
// (2^-12 of it, under the rounding of the shares) through LDS, where the product with the shares reads them transposed.
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
  int G, per, units, splits;       // query heads a key head; heads of a unit (a workgroup's), units
};

namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));

template <int BITS, int D> struct RawTile {
  static constexpr int QB = D * BITS / 32 / 4;            // 32-bit words of a quarter row
  static constexpr int GROUPS = D / 32;
  uint32_t kc[QB], vc[QB], km[GROUPS], vm[GROUPS];
};
template <int N> __device__ __forceinline__ void load_words(uint32_t (&w)[N], const unsigned char *p) {
  if constexpr (N == 2) {
    const u32x2 x = *reinterpret_cast<const u32x2 *>(p);
    w[0] = x[0], w[1] = x[1];
  } else {
#pragma unroll
    for (int i = 0; i < N / 4; i++) {
      const u32x4 x = *reinterpret_cast<const u32x4 *>(p + 16 * i);
#pragma unroll
      for (int j = 0; j < 4; j++) w[4 * i + j] = x[j];
    }
  }
}
__device__ __forceinline__ float step_of(uint32_t meta) { return (float)__builtin_bit_cast(f16, (uint16_t)meta); }
__device__ __forceinline__ float least_of(uint32_t meta) { return (float)__builtin_bit_cast(f16, (uint16_t)(meta >> 16)); }
template <int BITS, int D> struct DecodeLds {
  static constexpr int VROW = 2 * D + 16, PROW = 80;      // bytes of a position's values, of a head's 32 shares
  static constexpr int WAVE = 32 * VROW + 16 * PROW;
  static constexpr int join(int V) { return 4 * 4 * V * (D + 2) * 4; }
  static constexpr int bytes(int V) { return 4 * WAVE > join(V) ? 4 * WAVE : join(V); }
};

template <int BITS, int D, int V>
__global__ void __launch_bounds__(256, 3) k_cache_attention(DecodeArgs a, int dtype) {
  typedef Page<BITS, D> P;
  typedef DecodeLds<BITS, D> L;
  constexpr int GR = D / 32, NT = D / 16;
  __shared__ __attribute__((aligned(16))) unsigned char smem[L::bytes(V)];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), key = lane & 15, c = lane >> 4;
  const int64_t wg = xcd_remap(blockIdx.x, (int64_t)a.B * a.units * a.splits);
  const int split = (int)(wg % a.splits), unit = (int)(wg / a.splits % a.units), b = (int)(wg / a.splits / a.units);
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
  // this wavefront's pairs of tiles
  const int pairs = (tiles + 1) >> 1, parts = a.splits * 4, part = split * 4 + wave;
  const int p_end = (int)((int64_t)pairs * (part + 1) / parts);
  int pair = (int)((int64_t)pairs * part / parts);

  // the lane's heads: value j of the lane belongs to the unit's head c * V + j; row m of a product's first operand to head (m / 4) * V + m % 4
  float m[V], l[V], unscale[V], slope[V], qsum[V][GR];
  h8 qf[GR];
  {
    const int r = (key >> 2) * V + (key & 3);
    const bool here = (key & 3) < V && r < heads;
    float x[GR][8], top = 0.f;
    const int64_t at = b * a.q_sb + (first + (here ? r : 0)) * a.q_sh + 8 * c;
#pragma unroll
    for (int g = 0; g < GR; g++) {
      union { u32x4 raw; f16 h[8]; bf16 f[8]; } u;
      u.raw = *reinterpret_cast<const u32x4 *>(reinterpret_cast<const uint16_t *>(a.q) + at + 32 * g);
#pragma unroll
      for (int i = 0; i < 8; i++) {
        x[g][i] = here ? (dtype == BSP_F16 ? to_float(u.h[i]) : to_float(u.f[i])) : 0.f;
        top = fmaxf(top, fabsf(x[g][i]));
      }
    }
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    // 2^e so that the largest element is in [1024, 2048)
    const int e = top > 0.f && top < INFINITY ? 10 - ilogbf(top) : 0;
#pragma unroll
    for (int g = 0; g < GR; g++) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        qf[g][i] = (_Float16)ldexpf(x[g][i], e);
        sum += (float)qf[g][i];
      }
      sum += __shfl_xor(sum, 16);
      sum += __shfl_xor(sum, 32);
#pragma unroll
      for (int j = 0; j < V; j++) qsum[j][g] = __shfl(sum, 4 * c + j);
    }
#pragma unroll
    for (int j = 0; j < V; j++) {
      const int r2 = c * V + j, e2 = __shfl(e, 4 * c + j);
      unscale[j] = ldexpf(1.f, -e2);
      m[j] = r2 < heads ? -INFINITY : 0.f;
      l[j] = 0.f;
      slope[j] = a.slopes && r2 < heads ? a.slopes[first + r2] * kLog2e : 0.f;
    }
  }
  const bool capped = a.cap > 0.f;
  f32x4 o[NT];
#pragma unroll
  for (int n = 0; n < NT; n++) o[n] = f32x4{0.f, 0.f, 0.f, 0.f};

  unsigned char *values = smem + wave * L::WAVE, *shares = values + 32 * L::VROW;
  const int64_t page_bytes = P::bytes(a.block) * a.kv_heads;
  const unsigned char *pages = a.pages + P::bytes(a.block) * hk;
  const int k_codes = P::codes(a.block, 0) + c * (P::ROW / 4), v_codes = P::codes(a.block, 1) + c * (P::ROW / 4), k_meta = P::meta(a.block, 0), v_meta = P::meta(a.block, 1);

  if (pair < p_end) {
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
    look();
    struct Tile { int pos, n, mask; };
    auto fetch = [&](RawTile<BITS, D> &x, int at) {       // tile `at` of the lanes' 64
      const int page = __builtin_amdgcn_readlane(v_page, at), info = __builtin_amdgcn_readlane(v_info, at);
      const int row = 16 * (info & 0xff) + key, n = (info >> 8) & 0xff;
      const unsigned char *from = pages + page * page_bytes;
      load_words(x.kc, from + k_codes + row * P::ROW);
      load_words(x.vc, from + v_codes + row * P::ROW);
      load_words(x.km, from + k_meta + row * P::META);
      load_words(x.vm, from + v_meta + row * P::META);
      const bool here = key < n;                          // what lies behind the sequence's end stands for zeros
#pragma unroll
      for (int g = 0; g < GR; g++) x.km[g] = here ? x.km[g] : 0u, x.vm[g] = here ? x.vm[g] : 0u;
      return Tile{__builtin_amdgcn_readlane(v_pos, at), n, (info >> 16) & 0xffff};
    };
    RawTile<BITS, D> raw[2];
    Tile tile[2];
#pragma unroll
    for (int u = 0; u < 2; u++) tile[u] = fetch(raw[u], u);
    while (true) {
      // scores and values of the pair
      float y[2][V];
      uint32_t seen = 0;                                  // bit 4 u + j
#pragma unroll
      for (int u = 0; u < 2; u++) {
        float s[V];
#pragma unroll
        for (int j = 0; j < V; j++) s[j] = 0.f;
#pragma unroll
        for (int g = 0; g < GR; g++) {
          f16x2 p[4];
          chunk_codes<BITS>(raw[u].kc + g * (BITS / 4), p);
          h8 kf;
#pragma unroll
          for (int i = 0; i < 8; i++) kf[i] = p[i >> 1][i & 1];
          const f32x4 dot = __builtin_amdgcn_mfma_f32_16x16x32_f16(qf[g], kf, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
          const float step = step_of(raw[u].km[g]), least = least_of(raw[u].km[g]);
#pragma unroll
          for (int j = 0; j < V; j++) s[j] = fmaf(step, dot[j], fmaf(least, qsum[j][g], s[j]));
        }
        const float behind = (float)(len - 1 - tile[u].pos - key);
#pragma unroll
        for (int j = 0; j < V; j++) {
          float x = s[j] * unscale[j];
          if (capped) x = a.cap * kLog2e * fmaf(-2.f, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x * (2.f * kLog2e * a.scale / a.cap)) + 1.f), 1.f);
          else x *= a.scale * kLog2e;
          y[u][j] = fmaf(-slope[j], behind, x);
          seen |= (key < tile[u].n && (tile[u].mask >> (c * V + j) & 1)) ? 1u << (4 * u + j) : 0u;
        }
#pragma unroll
        for (int g = 0; g < GR; g++) {
          f16x2 p[4];
          chunk_codes<BITS>(raw[u].vc + g * (BITS / 4), p);
          const f16 step = __builtin_bit_cast(f16, (uint16_t)raw[u].vm[g]), least = __builtin_bit_cast(f16, (uint16_t)(raw[u].vm[g] >> 16));
          union { u32x4 w; f16x2 h[4]; } v;
#pragma unroll
          for (int i = 0; i < 4; i++) v.h[i] = __builtin_elementwise_fma(p[i], f16x2{step, step}, f16x2{least, least});
          *reinterpret_cast<u32x4 *>(values + (16 * u + key) * L::VROW + 64 * g + 16 * c) = v.w;
        }
      }
      // the next pair on its way
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
            sum[j] += e[u][j];
          }
        }
      };
      exponentials();
      bool move = false;
#pragma unroll
      for (int j = 0; j < V; j++) move |= sum[j] > 8192.f || (m[j] == -INFINITY && (seen & (0x11u << j)));
      if (__builtin_amdgcn_ballot_w64(move)) {
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
#pragma unroll
      for (int j = 0; j < V; j++) {
        l[j] += sum[j];
#pragma unroll
        for (int u = 0; u < 2; u++) *reinterpret_cast<f16 *>(shares + (4 * c + j) * L::PROW + 2 * (16 * u + key)) = (f16)e[u][j];
      }
      asm volatile("" ::: "memory");
      __builtin_amdgcn_wave_barrier();                    // LDS operations of one wavefront complete in order; this only pins the code order
      // (rows of no head hold whatever was there: they come out as rows of no head)
      const h8 pf = *reinterpret_cast<const h8 *>(shares + key * L::PROW + 16 * c);
      const uint32_t vat = (uint32_t)(uintptr_t)BSP_LDS_PTR(values) + (8 * c + (key >> 2)) * L::VROW + 8 * (key & 3);
#pragma unroll
      for (int n = 0; n < NT; n++) {
        typedef s16x4 __attribute__((address_space(3))) * lds_ptr;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(uintptr_t)(vat + 32 * n)), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(uintptr_t)(vat + 32 * n + 4 * L::VROW));
        typedef short s16x8 __attribute__((ext_vector_type(8)));
        const h8 vf = __builtin_bit_cast(h8, (s16x8)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        o[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pf, vf, o[n], 0, 0, 0);
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
      if (d == 0) to[0] = top, to[1] = sum;
      to[2 + d] = x0;
      to[3 + d] = x1;
    } else {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      uint16_t *to = reinterpret_cast<uint16_t *>(a.o) + b * a.o_sb + (first + r) * a.o_sh + d;
      x0 = sum == 0.f ? 0.f : x0 * inv;
      x1 = sum == 0.f ? 0.f : x1 * inv;
      *reinterpret_cast<uint32_t *>(to) = dtype == BSP_F16
          ? (uint32_t)__builtin_bit_cast(uint16_t, (f16)x0) | (uint32_t)__builtin_bit_cast(uint16_t, (f16)x1) << 16
          : (uint32_t)__builtin_bit_cast(uint16_t, (bf16)x0) | (uint32_t)__builtin_bit_cast(uint16_t, (bf16)x1) << 16;
    }
  }
}

// The splits of a head joined: two elements a thread
template <int D> __global__ void __launch_bounds__(256) k_cache_attention_join(DecodeArgs a, int dtype) {
  constexpr int ONE = D + 2;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (int64_t)a.B * a.H * (D / 2)) return;
  const int d = (int)(i % (D / 2)) * 2, h = (int)(i / (D / 2) % a.H), b = (int)(i / (D / 2) / a.H);
  const int per_key = (a.G + a.per - 1) / a.per, in_key = h % a.G, unit = h / a.G * per_key + in_key / a.per, r = in_key % a.per;
  const float *from = a.partial + (((int64_t)b * a.units + unit) * a.splits * a.per + r) * ONE;
  float top = -INFINITY;
  for (int s = 0; s < a.splits; s++) top = fmaxf(top, from[(int64_t)s * a.per * ONE]);
  float sum = 0.f, x0 = 0.f, x1 = 0.f;
  for (int s = 0; s < a.splits; s++) {
    const float *p = from + (int64_t)s * a.per * ONE;
    const float f = p[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(p[0] - top);
    sum = fmaf(f, p[1], sum);
    x0 = fmaf(f, p[2 + d], x0);
    x1 = fmaf(f, p[3 + d], x1);
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  x0 = sum == 0.f ? 0.f : x0 * inv;
  x1 = sum == 0.f ? 0.f : x1 * inv;
  uint16_t *to = reinterpret_cast<uint16_t *>(a.o) + b * a.o_sb + h * a.o_sh + d;
  *reinterpret_cast<uint32_t *>(to) = dtype == BSP_F16
      ? (uint32_t)__builtin_bit_cast(uint16_t, (f16)x0) | (uint32_t)__builtin_bit_cast(uint16_t, (f16)x1) << 16
      : (uint32_t)__builtin_bit_cast(uint16_t, (bf16)x0) | (uint32_t)__builtin_bit_cast(uint16_t, (bf16)x1) << 16;
}

template <int BITS, int D> int launch_decode(const DecodeArgs &a, int dtype, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)a.B * a.units * a.splits));
  if (a.per <= 4) hipLaunchKernelGGL((k_cache_attention<BITS, D, 1>), grid, dim3(256), 0, st, a, dtype);
  else if (a.per <= 8) hipLaunchKernelGGL((k_cache_attention<BITS, D, 2>), grid, dim3(256), 0, st, a, dtype);
  else hipLaunchKernelGGL((k_cache_attention<BITS, D, 4>), grid, dim3(256), 0, st, a, dtype);
  if (a.splits > 1) hipLaunchKernelGGL(k_cache_attention_join<D>, dim3((unsigned)cdiv((int64_t)a.B * a.H * (D / 2), 256)), dim3(256), 0, st, a, dtype);
  BSP_LAUNCH_CHECK();
  return BSP_OK;
}

// Sixteen heads to a workgroup at most, evenly where a key head has more
inline int heads_a_unit(int G) { return (G + (G + 15) / 16 - 1) / ((G + 15) / 16); }

}  // namespace
}  // namespace bsp

using namespace bsp;

// Workgroups to split a sequence's positions over: enough for four a compute unit, each with eight pairs of tiles a wavefront
// at least if the longest sequence fills its row of the table (lengths are on the device).
extern "C" int bsp_cache_attention_splits(int B, int H, int kv_heads, int block, int64_t blocks) {
  if (B <= 0 || H <= 0 || kv_heads <= 0 || H % kv_heads || block <= 0 || blocks <= 0) return BSP_ERR_ARG;
  const int G = H / kv_heads, per = heads_a_unit(G);
  const int64_t groups = (int64_t)B * kv_heads * ((G + per - 1) / per), pairs = (blocks * block + 31) / 32;
  int64_t n = (1024 + groups - 1) / groups;
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
                                   const int32_t *lengths, const int32_t *rows, int n_rows, float scale, float softcap, const float *slopes, void *workspace,
                                   int64_t workspace_bytes, int splits, void *stream) {
  if (!q || !o || !pages || !table || !lengths || B <= 0 || H <= 0 || kv_heads <= 0 || H % kv_heads || n_pages <= 0 || width <= 0 || splits < 1 || splits > 64) return BSP_ERR_ARG;
  if ((dtype != BSP_F16 && dtype != BSP_BF16) || bsp_cache_page_bytes(block, kv_heads, D, bits) <= 0) return BSP_ERR_UNSUPPORTED;
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(pages)) & 15) || (reinterpret_cast<uintptr_t>(o) & 3) || q_stride_b % 8 || q_stride_h % 8 || o_stride_b % 2 || o_stride_h % 2) return BSP_ERR_ARG;
  if (!(scale - scale == 0.f) || !(softcap >= 0.f) || !(softcap - softcap == 0.f) || (rows && n_rows <= 0)) return BSP_ERR_ARG;
  if ((int64_t)width * block >= ((int64_t)1 << 24) || (int64_t)n_pages * block >= ((int64_t)1 << 31) || (rows && n_rows > 65536)) return BSP_ERR_UNSUPPORTED;
  const int64_t need = bsp_cache_attention_workspace_bytes(B, H, kv_heads, D, splits);
  if (need > 0 && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) || workspace_bytes < need)) return BSP_ERR_CAPACITY;
  DecodeArgs a{};
  a.G = H / kv_heads;
  a.per = heads_a_unit(a.G);
  a.units = kv_heads * ((a.G + a.per - 1) / a.per);
  if ((int64_t)B * a.units * splits >= ((int64_t)1 << 31)) return BSP_ERR_UNSUPPORTED;
  a.q = q; a.q_sb = q_stride_b; a.q_sh = q_stride_h; a.o = o; a.o_sb = o_stride_b; a.o_sh = o_stride_h;
  a.pages = reinterpret_cast<const unsigned char *>(pages); a.n_pages = n_pages;
  a.table = table; a.table_sb = table_stride; a.width = width; a.lengths = lengths;
  a.rows = rows; a.n_rows = n_rows; a.slopes = slopes; a.scale = scale; a.cap = softcap;
  a.partial = reinterpret_cast<float *>(workspace);
  a.B = B; a.H = H; a.kv_heads = kv_heads; a.block = block; a.splits = splits;
  a.tile_shift = block == 16 ? 0 : block == 32 ? 1 : block == 64 ? 2 : 3;
  const hipStream_t st = as_stream(stream);
  if (bits == 4) return D == 64 ? launch_decode<4, 64>(a, dtype, st) : launch_decode<4, 128>(a, dtype, st);
  return D == 64 ? launch_decode<8, 64>(a, dtype, st) : launch_decode<8, 128>(a, dtype, st);
}
