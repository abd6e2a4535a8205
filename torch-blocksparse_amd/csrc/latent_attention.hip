// Attention of one new position a sequence over a cache of latent vectors (latent.h), the absorbed form: every head's key of position j is the latent vector c_j and the
// shared part r_j, its value is c_j:
//     y_j = cap * tanh(scale * (q . c_j + q_r . r_j) / cap) - slope_h * (n - 1 - j),   o = sum_j softmax_j(y) c_j        (no cap: scale * (q . c_j + q_r . r_j) - ...)
// over the positions j < n whose page the sequence holds and, with a layout, whose block is in row (n - 1) / block of head h.
//
// Each byte of the pages is read once for all heads of a workgroup (up to 64) and is key and value at once, so it goes to LDS, straight from global memory. A wavefront has
// sixteen heads.  Both products are taken transposed on the matrix units (16 x 16 x 32): scores as positions x heads, results as elements x heads.  A lane then has one head, so
// maximum, sum and rescaling are single registers, and the shares a lane has computed are the operand of the second product as they are: its other operand, positions across, comes from
// LDS by transposing reads in the same order of positions.
//
// A step of a workgroup is 64 positions: four groups of sixteen, each wavefront loads one.  With at most sixteen heads (HW = 1) each wavefront goes through groups of its own and
// needs no barrier; with up to 32 (HW = 2) two wavefronts, with more all four share their groups.
//
// All steps of all sequences are one row of work that is cut into equal pieces, one a workgroup, so that uneven lengths leave no compute unit idle: a workgroup finds its piece by
// a sum over the lengths.  A sequence that lies in several pieces is joined by a second kernel.
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
  float *partial;                  // two slots a workgroup, [heads a unit][latent + 2]: maximum, sum, sums
  int32_t *meta;                   // per item (sequence and unit) three ints: the workgroup that begins it, how many have a part (0, 1: nothing to join), the first part's slot
  int B, H, block, shift;          // shift: log2 of the groups of sixteen positions a block
  int units, per, pieces;          // workgroups' heads a sequence: units of `per`; pieces of the work
};

namespace {

template <typename T> struct Latent16;
template <> struct Latent16<f16> {
  typedef f16x8 frag8; typedef f16x4 frag4;
  static __device__ __forceinline__ f32x4 run(frag8 a, frag8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ f32x4 run(frag4 a, frag4 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x16f16(a, b, c, 0, 0, 0); }
};
template <> struct Latent16<bf16> {
  typedef bf16x8 frag8; typedef bf16x4 frag4;
  static __device__ __forceinline__ f32x4 run(frag8 a, frag8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ f32x4 run(frag4 a, frag4 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, a), __builtin_bit_cast(s16x4, b), c, 0, 0, 0); }
};

template <int LAT> struct LatentGeo {
  static constexpr int ROW = 2 * (LAT + kRope), LROW = 2 * LAT;               // bytes of a position, of its latent vector
  static constexpr int GROUP = 16 * ROW, STAGE = 4 * GROUP, RING = 2 * STAGE;   // sixteen positions: their latent vectors, then their shared parts
  static constexpr int JOIN = LAT + 4;                                         // floats of a head's sums when wavefronts are joined
  static constexpr int LDS = RING + 64 * 2 * 4;
  static_assert(64 * JOIN * 4 <= RING, "");
};

// where 16-byte chunk `chunk` of row r of a group lies: latent vectors with the chunks of 256 bytes exchanged by r, so that sixteen rows' reads of a chunk take sixteen places of
// the 64 banks, and so do transposing reads of eight rows' pairs of chunks; shared parts, of which two rows fill 256 bytes, by r / 2
__device__ __forceinline__ uint32_t latent_chunk(uint32_t chunk, uint32_t r) { return chunk ^ r; }
__device__ __forceinline__ uint32_t rope_chunk(uint32_t chunk, uint32_t r) { return chunk ^ (r >> 1); }

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

// An item is a sequence and a unit of its heads; its groups of sixteen positions
struct LatentItem {
  int b, unit, len, groups, entry;
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
    }
  }
  __device__ __forceinline__ int steps() const { return (groups + 3) >> 2; }
};

template <typename T, int LAT, int HW>
__global__ void __launch_bounds__(256, 1) k_latent_attention(LatentArgs a) {
  typedef LatentGeo<LAT> G;
  typedef Latent16<T> M;
  typedef typename M::frag8 frag8;
  typedef typename M::frag4 frag4;
  constexpr int NS = LAT / 32, NR = kRope / 32, NT = LAT / 16;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), key = lane & 15, c = lane >> 4;
  const int hw = wave % HW, mine = wave / HW * HW;                            // the wavefront's heads 16 hw .. of the unit; the first of the HW groups of a step that it goes through
  const uint32_t items = (uint32_t)(a.B * a.units), ring = (uint32_t)(uintptr_t)BSP_LDS_PTR(smem);

  // the workgroup's piece [lo, hi) of all steps, and the item that it begins in
  int64_t total = 0, lo, hi, begin = 0;
  uint32_t item = 0;
  int pieces;
  {
    int *sums = reinterpret_cast<int *>(smem + G::RING);                      // (where no tile goes)
    auto chunk_sum = [&](uint32_t base, int &own, int &before) {               // of 256 items: own steps, those of the items before it in the chunk; returns the chunk's
      const uint32_t i = base + tid;
      own = i < items ? LatentItem(a, i).steps() : 0;
      int x = own;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl_up(x, d);
        if (lane >= d) x += y;
      }
      __syncthreads();
      if (lane == 63) sums[wave] = x;
      __syncthreads();
      int all = 0;
      before = x - own;
#pragma unroll
      for (int w = 0; w < 4; w++) {
        before += w < wave ? sums[w] : 0;
        all += sums[w];
      }
      return __builtin_amdgcn_readfirstlane(all);
    };
    int own = 0, before = 0;
    for (uint32_t base = 0; base < items; base += 256) {
      total += chunk_sum(base, own, before);
      const uint32_t i = base + tid;
      if (i < items && own == 0) {                                            // nothing is seen: zeros
        if (blockIdx.x == 0) a.meta[3 * (int64_t)i + 1] = 0;
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
    pieces = total < a.pieces ? (int)total : a.pieces;    // (none is empty)
    if ((int)blockIdx.x >= pieces) return;
    lo = total * blockIdx.x / pieces;
    hi = total * (blockIdx.x + 1) / pieces;
    int64_t done = 0;
    for (uint32_t base = 0; base < items; base += 256) {
      if (items > 256 || base > 0) {
        const int all = chunk_sum(base, own, before);
        if (done + all <= lo) {
          done += all;
          continue;
        }
      }
      __syncthreads();
      if (own > 0 && done + before <= lo && lo < done + before + own) sums[4] = (int)base + tid, sums[5] = before;
      __syncthreads();
      item = (uint32_t)__builtin_amdgcn_readfirstlane(sums[4]);
      begin = done + __builtin_amdgcn_readfirstlane(sums[5]);
      break;
    }
  }

  const bool capped = a.cap > 0.f;
  const float factor = capped ? 2.f * kLog2e * a.scale / a.cap : a.scale * kLog2e, top_of_cap = a.cap * kLog2e;
  // addresses in a group: of the lane's row (positions across the matrix rows), and of the transposing reads
  const uint32_t row_at = key * G::LROW + (latent_chunk(c, key) << 4), rope_at = 16 * G::LROW + key * (2 * kRope) + (rope_chunk(c, key) << 4);
  const uint32_t tr_row = 4 * c + (key >> 2), tr_at = tr_row * G::LROW + (latent_chunk((key & 3) >> 1, tr_row) << 4) + 8 * (key & 1);

  for (int64_t at = lo; at < hi && item < items; item++) {
    const LatentItem it(a, item);
    const int steps = __builtin_amdgcn_readfirstlane(it.steps());
    if (steps == 0) continue;
    const int b = __builtin_amdgcn_readfirstlane(it.b), unit = __builtin_amdgcn_readfirstlane(it.unit), len = __builtin_amdgcn_readfirstlane(it.len);
    const int groups = __builtin_amdgcn_readfirstlane(it.groups), entry = __builtin_amdgcn_readfirstlane(it.entry);
    const int s0 = (int)(at - begin), s1 = begin + steps < hi ? steps : (int)(hi - begin);
    const int first = unit * a.per, heads = a.H - first < a.per ? a.H - first : a.per;
    const int head = 16 * hw + key;                       // the lane's head among the unit's
    const bool head_here = head < heads;

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
    struct Group { int pos, n, mask; };
    auto group_of = [&](int i) {
      const int lo32 = __builtin_amdgcn_readlane(v_lo, i), hi32 = __builtin_amdgcn_readlane(v_hi, i);
      return Group{__builtin_amdgcn_readlane(v_pos, i), __builtin_amdgcn_readlane(v_n, i), ((hw & 2 ? hi32 : lo32) >> (16 * (hw & 1))) & 0xffff};
    };
    // the wavefront's group of step s on its way to its place in stage s % 2
    auto issue = [&](int s) {
      const int i = 4 * (s - base) + wave;
      const int page = __builtin_amdgcn_readlane(v_page, i), sub = __builtin_amdgcn_readlane(v_sub, i), n = __builtin_amdgcn_readlane(v_n, i);
      const uint64_t from = reinterpret_cast<uint64_t>(a.pages) + ((int64_t)page * a.block + 16 * sub) * (int64_t)G::ROW;
      const i32x4b rows = {(int)(uint32_t)from, (int)(uint32_t)(from >> 32) & 0xffff, n * G::ROW, 0x00020000};
      const uint32_t dst = __builtin_amdgcn_readfirstlane(ring + (s & 1) * G::STAGE + wave * G::GROUP);
      constexpr int CPR = G::LROW / 16, RPI = 64 / CPR;   // chunks of a row, rows of a load
#pragma unroll
      for (int k = 0; k < 16 / RPI; k++) {
        const uint32_t r = k * RPI + lane / CPR;
        rows_to_lds(rows, r * G::ROW + (latent_chunk(lane % CPR, r) << 4), dst + k * 1024);
      }
#pragma unroll
      for (int k = 0; k < 2; k++) {
        const uint32_t r = 8 * k + lane / 8;
        rows_to_lds(rows, r * G::ROW + G::LROW + (rope_chunk(lane % 8, r) << 4), dst + 16 * G::LROW + k * 1024);
      }
    };

    look();
    issue(s0);
    Group now[HW], next[HW];
#pragma unroll
    for (int k = 0; k < HW; k++) now[k] = group_of(mine + k);

    // queries: the second operand, a head a lane
    frag8 q[NS], qr[NR];
    float slope = 0.f;
    {
      const T *pq = reinterpret_cast<const T *>(a.q) + b * a.q_sb + (first + (head_here ? head : 0)) * a.q_sh + 8 * c;
      const T *pr = reinterpret_cast<const T *>(a.qr) + b * a.qr_sb + (first + (head_here ? head : 0)) * a.qr_sh + 8 * c;
#pragma unroll
      for (int s = 0; s < NS; s++) q[s] = __builtin_bit_cast(frag8, head_here ? *reinterpret_cast<const u32x4 *>(pq + 32 * s) : u32x4{0, 0, 0, 0});
#pragma unroll
      for (int s = 0; s < NR; s++) qr[s] = __builtin_bit_cast(frag8, head_here ? *reinterpret_cast<const u32x4 *>(pr + 32 * s) : u32x4{0, 0, 0, 0});
      if (a.slopes && head_here) slope = a.slopes[first + head] * kLog2e;
    }
    float m = -INFINITY, l = 0.f;
    f32x4 o[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) o[n] = f32x4{0.f, 0.f, 0.f, 0.f};

    for (int s = s0; s < s1; s++) {
      BSP_WAIT_VM(0);
      asm volatile("" ::: "memory");
      if constexpr (HW > 1) {
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
      }
      if (s + 1 < s1) {
        if (s + 1 - base == 16) {
          base = s + 1;
          look();
        }
        issue(s + 1);
#pragma unroll
        for (int k = 0; k < HW; k++) next[k] = group_of(4 * (s + 1 - base) + mine + k);
      }
      const uint32_t stage = ring + (s & 1) * G::STAGE + mine * G::GROUP;
      // scores: value 4 k + i is that of position 4 c + i of group k
      float y[4 * HW];
      uint32_t seen = 0;
#pragma unroll
      for (int k = 0; k < HW; k++) {
        f32x4 acc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
        const uint32_t group = stage + k * G::GROUP;
#pragma unroll
        for (int t = 0; t < NS; t++) acc[t & 1] = M::run(latent_read<frag8>((group + (row_at ^ ((t & 3) << 6))) + (t >> 2) * 256), q[t], acc[t & 1]);
#pragma unroll
        for (int t = 0; t < NR; t++) acc[t & 1] = M::run(latent_read<frag8>(group + (rope_at ^ (t << 6))), qr[t], acc[t & 1]);
        const bool sees = head_here && (now[k].mask >> key & 1);
        const float behind = (float)(len - 1 - now[k].pos - 4 * c);
#pragma unroll
        for (int i = 0; i < 4; i++) {
          float x = (acc[0][i] + acc[1][i]) * factor;
          if (capped) {
            asm volatile("");                             // (a branch: not computed where there is no cap)
            x = top_of_cap * fmaf(-2.f, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x) + 1.f), 1.f);
          }
          y[4 * k + i] = fmaf(-slope, behind - (float)i, x);
          seen |= sees && 4 * c + i < now[k].n ? 1u << (4 * k + i) : 0u;
        }
      }
      // shares relative to the running maximum, which moves when they grow past 8192
      float e[4 * HW], sum;
      auto exponentials = [&]() {
        const float ms = m == -INFINITY ? 0.f : m;
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < 4 * HW; i++) {
          e[i] = seen >> i & 1 ? __builtin_amdgcn_exp2f(y[i] - ms) : 0.f;
          sum += e[i];
        }
      };
      exponentials();
      if (__builtin_amdgcn_ballot_w64(sum > 8192.f || (m == -INFINITY && seen != 0))) {
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4 * HW; i++) top = fmaxf(top, seen >> i & 1 ? y[i] : -INFINITY);
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float mn = fmaxf(m, top), f = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
        l *= f;
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int i = 0; i < 4; i++) o[n][i] *= f;
        m = mn;
        exponentials();
      }
      l += sum;
      // results, the shares in two terms: what they are rounded to and what that leaves out
      if constexpr (HW == 1) {
        frag4 most, rest;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          most[i] = from_float<T>(e[i]);
          rest[i] = from_float<T>(e[i] - to_float(most[i]));
        }
#pragma unroll
        for (int n0 = 0; n0 < NT; n0 += 4) {
          frag4 v[4];
#pragma unroll
          for (int n = 0; n < 4; n++) v[n] = __builtin_bit_cast(frag4, latent_read_tr(stage + (tr_at ^ (((n0 + n) & 7) << 5)) + ((n0 + n) >> 3) * 256));
#pragma unroll
          for (int n = 0; n < 4; n++) o[n0 + n] = M::run(v[n], most, o[n0 + n]);
#pragma unroll
          for (int n = 0; n < 4; n++) o[n0 + n] = M::run(v[n], rest, o[n0 + n]);
        }
      } else {
#pragma unroll
        for (int k = 0; k < HW; k += 2) {
          frag8 most, rest;
#pragma unroll
          for (int i = 0; i < 8; i++) {
            most[i] = from_float<T>(e[4 * k + i]);
            rest[i] = from_float<T>(e[4 * k + i] - to_float(most[i]));
          }
#pragma unroll
          for (int n0 = 0; n0 < NT; n0 += 4) {
            frag8 v[4];
#pragma unroll
            for (int n = 0; n < 4; n++) {
              const uint32_t from = stage + k * G::GROUP + (tr_at ^ (((n0 + n) & 7) << 5)) + ((n0 + n) >> 3) * 256;
              typedef short s16x8 __attribute__((ext_vector_type(8)));
              v[n] = __builtin_bit_cast(frag8, (s16x8)__builtin_shufflevector(latent_read_tr(from), latent_read_tr(from + G::GROUP), 0, 1, 2, 3, 4, 5, 6, 7));
            }
#pragma unroll
            for (int n = 0; n < 4; n++) o[n0 + n] = M::run(v[n], most, o[n0 + n]);
#pragma unroll
            for (int n = 0; n < 4; n++) o[n0 + n] = M::run(v[n], rest, o[n0 + n]);
          }
        }
      }
#pragma unroll
      for (int k = 0; k < HW; k++) now[k] = next[k];
    }

    // the wavefronts' results: per head the maximum, the sum, LAT sums
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    __syncthreads();
    float *join = reinterpret_cast<float *>(smem), *stats = reinterpret_cast<float *>(smem + G::RING);
    {
      const int r = 16 * wave + key;
      if (c == 0) stats[2 * r] = m, stats[2 * r + 1] = l;
#pragma unroll
      for (int n = 0; n < NT; n++) *reinterpret_cast<f32x4 *>(join + r * G::JOIN + 16 * n + 4 * c) = o[n];
    }
    __syncthreads();
    const bool whole = s0 == 0 && s1 == steps;
    const int slot = 2 * blockIdx.x + (at > lo ? 1 : 0);
    if (tid == 0 && s0 == 0) {
      int parts = 1;
      if (!whole) {                                       // the piece that the item's last step is in
        const int64_t last = ((begin + steps) * pieces - 1) / total;
        parts = (int)(last - blockIdx.x) + 1;
      }
      int32_t *to = a.meta + 3 * (int64_t)item;
      to[0] = blockIdx.x; to[1] = parts; to[2] = slot;
    }
    for (int i = tid; i < heads * (LAT / 8); i += 256) {
      const int h = i / (LAT / 8), d = i % (LAT / 8) * 8;
      constexpr int PW = 4 / HW;
      float top = -INFINITY, sum = 0.f, x[8] = {};
#pragma unroll
      for (int p = 0; p < PW; p++) top = fmaxf(top, stats[2 * (16 * (p * HW + h / 16) + h % 16)]);
#pragma unroll
      for (int p = 0; p < PW; p++) {
        const int r = 16 * (p * HW + h / 16) + h % 16;
        const float f = stats[2 * r] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(stats[2 * r] - top);
        sum = fmaf(f, stats[2 * r + 1], sum);
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = fmaf(f, join[r * G::JOIN + d + e], x[e]);
      }
      if (whole) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        union { u32x4 raw; T e[8]; } out;
#pragma unroll
        for (int e = 0; e < 8; e++) out.e[e] = from_float<T>(sum == 0.f ? 0.f : x[e] * inv);
        *reinterpret_cast<u32x4 *>(reinterpret_cast<T *>(a.o) + b * a.o_sb + (first + h) * a.o_sh + d) = out.raw;
      } else {
        float *to = a.partial + ((int64_t)slot * a.per + h) * (LAT + 2);
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        if (d == 0) *reinterpret_cast<f32x2 *>(to) = f32x2{top, sum};
#pragma unroll
        for (int e = 0; e < 8; e += 2) *reinterpret_cast<f32x2 *>(to + 2 + d + e) = f32x2{x[e], x[e + 1]};
      }
    }
    __syncthreads();
    at = begin + s1;
    begin += steps;
  }
}

// The parts of a sequence's head joined: a workgroup a head, a part's maximum and sum a lane at a time, then the parts among its four wavefronts.  Parts that saw nothing have
// a factor of 0.
template <typename T, int LAT> __global__ void __launch_bounds__(256) k_latent_join(LatentArgs a) {
  constexpr int N = LAT / 64;
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  __shared__ float sums[4][LAT + 2], tops[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Quotient at(blockIdx.x, a.H);
  const int b = (int)at.q, h = (int)at.r, unit = h / a.per, r = h % a.per;
  const int32_t *meta = a.meta + 3 * ((int64_t)b * a.units + unit);
  const int parts = meta[1];
  if (parts <= 1) return;
  const int from = meta[0], slot = meta[2];
  auto part = [&](int p) { return a.partial + ((int64_t)(p == 0 ? slot : 2 * (from + p)) * a.per + r) * (LAT + 2); };
  float top = -INFINITY;
  for (int p = tid; p < parts; p += 256) top = fmaxf(top, part(p)[0]);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
  if (lane == 0) tops[wave] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 4; w++) top = fmaxf(top, tops[w]);
  float sum = 0.f, x[N] = {};
  for (int p0 = wave; p0 < parts; p0 += 16) {             // four of the wavefront's parts on their way
    f32x2 own[4];
    float v[4][N];
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const float *p = part(p0 + 4 * u < parts ? p0 + 4 * u : p0);
      own[u] = *reinterpret_cast<const f32x2 *>(p);
#pragma unroll
      for (int e = 0; e < N; e += 2) {
        const f32x2 w = *reinterpret_cast<const f32x2 *>(p + 2 + 64 * e + 2 * lane);
        v[u][e] = w[0];
        v[u][e + 1] = w[1];
      }
    }
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const float f = p0 + 4 * u >= parts || own[u][0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(own[u][0] - top);
      sum = fmaf(f, own[u][1], sum);
#pragma unroll
      for (int e = 0; e < N; e++) x[e] = fmaf(f, v[u][e], x[e]);
    }
  }
  if (lane == 0) sums[wave][LAT] = sum;
#pragma unroll
  for (int e = 0; e < N; e += 2) *reinterpret_cast<f32x2 *>(&sums[wave][0] + 64 * e + 2 * lane) = f32x2{x[e], x[e + 1]};
  __syncthreads();
  sum = 0.f;
#pragma unroll
  for (int w = 0; w < 4; w++) sum += sums[w][LAT];
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  for (int d = tid; d < LAT; d += 256) {
    const float y = (sums[0][d] + sums[1][d]) + (sums[2][d] + sums[3][d]);
    reinterpret_cast<T *>(a.o)[b * a.o_sb + h * a.o_sh + d] = from_float<T>(sum == 0.f ? 0.f : y * inv);
  }
}

template <typename T, int LAT, int HW> int launch_latent(const LatentArgs &a, hipStream_t st) {
  static std::atomic<uint64_t> done{0};
  if (LatentGeo<LAT>::LDS > 65536 && !raise_lds_limit(reinterpret_cast<const void *>(k_latent_attention<T, LAT, HW>), LatentGeo<LAT>::LDS, done)) return BSP_ERR_HIP;
  hipLaunchKernelGGL((k_latent_attention<T, LAT, HW>), dim3((unsigned)a.pieces), dim3(256), LatentGeo<LAT>::LDS, st, a);
  return BSP_OK;
}
template <typename T, int LAT> int launch_latent(const LatentArgs &a, bool joined, hipStream_t st) {
  const int rc = a.per <= 16 ? launch_latent<T, LAT, 1>(a, st) : a.per <= 32 ? launch_latent<T, LAT, 2>(a, st) : launch_latent<T, LAT, 4>(a, st);
  if (rc != BSP_OK) return rc;
  if (joined) hipLaunchKernelGGL((k_latent_join<T, LAT>), dim3((unsigned)((int64_t)a.B * a.H)), dim3(256), 0, st, a);
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
  const int64_t meta = ((int64_t)B * latent_units(H) * 12 + 15) / 16 * 16;
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
  a.units = latent_units(H); a.per = bsp_latent_attention_heads(H); a.pieces = latent_pieces(B, H, block, most_blocks);
  a.meta = reinterpret_cast<int32_t *>(workspace);
  a.partial = reinterpret_cast<float *>(reinterpret_cast<unsigned char *>(workspace) + ((int64_t)B * a.units * 12 + 15) / 16 * 16);
  const bool joined = most_blocks * block > 64;           // (else no sequence has more than one step)
  return dtype == BSP_F16 ? launch_latent<f16>(a, latent, joined, as_stream(stream)) : launch_latent<bf16>(a, latent, joined, as_stream(stream));
}
