// Rotated positions: of each row of D elements the pairs (a, b) of the first 2 n are turned by position * frequency,
//     (a, b) -> (a cos - b sin, a sin + b cos),
// the others are copied; the gradient is the same with the angle's sign changed.  Pair p is elements p and n + p, or 2 p and 2 p + 1 (neighbours).
//
// It moves each element in and out once and is bound by that.  A thread has the 16-byte chunks of 16 / size pairs (a copied chunk) of one position and goes through several
// heads with them, four at a time on their way, so that the sines and cosines (rotation.h: from the position, no table), sixty operations a pair, are shared.  Measured: bf16 4 x (32 and 8)
// heads x 4096 x 128, 336 MB: 59 us back to back (5.6 TB/s, of which a cache level has some; 65 us, 5.2 TB/s, on fresh tensors), fp32 2 x 24 x 2023 x 64 9 us; vector units 40 % of the cycles.
#include "rotation.h"

namespace bsp {

struct RotateOperand {
  const void *x; void *y;
  int64_t x_sz, x_sh, x_sl, y_sz, y_sh, y_sl;
};
struct RotateArgs {
  RotateOperand of[2];
  int heads[2];                    // of[1]: none, or as many
  const uint64_t *fractions;
  const int32_t *positions; int64_t p_sz, p_sl;          // NULL: position l
  uint32_t tokens, L, items;       // Z * L; chunks of a thread's kind a row
  uint32_t turning;                // the first of them are pairs
  int pairs, groups, per;          // threads that share a position's heads, heads of each
  float sign;
};

namespace {

template <typename T> union Chunk { u32x4 raw; T e[16 / sizeof(T)]; };

template <typename T, bool NEIGHBOURS> __global__ void __launch_bounds__(256) k_rotate(RotateArgs a) {
  constexpr int N = 16 / sizeof(T), U = 4;
  const uint32_t id = blockIdx.x * 256u + threadIdx.x;
  const Quotient row(id, a.items), at(row.q, a.tokens), place(at.r, a.L);
  const uint32_t item = row.r, z = place.q, l = place.r;
  if (at.q >= (uint32_t)a.groups) return;
  const bool turning = item < a.turning;
  // where the thread's two chunks are (a copied row's: the second is none)
  const int first = !turning ? 2 * a.pairs + (int)(item - a.turning) * N : NEIGHBOURS ? (int)item * 2 * N : (int)item * N;
  const int second = NEIGHBOURS ? first + N : first + a.pairs;
  float cos[N], sin[N];
  if (turning) {
    const int32_t position = a.positions ? a.positions[z * a.p_sz + l * a.p_sl] : (int32_t)l;
#pragma unroll
    for (int i = 0; i < N; i++) {
      const Turn t = turn_of(position, a.fractions[item * N + i]);
      cos[i] = t.cos;
      sin[i] = a.sign * t.sin;
    }
  }
  const int all = a.heads[0] + a.heads[1], begin = (int)at.q * a.per, end = begin + a.per < all ? begin + a.per : all;
  for (int h0 = begin; h0 < end; h0 += U) {
    Chunk<T> x[U], y[U];
    const T *from[U];
    T *to[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int h = h0 + u < end ? h0 + u : end - 1;
      const bool other = h >= a.heads[0];
      const RotateOperand &o = a.of[other];
      const int64_t hh = other ? h - a.heads[0] : h;
      from[u] = reinterpret_cast<const T *>(o.x) + z * o.x_sz + hh * o.x_sh + l * o.x_sl;
      to[u] = reinterpret_cast<T *>(o.y) + z * o.y_sz + hh * o.y_sh + l * o.y_sl;
      if (h0 + u < end) {
        x[u].raw = *reinterpret_cast<const u32x4 *>(from[u] + first);
        if (turning) y[u].raw = *reinterpret_cast<const u32x4 *>(from[u] + second);
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (h0 + u >= end) break;
      if (turning) {
        T p[2 * N];
#pragma unroll
        for (int i = 0; i < N; i++) p[i] = x[u].e[i], p[N + i] = y[u].e[i];
#pragma unroll
        for (int i = 0; i < N; i++) {
          const int ia = NEIGHBOURS ? 2 * i : i, ib = NEIGHBOURS ? 2 * i + 1 : N + i;
          turn_pair(to_float(p[ia]), to_float(p[ib]), cos[i], sin[i], p[ia], p[ib]);
        }
#pragma unroll
        for (int i = 0; i < N; i++) x[u].e[i] = p[i], y[u].e[i] = p[N + i];
        *reinterpret_cast<u32x4 *>(to[u] + second) = y[u].raw;
      }
      *reinterpret_cast<u32x4 *>(to[u] + first) = x[u].raw;
    }
  }
}

template <typename T> void launch_rotate(const RotateArgs &a, bool neighbours, unsigned grid, hipStream_t st) {
  if (neighbours) hipLaunchKernelGGL((k_rotate<T, true>), dim3(grid), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((k_rotate<T, false>), dim3(grid), dim3(256), 0, st, a);
}

}  // namespace
}  // namespace bsp

using namespace bsp;

extern "C" int bsp_rotate(int dtype, int Z, int64_t length, int D, int pairs, int neighbours, int back, const uint64_t *fractions, const int32_t *positions,
                          int64_t pos_stride_z, int64_t pos_stride_l, const void *x0, void *y0, int H0, const int64_t *strides0, const void *x1, void *y1, int H1,
                          const int64_t *strides1, void *stream) {
  if (dtype != BSP_F16 && dtype != BSP_BF16 && dtype != BSP_F32) return BSP_ERR_UNSUPPORTED;
  if (Z <= 0 || length <= 0 || length >= ((int64_t)1 << 31) || D <= 0 || D % 8 || !rotation_ok(fractions, pairs, D) || H0 <= 0 || H1 < 0) return BSP_ERR_ARG;
  const int n = dtype == BSP_F32 ? 4 : 8;
  const void *ptrs[] = {x0, y0, x1, y1};
  for (int i = 0; i < (H1 ? 4 : 2); i++)
    if (!ptrs[i] || (reinterpret_cast<uintptr_t>(ptrs[i]) & 15)) return BSP_ERR_ARG;
  if (!strides0 || (H1 && !strides1)) return BSP_ERR_ARG;
  RotateArgs a{};
  for (int o = 0; o < (H1 ? 2 : 1); o++) {
    const int64_t *s = o ? strides1 : strides0;
    for (int i = 0; i < 6; i++)
      if (s[i] % n) return BSP_ERR_ARG;
    a.of[o] = RotateOperand{o ? x1 : x0, o ? y1 : y0, s[0], s[1], s[2], s[3], s[4], s[5]};
  }
  a.heads[0] = H0; a.heads[1] = H1;
  a.fractions = fractions; a.positions = positions; a.p_sz = pos_stride_z; a.p_sl = pos_stride_l;
  a.pairs = pairs; a.turning = (uint32_t)(pairs / n); a.items = (uint32_t)((D - pairs) / n);
  a.sign = back ? -1.f : 1.f;
  const int64_t tokens = (int64_t)Z * length, heads = (int64_t)H0 + H1;
  // (a grid has fewer than 2^32 threads)
  if (tokens >= ((int64_t)1 << 32) || heads >= ((int64_t)1 << 30) || tokens * a.items >= ((int64_t)1 << 32)) return BSP_ERR_UNSUPPORTED;
  a.tokens = (uint32_t)tokens; a.L = (uint32_t)length;
  // heads of a thread: one in small launches, up to four where there are threads enough without (bf16, 32 and 8 heads of 128, one a thread and four: 64 positions 3.1 and 3.9 us, 512 4.8 and 4.6,
  // 2048 10.9 and 9.0, 4 x 4096 78 and 59; eight: 5.4, 6.0, 10.1 and 59)
  const double threads = (double)tokens * a.items * (double)heads / 65536.;
  int per = threads < 1. ? 1 : threads > 4. ? 4 : (int)threads;
  while ((double)(tokens * a.items) * (double)((heads + per - 1) / per) >= 4294967040. && per < heads) per *= 2;
  a.per = per; a.groups = (int)((heads + per - 1) / per);
  const int64_t total = tokens * a.items * a.groups;
  if (total >= ((int64_t)1 << 32) - 256) return BSP_ERR_UNSUPPORTED;
  const unsigned grid = (unsigned)((total + 255) / 256);
  const hipStream_t st = as_stream(stream);
  if (dtype == BSP_F16) launch_rotate<f16>(a, neighbours != 0, grid, st);
  else if (dtype == BSP_BF16) launch_rotate<bf16>(a, neighbours != 0, grid, st);
  else launch_rotate<float>(a, neighbours != 0, grid, st);
  BSP_LAUNCH_CHECK();
  return BSP_OK;
}
