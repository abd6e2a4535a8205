// Keys and values into the pages of a quantised cache, and back (layout: cache.h).
//
// Of 32 neighbouring elements x (taken into [-65504, 65504], the range of fp16) least = fp16(min x), step = fp16((max x - least) /
// (2^bits - 1)), code = the integer nearest to (x - least) / step, ties to the even one, within 0 .. 2^bits - 1; step's quotient is rounded to fp32 first, and below zero where least is rounded up past the max.  A group with a NaN
// reads back as NaN.  The codes are those of exact arithmetic: a quotient is computed in fp32 and, where that lies close to the middle of two
// integers, decided in 64 bits.
//
// Both kernels move each byte once; the read is bound by that, the write by its vector operations.  A thread has a chunk of eight elements: 16 bytes in 16-bit types, and the four
// threads of a group agree on its range by two exchanges within the quad.  Tensors outside the cache are streamed past the L2 (non-temporal): nothing reads them
// soon.  Measured: 16384 positions of 16 heads of 64, fp16, 8 bits (67 MB and 38 MB): written in 33 us (4 of them the launch that says whose a slot is), read back in 27, or
// in 16 where a cache level still holds them.  One after the other 45 us: 51 without the streaming, 58 before a thread's place was found without divisions and the rounded
// quotient taken from the low bits of one sum.  The write's vector units are busy for 68 % of its cycles, 85 to 100 % over more positions.
// 32749 positions of 8 heads of 128, bf16, 4 bits (176 MB) read in 41 us, 52 without the streaming.
#include "cache.h"

namespace bsp {

struct CacheArgs {
  const void *k, *v;               // write: [T, heads, D], strides in elements
  void *ko, *vo;                   // read: [T, heads, D], contiguous
  int64_t k_st, k_sh, v_st, v_sh;
  const int32_t *slots;
  int32_t *owner;
  unsigned char *pages;
  int64_t capacity;                // positions of the cache
  int T, heads, block, block_shift;
};

namespace {

// value of the neighbour xor 1, xor 2 in the quad
__device__ __forceinline__ float quad1(float v) { return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0xB1, 0xf, 0xf, true)); }
__device__ __forceinline__ float quad2(float v) { return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x4E, 0xf, 0xf, true)); }

template <typename T> __device__ __forceinline__ void load8(float (&x)[8], const T *p) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const f32x4 v = __builtin_nontemporal_load(reinterpret_cast<const f32x4 *>(p + 4 * i));
#pragma unroll
      for (int j = 0; j < 4; j++) x[4 * i + j] = v[j];
    }
  } else {
    union { u32x4 raw; T e[8]; } u;
    u.raw = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p));
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = to_float(u.e[i]);
  }
}

// Which of the positions of a slot that is given twice is written: the last.  owner[slot] (zero between calls) becomes the
// greatest number t + 1 among them.
__global__ void __launch_bounds__(256) k_cache_owner(CacheArgs a) {
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t >= a.T) return;
  const int slot = a.slots[t];
  if (slot >= 0 && slot < a.capacity) atomicMax(a.owner + slot, t + 1);
}

// A workgroup per position.  SCAN: few positions, a later one with the same slot is looked for here; else owner says which is last.
template <typename T, int BITS, int D, bool SCAN> __global__ void __launch_bounds__(256) k_cache_write(CacheArgs a) {
  typedef Page<BITS, D> P;
  constexpr int CHUNKS = D / 8;
  const int t = (int)xcd_remap(blockIdx.x, a.T), tid = threadIdx.x;
  const int slot = as_table(a.slots)[t];
  if (slot < 0 || slot >= a.capacity) return;
  if constexpr (SCAN) {
    bool later = false;
    for (int i = t + 1 + tid; i < a.T; i += 256) later |= a.slots[i] == slot;
    if (__syncthreads_or(later)) return;
  } else {
    __shared__ int last;
    if (tid == 0) last = a.owner[slot];
    __syncthreads();
    if (last != t + 1) return;
    if (tid == 0) a.owner[slot] = 0;                    // (another position of the slot that looks from now on finds 0: not the last either)
  }
  const int page = slot >> a.block_shift, at = slot & (a.block - 1);
  const int j = tid % CHUNKS, g = j >> 2, c = j & 3;
  for (int m = tid / CHUNKS; m < 2 * a.heads; m += 256 / CHUNKS) {
    const int value = m >= a.heads, head = value ? m - a.heads : m;
    float x[8];
    load8<T>(x, (value ? reinterpret_cast<const T *>(a.v) + t * a.v_st + head * a.v_sh : reinterpret_cast<const T *>(a.k) + t * a.k_st + head * a.k_sh) + 8 * j);
    // the group's range, into that of fp16 here: elements outside get the codes of its ends below
    bool nan = false;
    float lo = x[0], hi = x[0];
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      nan |= __builtin_isunordered(x[e], x[e + 1]);
      lo = fminf(fminf(lo, x[e]), x[e + 1]);
      hi = fmaxf(fmaxf(hi, x[e]), x[e + 1]);
    }
    float bad = nan ? 1.f : 0.f;
    lo = fminf(lo, quad1(lo));
    hi = fmaxf(hi, quad1(hi));
    bad = fmaxf(bad, quad1(bad));
    lo = fminf(lo, quad2(lo));
    hi = fmaxf(hi, quad2(hi));
    bad = fmaxf(bad, quad2(bad));
    lo = fminf(fmaxf(lo, -65504.f), 65504.f);
    hi = fminf(fmaxf(hi, -65504.f), 65504.f);
    constexpr int MOST = (1 << BITS) - 1;
    f16 least = (f16)lo, step;
    {
      const double range = (double)hi - (double)(float)least;
      const float r = (float)range;
      step = (f16)((double)r == range ? r / (float)MOST : (float)(range / (double)MOST));   // (the same number: both quotients are rounded to the nearest)
    }
    if (bad != 0.f) least = __builtin_bit_cast(f16, (uint16_t)0x7e00), step = (f16)0.f;
    const float l32 = (float)least, s32 = (float)step;
    uint32_t w[2] = {0u, 0u};
    if (s32 != 0.f) {                                   // (below zero where the least value was rounded up past the greatest one)
      // the quotient rounded in the low bits of 1.5 * 2^23 + it
      const float inv = __builtin_amdgcn_rcpf(s32), magic = 12582912.f;
      uint32_t code[8];
      float off = 0.f;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float d = x[e] - l32, r = fmaf(d, inv, magic);
        off = fmaxf(off, fabsf(fmaf(d, inv, magic - r)));
        code[e] = __builtin_bit_cast(uint32_t, fminf(fmaxf(r, magic), magic + (float)MOST));
      }
      // x - least is off by 2^-24 of itself, the reciprocal by 2^-23, so the quotient by 3 * 2^-24 * MOST: decided in 64 bits where the middle is as near
      if (off > 0.5f - MOST * 0x1p-22f) {
        const double h = 0.5 * fabs((double)s32);
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const int n0 = (int)(code[e] & 0x1ffu);
          const double rest = ((double)x[e] - (double)l32) - (double)n0 * (double)s32, rem = s32 < 0.f ? -rest : rest;
          const bool odd = n0 & 1;
          const int m = n0 + (rem > h || (rem == h && odd) ? 1 : 0) - (rem < -h || (rem == -h && odd) ? 1 : 0);
          code[e] = (uint32_t)(m < 0 ? 0 : m > MOST ? MOST : m);
        }
      }
      if constexpr (BITS == 4) {
#pragma unroll
        for (int e = 0; e < 8; e++) w[0] |= (code[e] & 15u) << (4 * (e >> 1) + 16 * (e & 1));
      } else {
#pragma unroll
        for (int e = 0; e < 2; e++)
          w[e] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(code[4 * e + 3], code[4 * e + 2], 0x0c0c0400u), __builtin_amdgcn_perm(code[4 * e + 1], code[4 * e], 0x0c0c0400u), 0x05040100u);
      }
    }
    unsigned char *base = a.pages + ((int64_t)page * a.heads + head) * P::bytes(a.block);
    unsigned char *to = base + P::codes(a.block, value) + at * P::ROW + P::chunk(c, g);
    if constexpr (BITS == 4) *reinterpret_cast<uint32_t *>(to) = w[0];
    else *reinterpret_cast<u32x2 *>(to) = u32x2{w[0], w[1]};
    if (c == 0)
      *reinterpret_cast<uint32_t *>(base + P::meta(a.block, value) + at * P::META + 4 * g) =
          (uint32_t)__builtin_bit_cast(uint16_t, step) | (uint32_t)__builtin_bit_cast(uint16_t, least) << 16;
  }
}

// A workgroup per position, a chunk a thread.  Slots outside the cache read as zeros.
template <typename T, int BITS, int D> __global__ void __launch_bounds__(256) k_cache_read(CacheArgs a) {
  typedef Page<BITS, D> P;
  constexpr int CHUNKS = D / 8;
  const int t = (int)xcd_remap(blockIdx.x, a.T), tid = threadIdx.x;
  const int slot = as_table(a.slots)[t];
  const bool here = slot >= 0 && slot < a.capacity;
  const int page = here ? slot >> a.block_shift : 0, at = here ? slot & (a.block - 1) : 0;
  const int j = tid % CHUNKS, g = j >> 2, c = j & 3;
  for (int m = tid / CHUNKS; m < 2 * a.heads; m += 256 / CHUNKS) {
    const int value = m >= a.heads, head = value ? m - a.heads : m;
    float x[8] = {};
    if (here) {
      const unsigned char *base = a.pages + ((int64_t)page * a.heads + head) * P::bytes(a.block);
      const uint32_t *from = reinterpret_cast<const uint32_t *>(base + P::codes(a.block, value) + at * P::ROW + P::chunk(c, g));
      const uint32_t meta = *reinterpret_cast<const uint32_t *>(base + P::meta(a.block, value) + at * P::META + 4 * g);
      const float step = (float)__builtin_bit_cast(f16, (uint16_t)meta), least = (float)__builtin_bit_cast(f16, (uint16_t)(meta >> 16));
      uint32_t w[2] = {from[0], BITS == 8 ? from[BITS == 8 ? 1 : 0] : 0u};
      f16x2 p[4];
      chunk_codes<BITS>(w, p);
#pragma unroll
      for (int e = 0; e < 8; e++) x[e] = fmaf((float)p[e >> 1][e & 1], step, least);
      if constexpr (__is_same(T, f16)) {                // (where the rounding of the step takes an element past fp16's range: NaN stays NaN)
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = x[e] > 65504.f ? 65504.f : x[e];
      }
    }
    T *to = reinterpret_cast<T *>(value ? a.vo : a.ko) + ((int64_t)t * a.heads + head) * D + 8 * j;
    if constexpr (sizeof(T) == 4) {
      __builtin_nontemporal_store(f32x4{x[0], x[1], x[2], x[3]}, reinterpret_cast<f32x4 *>(to));
      __builtin_nontemporal_store(f32x4{x[4], x[5], x[6], x[7]}, reinterpret_cast<f32x4 *>(to + 4));
    } else {
      union { u32x4 raw; T e[8]; } u;
#pragma unroll
      for (int e = 0; e < 8; e++) u.e[e] = from_float<T>(x[e]);
      __builtin_nontemporal_store(u.raw, reinterpret_cast<u32x4 *>(to));
    }
  }
}

// few positions: each workgroup reads the slots behind its own, which costs less than the launch that says whose a slot is
constexpr int kScan = 512;

template <typename T, int BITS, int D> int launch_cache(const CacheArgs &a, bool write, hipStream_t st) {
  if (!write) {
    hipLaunchKernelGGL((k_cache_read<T, BITS, D>), dim3((unsigned)a.T), dim3(256), 0, st, a);
  } else if (a.T <= kScan) {
    hipLaunchKernelGGL((k_cache_write<T, BITS, D, true>), dim3((unsigned)a.T), dim3(256), 0, st, a);
  } else {
    hipLaunchKernelGGL(k_cache_owner, dim3((unsigned)cdiv(a.T, 256)), dim3(256), 0, st, a);
    hipLaunchKernelGGL((k_cache_write<T, BITS, D, false>), dim3((unsigned)a.T), dim3(256), 0, st, a);
  }
  BSP_LAUNCH_CHECK();
  return BSP_OK;
}
template <typename T> int launch_cache(const CacheArgs &a, int bits, int D, bool write, hipStream_t st) {
  if (bits == 4) return D == 64 ? launch_cache<T, 4, 64>(a, write, st) : launch_cache<T, 4, 128>(a, write, st);
  return D == 64 ? launch_cache<T, 8, 64>(a, write, st) : launch_cache<T, 8, 128>(a, write, st);
}
int launch_cache(int dtype, const CacheArgs &a, int bits, int D, bool write, hipStream_t st) {
  return dtype == BSP_F16 ? launch_cache<f16>(a, bits, D, write, st) : dtype == BSP_BF16 ? launch_cache<bf16>(a, bits, D, write, st) : launch_cache<float>(a, bits, D, write, st);
}

int cache_args(int dtype, const void *pages, int n_pages, int block, int heads, int D, int bits, const int32_t *slots, int T, CacheArgs &a) {
  if (!pages || (reinterpret_cast<uintptr_t>(pages) & 15) || n_pages <= 0 || heads <= 0 || !slots || T <= 0) return BSP_ERR_ARG;
  if (bsp_cache_page_bytes(block, heads, D, bits) <= 0 || (dtype != BSP_F16 && dtype != BSP_BF16 && dtype != BSP_F32)) return BSP_ERR_UNSUPPORTED;
  if ((int64_t)n_pages * block >= ((int64_t)1 << 31) || (int64_t)T * 256 >= ((int64_t)1 << 32)) return BSP_ERR_UNSUPPORTED;   // (a grid has fewer than 2^32 threads)
  a = CacheArgs{};
  a.pages = reinterpret_cast<unsigned char *>(const_cast<void *>(pages));
  a.capacity = (int64_t)n_pages * block;
  a.block = block; a.block_shift = __builtin_ctz(block); a.heads = heads; a.slots = slots; a.T = T;
  return BSP_OK;
}

}  // namespace
}  // namespace bsp

using namespace bsp;

extern "C" int64_t bsp_cache_page_bytes(int block, int heads, int D, int bits) {
  if ((block != 16 && block != 32 && block != 64 && block != 128) || heads <= 0 || (D != 64 && D != 128) || (bits != 4 && bits != 8)) return BSP_ERR_UNSUPPORTED;
  return 2 * (int64_t)block * heads * (D * bits / 8 + D / 8);
}

extern "C" int bsp_cache_write(int dtype, void *pages, int n_pages, int block, int heads, int D, int bits, const void *k, int64_t k_stride_t, int64_t k_stride_h,
                               const void *v, int64_t v_stride_t, int64_t v_stride_h, const int32_t *slots, int T, int32_t *owner, void *stream) {
  CacheArgs a;
  const int rc = cache_args(dtype, pages, n_pages, block, heads, D, bits, slots, T, a);
  if (rc != BSP_OK) return rc;
  const int unit = dtype == BSP_F32 ? 4 : 8;
  if (!k || !v || !owner || ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15)) return BSP_ERR_ARG;
  if (k_stride_t % unit || k_stride_h % unit || v_stride_t % unit || v_stride_h % unit) return BSP_ERR_ARG;
  a.k = k; a.v = v; a.k_st = k_stride_t; a.k_sh = k_stride_h; a.v_st = v_stride_t; a.v_sh = v_stride_h;
  a.owner = owner;
  return launch_cache(dtype, a, bits, D, true, as_stream(stream));
}

extern "C" int bsp_cache_read(int dtype, const void *pages, int n_pages, int block, int heads, int D, int bits, void *k, void *v, const int32_t *slots, int T, void *stream) {
  CacheArgs a;
  const int rc = cache_args(dtype, pages, n_pages, block, heads, D, bits, slots, T, a);
  if (rc != BSP_OK) return rc;
  if (!k || !v || ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15)) return BSP_ERR_ARG;
  a.ko = k; a.vo = v;
  return launch_cache(dtype, a, bits, D, false, as_stream(stream));
}
