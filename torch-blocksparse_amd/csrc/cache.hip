// Keys and values into the pages of a quantised cache, and back (layout: cache.h).
//
// Of 32 neighbouring elements x (taken into [-65504, 65504], the range of fp16) least = fp16(min x), step = fp16((max x - least) /
// (2^bits - 1)), code = the integer nearest to (x - least) / step, ties to the even one, within 0 .. 2^bits - 1; step's quotient is rounded to fp32 first, and below zero where least is rounded up past the max.  A group with a NaN
// reads back as NaN.  The codes are those of exact arithmetic: a quotient is computed in fp32 and, where that lies close to the middle of two
// integers, decided in 64 bits.
//
// Both kernels move each byte once; the read is bound by that, the write by its vector operations.  A thread has a chunk of eight elements: 16 bytes in 16-bit types, and the four
// threads of a group agree on its range by two exchanges within the quad.  Tensors outside the cache are streamed past the L2 (non-temporal): nothing reads them
// soon.  Measured: 16384 positions of 16 heads of 64, fp16, 8 bits (67 MB and 38 MB): written in 30 us (2 to 4 of them the launch that says whose a slot is), read back in 27, or
// in 16 where a cache level still holds them.  One after the other 46 us: 48 with a division in two forms and keys and values in one wavefront, 54 without the streaming, 61 before a
// thread's place was found without divisions and the rounded quotient taken from the low bits of one sum.
// 32749 positions of 8 heads of 128, bf16, 4 bits (176 MB) read in 41 us, 52 without the streaming.
//
// With a rotation (rotation.h) the keys are turned first, all of it in 64 bits, as what rounding in between would leave out decides codes: the vector units do fp64 at the
// rate of fp32.  A workgroup computes its position's sines and cosines once, into LDS, and a thread takes the other chunk of its pairs from the lane that has it.  Measured: 16384
// positions of 8 heads of 128, fp16, 8 bits (67 MB read, 38 MB written): 37 us and the slots' owners 4, where the plain write takes 28.  Its vector units have 250 instructions a
// wavefront, 66 % of its cycles; with 302 it took 42.5.  Taking all eight elements of the other lane before the first is used, and LDS without conflicts, did not change it.
#include "cache.h"
#include "rotation.h"
#include "slots.h"

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
  const int32_t *positions;        // write, with a rotation
  const uint64_t *fractions;
  int pairs, neighbours;
};

namespace {

// value of the neighbour xor 1, xor 2 in the quad
__device__ __forceinline__ float quad1(float v) { return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0xB1, 0xf, 0xf, true)); }
__device__ __forceinline__ float quad2(float v) { return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x4E, 0xf, 0xf, true)); }

// (greater() below hides from the compiler that it wrote v just before: a lane's value is read by another two cycles later at the earliest)
__device__ __forceinline__ double quad1(double v) {
  asm volatile("s_nop 1" : "+v"(v));
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t l = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, 0xB1, 0xf, 0xf, true), h = __builtin_amdgcn_update_dpp(0, (int)(b >> 32), 0xB1, 0xf, 0xf, true);
  return __builtin_bit_cast(double, (uint64_t)h << 32 | l);
}
__device__ __forceinline__ double quad2(double v) {
  asm volatile("s_nop 1" : "+v"(v));
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t l = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, 0x4E, 0xf, 0xf, true), h = __builtin_amdgcn_update_dpp(0, (int)(b >> 32), 0x4E, 0xf, 0xf, true);
  return __builtin_bit_cast(double, (uint64_t)h << 32 | l);
}
// the lesser and the greater of two, NaN if one is; the double's leaves NaN out (no operation has it otherwise), and is one instruction where fmax is three, which quiet its operands
__device__ __forceinline__ float lesser(float a, float b) { return __builtin_elementwise_minimum(a, b); }
__device__ __forceinline__ float greater(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ double greater(double a, double b) {
  double r;
  asm("v_max_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}

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

// The codes of the thread's eight elements (words), least value and step of their group, which the four threads of a quad have.  X: float, or double for what a rotation
// left (whose least element is rounded to fp32 on its way to fp16)
template <int BITS, typename X> __device__ __forceinline__ void quantise(const X (&x)[8], uint32_t (&w)[2], f16 &least, f16 &step) {
  constexpr int MOST = (1 << BITS) - 1;
  // the group's range, into that of fp16 here: elements outside get the codes of its ends below
  float y[8];
#pragma unroll
  for (int e = 0; e < 8; e++) y[e] = (float)x[e];
  float lo = lesser(y[0], y[1]);                        // (rounding keeps the order)
  X hi = greater(x[0], x[1]);
#pragma unroll
  for (int e = 2; e < 8; e += 2) {
    lo = lesser(lesser(lo, y[e]), y[e + 1]);
    hi = greater(greater(hi, x[e]), x[e + 1]);
  }
  lo = lesser(lo, quad1(lo));
  hi = greater(hi, quad1(hi));
  lo = lesser(lo, quad2(lo));
  hi = greater(hi, quad2(hi));
  const bool bad = lo != lo;
  lo = fminf(fmaxf(lo, -65504.f), 65504.f);
  hi = hi < (X)-65504 ? (X)-65504 : hi > (X)65504 ? (X)65504 : hi;
  asm("" : "+v"(lo));                                   // (or the compiler makes one rounding of the two)
  least = (f16)lo;
  {
    constexpr double inv = 1. / MOST;
    const double range = (double)hi - (double)(float)least, q = range * inv;
    float nearest = (float)fma(fma(-(double)MOST, q, range), inv, q);   // (one step from a quotient that is off by its last bit: rounded to the nearest)
    asm("" : "+v"(nearest));
    step = (f16)nearest;
  }
  if (bad) least = __builtin_bit_cast(f16, (uint16_t)0x7e00), step = (f16)0.f;
  const float l32 = (float)least, s32 = (float)step;
  if (s32 == 0.f) return;
  // (step is below zero where the least value was rounded up past the greatest one)
  // the quotient rounded in the low bits of 1.5 * 2^23 + it
  const float inv = __builtin_amdgcn_rcpf(s32), magic = 12582912.f;
  float n[8], off = 0.f;
#pragma unroll
  for (int e = 0; e < 8; e++) {
    const float d = y[e] - l32;
    n[e] = fmaf(d, inv, magic) - magic;
    off = fmaxf(off, fabsf(fmaf(d, inv, -n[e])));
  }
  // x - least is off by 2^-24 of itself, the reciprocal by 2^-23, so the quotient by 3 * 2^-24 * MOST, and by 2^-24 x / step more where x was rounded: decided in 64 bits where
  // the middle is as near
  float sure = 0.5f - MOST * 0x1p-22f;
  if constexpr (sizeof(X) == 8) sure -= fmaxf(fabsf(lo), fabsf((float)hi)) * fabsf(inv) * 0x1p-23f;
  if (off > sure) {
    const double h = 0.5 * fabs((double)s32);
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const double d = (double)x[e] - (double)l32;
      // (turned elements that fp32 does not tell apart may be many codes from n: their quotient in 64 bits, by the same reciprocal, is less than one off)
      const float n0 = __builtin_amdgcn_fmed3f(sizeof(X) == 8 ? (float)__builtin_rint(d * (double)inv) : n[e], 0.f, (float)MOST);
      const double rest = d - (double)n0 * (double)s32, rem = s32 < 0.f ? -rest : rest;
      const bool odd = (int)n0 & 1;
      n[e] = n0 + (rem > h || (rem == h && odd) ? 1.f : 0.f) - (rem < -h || (rem == -h && odd) ? 1.f : 0.f);
    }
  }
  if constexpr (BITS == 4) {
#pragma unroll
    for (int e = 0; e < 8; e++) n[e] = __builtin_amdgcn_fmed3f(n[e], 0.f, 15.f);
    const float even = fmaf(fmaf(fmaf(n[6], 16.f, n[4]), 16.f, n[2]), 16.f, n[0]), odd = fmaf(fmaf(fmaf(n[7], 16.f, n[5]), 16.f, n[3]), 16.f, n[1]);
    w[0] = (uint32_t)even | (uint32_t)odd << 16;
  } else {                                              // (the conversion keeps to 0 .. 255)
#pragma unroll
    for (int e = 0; e < 8; e++) w[e >> 2] = __builtin_amdgcn_cvt_pk_u8_f32(n[e], e & 3, w[e >> 2]);
  }
}

// The turned elements of the thread's chunk j
template <int CHUNKS> __device__ __forceinline__ void turn_chunk(double (&y)[8], const float (&x)[8], int j, int pairs, bool neighbours, const TurnF64 *turns) {
  if (neighbours) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const double p = x[2 * i], q = x[2 * i + 1];
      if (4 * j < pairs) {                                // (a multiple of four)
        const TurnF64 t = turns[4 * j + i];
        y[2 * i] = fma(p, t.cos, -q * t.sin);
        y[2 * i + 1] = fma(p, t.sin, q * t.cos);
      } else {
        y[2 * i] = p;
        y[2 * i + 1] = q;
      }
    }
    return;
  }
  const int half = pairs >> 3;                            // chunks
  const bool low = j < half, turned = j < 2 * half;
  const int lane = threadIdx.x & 63, other = turned ? (low ? lane + half : lane - half) : lane;   // (of the same head, so of the same wavefront)
#pragma unroll
  for (int e = 0; e < 8; e++) {
    const float b = __shfl(x[e], other);
    y[e] = x[e];
    if (turned) {
      const TurnF64 t = turns[8 * (low ? j : j - half) + e];
      y[e] = fma((double)x[e], t.cos, (low ? -(double)b : (double)b) * t.sin);
    }
  }
}

// A workgroup per position.  SCAN: few positions, a later one with the same slot is looked for here; else owner says which is last.
template <typename T, int BITS, int D, bool SCAN, bool ROTATED> __global__ void __launch_bounds__(256) k_cache_write(CacheArgs a) {
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
  __shared__ TurnF64 turns[ROTATED ? D / 2 : 1];
  if constexpr (ROTATED) {
    if (tid < a.pairs) turns[tid] = turn_of_f64(as_table(a.positions)[t], a.fractions[tid]);
    __syncthreads();
  }
  // wavefronts 0 and 2 have keys, 1 and 3 values
  const int page = slot >> a.block_shift, at = slot & (a.block - 1), wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, value = wave & 1;
  const int j = lane % CHUNKS, g = j >> 2, c = j & 3;
  const T *from = (value ? reinterpret_cast<const T *>(a.v) + t * a.v_st : reinterpret_cast<const T *>(a.k) + t * a.k_st) + 8 * j;
  const int64_t stride = value ? a.v_sh : a.k_sh, bytes = P::bytes(a.block);
  unsigned char *codes = a.pages + (int64_t)page * a.heads * bytes + P::codes(a.block, value) + at * P::ROW + P::chunk(c, g);
  unsigned char *meta = a.pages + (int64_t)page * a.heads * bytes + P::meta(a.block, value) + at * P::META + 4 * g;
  constexpr int HEADS = 64 / CHUNKS;                    // of a wavefront
  for (int head = (wave >> 1) * HEADS + lane / CHUNKS; head < a.heads; head += 2 * HEADS) {
    float x[8];
    load8<T>(x, from + head * stride);
    uint32_t w[2] = {0u, 0u};
    f16 least, step;
    if (ROTATED && !value) {
      double y[8];
      turn_chunk<CHUNKS>(y, x, j, a.pairs, a.neighbours, turns);
      quantise<BITS>(y, w, least, step);
    } else {
      quantise<BITS>(x, w, least, step);
    }
    unsigned char *to = codes + head * bytes;
    if constexpr (BITS == 4) *reinterpret_cast<uint32_t *>(to) = w[0];
    else *reinterpret_cast<u32x2 *>(to) = u32x2{w[0], w[1]};
    if (c == 0) *reinterpret_cast<uint32_t *>(meta + head * bytes) = (uint32_t)__builtin_bit_cast(uint16_t, step) | (uint32_t)__builtin_bit_cast(uint16_t, least) << 16;
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

template <typename T, int BITS, int D, bool ROTATED> void launch_cache_write(const CacheArgs &a, hipStream_t st) {
  if (a.T <= kScan) {
    hipLaunchKernelGGL((k_cache_write<T, BITS, D, true, ROTATED>), dim3((unsigned)a.T), dim3(256), 0, st, a);
  } else {
    launch_slot_owners(a.slots, a.T, a.capacity, a.owner, st);
    hipLaunchKernelGGL((k_cache_write<T, BITS, D, false, ROTATED>), dim3((unsigned)a.T), dim3(256), 0, st, a);
  }
}
template <typename T, int BITS, int D> int launch_cache(const CacheArgs &a, bool write, hipStream_t st) {
  if (!write) hipLaunchKernelGGL((k_cache_read<T, BITS, D>), dim3((unsigned)a.T), dim3(256), 0, st, a);
  else if (a.fractions) launch_cache_write<T, BITS, D, true>(a, st);
  else launch_cache_write<T, BITS, D, false>(a, st);
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

static int cache_write(int dtype, void *pages, int n_pages, int block, int heads, int D, int bits, const void *k, int64_t k_stride_t, int64_t k_stride_h,
                       const void *v, int64_t v_stride_t, int64_t v_stride_h, const int32_t *slots, int T, int32_t *owner, CacheArgs &a) {
  const int rc = cache_args(dtype, pages, n_pages, block, heads, D, bits, slots, T, a);
  if (rc != BSP_OK) return rc;
  const int unit = dtype == BSP_F32 ? 4 : 8;
  if (!k || !v || !owner || ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15)) return BSP_ERR_ARG;
  if (k_stride_t % unit || k_stride_h % unit || v_stride_t % unit || v_stride_h % unit) return BSP_ERR_ARG;
  a.k = k; a.v = v; a.k_st = k_stride_t; a.k_sh = k_stride_h; a.v_st = v_stride_t; a.v_sh = v_stride_h;
  a.owner = owner;
  return BSP_OK;
}

extern "C" int bsp_cache_write(int dtype, void *pages, int n_pages, int block, int heads, int D, int bits, const void *k, int64_t k_stride_t, int64_t k_stride_h,
                               const void *v, int64_t v_stride_t, int64_t v_stride_h, const int32_t *slots, int T, int32_t *owner, void *stream) {
  CacheArgs a;
  const int rc = cache_write(dtype, pages, n_pages, block, heads, D, bits, k, k_stride_t, k_stride_h, v, v_stride_t, v_stride_h, slots, T, owner, a);
  return rc != BSP_OK ? rc : launch_cache(dtype, a, bits, D, true, as_stream(stream));
}

extern "C" int bsp_cache_write_rotated(int dtype, void *pages, int n_pages, int block, int heads, int D, int bits, const void *k, int64_t k_stride_t, int64_t k_stride_h,
                                       const void *v, int64_t v_stride_t, int64_t v_stride_h, const int32_t *slots, int T, int32_t *owner, const uint64_t *fractions, int pairs,
                                       int neighbours, const int32_t *positions, void *stream) {
  CacheArgs a;
  const int rc = cache_write(dtype, pages, n_pages, block, heads, D, bits, k, k_stride_t, k_stride_h, v, v_stride_t, v_stride_h, slots, T, owner, a);
  if (rc != BSP_OK) return rc;
  if (!rotation_ok(fractions, pairs, D) || !positions) return BSP_ERR_ARG;
  a.fractions = fractions; a.pairs = pairs; a.neighbours = neighbours != 0; a.positions = positions;
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
