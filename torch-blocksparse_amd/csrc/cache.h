// The pages of a quantised key-value cache (cache.hip writes and reads them back, cache_attention.hip attends over them).
//
// A page holds `block` consecutive positions of a sequence for every key head.  Page p, head h start at byte (p * heads + h) * page_bytes:
//     codes of the keys [block][D * bits / 8], steps and least values of the keys [block][D / 32] (fp16 step, fp16 least), then the same of the values.
// A group of 32 consecutive elements of a head stands for least + code * step.  What one workgroup reads of a page lies together, and
// a position's bytes are 5 / 8 (9 / 8) of its elements.
//
// Order of the codes.  Eight elements (a chunk) are `bits` bytes.  Chunk 4 g + c (the c-th of group g) is stored as number
// c * (D / 32) + g of its row: a lane of the attention kernel then finds chunk c of all groups in one run of bytes, which is its part of
// the D / 32 MFMA operands (one a group, so that a group's step multiplies the finished product).  In four bits, element 2 i of a
// chunk is nibble i and element 2 i + 1 nibble 4 + i: one shift and one `and` give two neighbours in the halves of a register.
#ifndef BSP_CACHE_H
#define BSP_CACHE_H
#include "bsp_common.h"

namespace bsp {

template <int BITS, int D> struct Page {
  static constexpr int GROUPS = D / 32, ROW = D * BITS / 8, META = 4 * GROUPS, CHUNK = BITS;   // bytes of a position's codes, of its steps, of a chunk
  static constexpr int64_t bytes(int block) { return 2 * (int64_t)block * (ROW + META); }
  static __host__ __device__ __forceinline__ int codes(int block, int value) { return value * block * (ROW + META); }
  static __host__ __device__ __forceinline__ int meta(int block, int value) { return value * block * (ROW + META) + block * ROW; }
  static __host__ __device__ __forceinline__ int chunk(int c, int g) { return (c * GROUPS + g) * CHUNK; }
};

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// (bits & mask) | 0x64006400, one operation: its two constants are in a scalar and in a vector register, as one instruction reads one scalar
__device__ __forceinline__ f16x2 code_pair(uint32_t bits, uint32_t mask, uint32_t magic) {
  uint32_t x;
  asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(x) : "v"(bits), "s"(mask), "v"(magic));
  return __builtin_bit_cast(f16x2, x);
}
// The eight codes of a chunk as fp16, in order: 0x6400 | code is the number 1024 + code, and 0x6400 | code << 4 (the nibbles 1 and 5 as they
// lie) 1024 + 16 code.
template <int BITS> __device__ __forceinline__ void chunk_codes(const uint32_t *w, f16x2 (&out)[4]) {
  const uint32_t magic = 0x64006400u;
  const f16x2 minus = {(_Float16)-1024.f, (_Float16)-1024.f};
  if constexpr (BITS == 4) {
    const uint32_t lo = w[0], hi = lo >> 8;
    const f16x2 sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f}, minus64 = {(_Float16)-64.f, (_Float16)-64.f};
    out[0] = code_pair(lo, 0x000f000fu, magic) + minus;
    out[1] = __builtin_elementwise_fma(code_pair(lo, 0x00f000f0u, magic), sixteenth, minus64);
    out[2] = code_pair(hi, 0x000f000fu, magic) + minus;
    out[3] = __builtin_elementwise_fma(code_pair(hi, 0x00f000f0u, magic), sixteenth, minus64);
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) out[i] = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(magic, w[i >> 1], i & 1 ? 0x05030502u : 0x05010500u)) + minus;
  }
}
// The same as operands of a product that is multiplied by 2^24 afterwards: a code is the bit pattern of the fp16 number code * 2^-24, which the matrix
// units take as it is.  In four bits elements 2, 3, 6 and 7 are 16 times that (code_up), for the other operand to make good.
template <int BITS> __device__ __forceinline__ void chunk_bits(const uint32_t *w, uint32_t (&out)[4]) {
  if constexpr (BITS == 4) {
    const uint32_t lo = w[0], hi = lo >> 8;
    out[0] = lo & 0x000f000fu;
    out[1] = lo & 0x00f000f0u;
    out[2] = hi & 0x000f000fu;
    out[3] = hi & 0x00f000f0u;
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) out[i] = __builtin_amdgcn_perm(0, w[i >> 1], i & 1 ? 0x0c030c02u : 0x0c010c00u);
  }
}
template <int BITS> __device__ __forceinline__ constexpr int code_up(int i) { return BITS == 4 && (i & 2) ? 4 : 0; }    // log2 of that factor

}  // namespace bsp
#endif
