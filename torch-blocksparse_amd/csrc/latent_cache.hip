// Latent vectors into the pages of a cache, and back.  A row of a page is a position's latent vector and, behind it, the kRope = 64 elements of the key part that all heads
// share, in a 16-bit type; row `slot` of the cache starts at element slot * (latent + 64).  With a rotation (rotation.h) those 64 are turned on the way, in fp32, and rounded once.
//
// Bound by the bytes.  A workgroup has eight positions: their latent vectors in chunks of 16 bytes, their shared parts a pair of elements a thread, so that no angle is computed
// twice.  Measured: 20011 positions of 512 + 64 in bf16 with a rotation (46 MB): 12 us (3.8 TB/s), 2.5 more for the launch that says whose a slot is; 131072 of them (302 MB) 58 us with
// it (5.2 TB/s), 262144 120.  Read back: 9.4, 51 and 103 us (4.9 and 5.9 TB/s).
#include "latent.h"
#include "rotation.h"
#include "slots.h"

namespace bsp {

struct LatentCacheArgs {
  const void *c, *r;               // write: [T, latent], [T, 64], strides in elements
  void *co, *ro;                   // read: contiguous
  int64_t c_st, r_st;
  const int32_t *slots;
  int32_t *owner;
  void *pages;
  int64_t capacity;
  int T, latent, chunk_shift;      // log2 of the latent vector's chunks of eight elements
  const int32_t *positions;        // write, with a rotation
  const uint64_t *fractions;
  int pairs, neighbours;
};

namespace {

constexpr int kTogether = 8;       // positions of a workgroup

template <typename T, bool SCAN> __global__ void __launch_bounds__(256) k_latent_write(LatentCacheArgs a) {
  __shared__ int32_t place[kTogether];                  // the position's slot, or -1: it is not written
  const int first = blockIdx.x * kTogether, tid = threadIdx.x;
  if (tid < kTogether) {
    const int t = first + tid;
    int slot = t < a.T ? a.slots[t] : -1;
    if (slot < 0 || slot >= a.capacity) slot = -1;
    if (!SCAN && slot >= 0) {
      if (a.owner[slot] == t + 1) a.owner[slot] = 0;    // (another position of the slot that looks from now on finds 0: not the last either)
      else slot = -1;
    }
    place[tid] = slot;
  }
  __syncthreads();
  if constexpr (SCAN) {                                 // few positions: a later one with the same slot is looked for here
    const int i = tid >> 5, t = first + i, slot = place[i];
    bool later = false;
    if (slot >= 0)
      for (int u = t + 1 + (tid & 31); u < a.T; u += 32) later |= a.slots[u] == slot;
    __syncthreads();
    if (later) place[i] = -1;
    __syncthreads();
  }
  const int row = a.latent + kRope;
  T *pages = reinterpret_cast<T *>(a.pages);
  const T *pc = reinterpret_cast<const T *>(a.c), *pr = reinterpret_cast<const T *>(a.r);
#pragma unroll 2
  for (int i = tid; i < kTogether << a.chunk_shift; i += 256) {
    const int p = i >> a.chunk_shift, ch = i & ((1 << a.chunk_shift) - 1), slot = place[p];
    if (slot < 0) continue;
    *reinterpret_cast<u32x4 *>(pages + (int64_t)slot * row + 8 * ch) = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(pc + (first + p) * a.c_st + 8 * ch));
  }
  const int p = tid >> 5, i = tid & 31, slot = place[p];
  if (slot < 0) return;
  const bool turning = i < a.pairs;
  const int ia = !turning || a.neighbours ? 2 * i : i, ib = !turning || a.neighbours ? 2 * i + 1 : a.pairs + i;
  const T *from = pr + (first + p) * a.r_st;
  T *to = pages + (int64_t)slot * row + a.latent;
  T x = from[ia], y = from[ib];
  if (turning) {
    const Turn t = turn_of(a.positions[first + p], a.fractions[i]);
    turn_pair(to_float(x), to_float(y), t.cos, t.sin, x, y);
  }
  to[ia] = x;
  to[ib] = y;
}

// A chunk of eight elements a thread.  Slots outside the cache read as zeros.
__global__ void __launch_bounds__(256) k_latent_read(LatentCacheArgs a) {
  const uint32_t id = blockIdx.x * 256u + threadIdx.x, chunks = (uint32_t)(a.latent + kRope) >> 3;
  const Quotient at(id, chunks);
  if (at.q >= (uint32_t)a.T) return;
  const int slot = a.slots[at.q], ch = (int)at.r;
  u32x4 x = {0, 0, 0, 0};
  if (slot >= 0 && slot < a.capacity) x = *reinterpret_cast<const u32x4 *>(reinterpret_cast<const uint16_t *>(a.pages) + (int64_t)slot * (a.latent + kRope) + 8 * ch);
  const int own = a.latent >> 3;
  uint16_t *to = ch < own ? reinterpret_cast<uint16_t *>(a.co) + (int64_t)at.q * a.latent + 8 * ch : reinterpret_cast<uint16_t *>(a.ro) + (int64_t)at.q * kRope + 8 * (ch - own);
  __builtin_nontemporal_store(x, reinterpret_cast<u32x4 *>(to));
}

// Up to here each workgroup reads the slots behind its own, which costs less than a launch that says whose a slot is (64 positions 2.8 and 4.4 us, 512 4.3 and 5.1, 1024 6.1 and 5.2).
constexpr int kScan = 512;

template <typename T> void launch_latent_write(const LatentCacheArgs &a, hipStream_t st) {
  const dim3 grid((unsigned)cdiv(a.T, kTogether));
  if (a.T <= kScan) {
    hipLaunchKernelGGL((k_latent_write<T, true>), grid, dim3(256), 0, st, a);
  } else {
    launch_slot_owners(a.slots, a.T, a.capacity, a.owner, st);
    hipLaunchKernelGGL((k_latent_write<T, false>), grid, dim3(256), 0, st, a);
  }
}

int latent_cache_args(int dtype, const void *pages, int n_pages, int block, int latent, const int32_t *slots, int T, LatentCacheArgs &a) {
  if (!pages || (reinterpret_cast<uintptr_t>(pages) & 15) || n_pages <= 0 || !slots || T <= 0) return BSP_ERR_ARG;
  if ((dtype != BSP_F16 && dtype != BSP_BF16) || !latent_ok(latent, block)) return BSP_ERR_UNSUPPORTED;
  if ((int64_t)n_pages * block >= ((int64_t)1 << 31) || T >= (1 << 24)) return BSP_ERR_UNSUPPORTED;   // (a grid has fewer than 2^32 threads)
  a = LatentCacheArgs{};
  a.pages = const_cast<void *>(pages);
  a.capacity = (int64_t)n_pages * block;
  a.latent = latent; a.chunk_shift = __builtin_ctz(latent) - 3; a.slots = slots; a.T = T;
  return BSP_OK;
}

}  // namespace
}  // namespace bsp

using namespace bsp;

extern "C" int bsp_latent_write(int dtype, void *pages, int n_pages, int block, int latent, const void *c, int64_t c_stride_t, const void *r, int64_t r_stride_t, const int32_t *slots,
                                int T, int32_t *owner, const uint64_t *fractions, int pairs, int neighbours, const int32_t *positions, void *stream) {
  LatentCacheArgs a;
  const int rc = latent_cache_args(dtype, pages, n_pages, block, latent, slots, T, a);
  if (rc != BSP_OK) return rc;
  if (!c || !r || !owner || (reinterpret_cast<uintptr_t>(c) & 15) || (reinterpret_cast<uintptr_t>(r) & 1) || c_stride_t % 8) return BSP_ERR_ARG;
  if (fractions && (!rotation_ok(fractions, pairs, kRope) || !positions)) return BSP_ERR_ARG;
  a.c = c; a.r = r; a.c_st = c_stride_t; a.r_st = r_stride_t; a.owner = owner;
  if (fractions) a.fractions = fractions, a.pairs = pairs, a.neighbours = neighbours != 0, a.positions = positions;
  const hipStream_t st = as_stream(stream);
  if (dtype == BSP_F16) launch_latent_write<f16>(a, st);
  else launch_latent_write<bf16>(a, st);
  BSP_LAUNCH_CHECK();
  return BSP_OK;
}

extern "C" int bsp_latent_read(int dtype, const void *pages, int n_pages, int block, int latent, void *c, void *r, const int32_t *slots, int T, void *stream) {
  LatentCacheArgs a;
  const int rc = latent_cache_args(dtype, pages, n_pages, block, latent, slots, T, a);
  if (rc != BSP_OK) return rc;
  if (!c || !r || ((reinterpret_cast<uintptr_t>(c) | reinterpret_cast<uintptr_t>(r)) & 15)) return BSP_ERR_ARG;
  a.co = c; a.ro = r;
  hipLaunchKernelGGL(k_latent_read, dim3((unsigned)cdiv((int64_t)T * ((latent + kRope) / 8), 256)), dim3(256), 0, as_stream(stream), a);
  BSP_LAUNCH_CHECK();
  return BSP_OK;
}
