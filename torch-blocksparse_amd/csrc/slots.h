// Which of the positions that are given one slot of a cache is written (cache.hip, latent_cache.hip): the last.
#ifndef BSP_SLOTS_H
#define BSP_SLOTS_H
#include "bsp_common.h"

namespace bsp {
namespace {

// owner[slot] (zero between calls) becomes the greatest number t + 1 among the positions t of the slot
__global__ void __launch_bounds__(256) k_slot_owner(const int32_t *slots, int T, int64_t capacity, int32_t *owner) {
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t >= T) return;
  const int slot = slots[t];
  if (slot >= 0 && slot < capacity) atomicMax(owner + slot, t + 1);
}
void launch_slot_owners(const int32_t *slots, int T, int64_t capacity, int32_t *owner, hipStream_t st) {
  hipLaunchKernelGGL(k_slot_owner, dim3((unsigned)cdiv(T, 256)), dim3(256), 0, st, slots, T, capacity, owner);
}

}  // namespace
}  // namespace bsp
#endif
