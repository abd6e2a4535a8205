// The pages of a cache of latent vectors (latent_cache.hip writes them and reads them back, latent_attention.hip attends over them): row `slot` = page * block + offset has
// the position's latent vector and, behind it, the key part that all heads share, both in one 16-bit type.
#ifndef BSP_LATENT_H
#define BSP_LATENT_H
#include "bsp_common.h"

namespace bsp {

constexpr int kRope = 64;          // elements of the shared key part
inline bool latent_ok(int latent, int block) { return (latent == 128 || latent == 256 || latent == 512) && (block == 16 || block == 32 || block == 64 || block == 128); }

}  // namespace bsp
#endif
