// The counter-based generator of the normals and of dropout's masks: Philox4x32 with 10 rounds (Salmon, Moraes, Dror
// and Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011). A round multiplies words 0 and 2 by the
// published constants 0xD2511F53 and 0xCD9E8D57, keeps the low halves and XORs the high halves with words 1, 3 and
// the key; the key is bumped by the Weyl increments 0x9E3779B9 and 0xBB67AE85 between rounds.
#pragma once
#include "common.h"

namespace psgdk {

__device__ __forceinline__ void philox4x32_10(uint32_t (&c)[4], uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    // one 32 x 32 -> 64-bit product per word (one v_mad_u64_u32) rather than separate low and high multiplies
    const uint64_t p0 = (uint64_t)0xD2511F53u * c[0], p1 = (uint64_t)0xCD9E8D57u * c[2];
    const uint32_t lo0 = (uint32_t)p0, hi0 = (uint32_t)(p0 >> 32);
    const uint32_t lo1 = (uint32_t)p1, hi1 = (uint32_t)(p1 >> 32);
    c[0] = hi1 ^ c[1] ^ k0;
    c[1] = lo1;
    c[2] = hi0 ^ c[3] ^ k1;
    c[3] = lo0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
}

}  // namespace psgdk
