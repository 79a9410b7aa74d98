// threefry.hpp — the block function of Threefry-2x32, 20 rounds (nx_c_random.c:36-133), for the
// generator of the contract (move.hip) and the operators that draw as they go (dropout.hip).
#pragma once

#include "nxh_common.hpp"

__device__ __forceinline__ uint32_t rotl32(uint32_t x, int r) { return (x << r) | (x >> (32 - r)); }
// (x0, x1), a counter, becomes 64 random bits.
__device__ __forceinline__ void threefry_block(uint32_t k0, uint32_t k1, uint32_t &x0, uint32_t &x1) {
  const uint32_t ks[3] = {k0, k1, 0x1BD11BDAu ^ k0 ^ k1};
  x0 += k0;
  x1 += k1;
  constexpr int rots[8] = {13, 15, 26, 6, 17, 29, 16, 24};
#pragma unroll
  for (int r = 0; r < 20; r++) {
    x0 += x1;
    x1 = rotl32(x1, rots[r % 8]);
    x1 ^= x0;
    if ((r + 1) % 4 == 0) {
      const int s = (r + 1) / 4;
      x0 += ks[s % 3];
      x1 += ks[(s + 1) % 3] + (uint32_t)s;
    }
  }
}
