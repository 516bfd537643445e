// Random words for dropout: Philox4x32 with seven rounds, the counter-based
// generator of Salmon, Moraes, Dror and Shaw ("Parallel random numbers: as easy
// as 1, 2, 3", SC11; seven rounds are the fewest that pass all of its tests).
// Four words from a 128-bit counter and a 64-bit key; nothing is stored between
// calls. A round is two 32 x 32 -> 64 products (one instruction each, at a
// quarter of the rate) and two three-way exclusive ors; the round keys are
// uniform and stay in scalar registers.
#pragma once

#include "ngdn_common.h"

namespace ngdn {

struct PhiloxKey {
  uint32_t k0, k1, c2, c3;      // the key and the counter's upper half
  __device__ __forceinline__ PhiloxKey(uint64_t seed, uint64_t offset)
      : k0((uint32_t)seed), k1((uint32_t)(seed >> 32)), c2((uint32_t)offset), c3((uint32_t)(offset >> 32)) {}
};

__device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) {
  return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96);
}

// the words of counter (block, offset)
__device__ __forceinline__ void philox(const PhiloxKey& key, uint64_t block, uint32_t* out) {
  uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = key.c2, c3 = key.c3;
  uint32_t k0 = key.k0, k1 = key.k1;
#pragma unroll
  for (int r = 0; r < 7; ++r) {
    const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
    c0 = xor3((uint32_t)(b >> 32), c1, k0);
    c2 = xor3((uint32_t)(a >> 32), c3, k1);
    c1 = (uint32_t)b;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  out[0] = c0; out[1] = c1; out[2] = c2; out[3] = c3;
}

// words i .. i + 7 of the stream whose word i is word i % 4 of block i / 4;
// aligned: i is a multiple of four in every lane
__device__ __forceinline__ void philox8(const PhiloxKey& key, uint64_t i, bool aligned, uint32_t* w) {
  uint32_t t[12];
  philox(key, i >> 2, t);
  philox(key, (i >> 2) + 1, t + 4);
  if (aligned) {
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = t[e];
  } else {
    philox(key, (i >> 2) + 2, t + 8);
    // by masks: chosen by a condition, the words would become an array in memory
    const uint32_t one = 0u - (uint32_t)(i & 1), two = 0u - (uint32_t)(i >> 1 & 1);
#pragma unroll
    for (int e = 0; e < 11; ++e) t[e] ^= (t[e] ^ t[e + 1]) & one;
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = t[e] ^ ((t[e] ^ t[e + 2]) & two);
  }
}

}  // namespace ngdn
