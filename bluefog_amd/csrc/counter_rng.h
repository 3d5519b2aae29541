// Copyright 2026. Licensed under the Apache License, Version 2.0.
//
// Counter-based random bits for the dropout masks: Philox4x32 with 7 rounds
// (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3",
// SC 2011; 7 rounds are the fewest that the paper reports as passing BigCrush,
// and a round is what the masks cost). A mask is a function of (seed, offset,
// position): the backward pass computes it again, nothing is stored.
//
// One call gives four words, used as eight 16-bit values. An element is kept
// if its value is at least `threshold` = round(65536 p), so p is held to 16
// bits and the kept elements are scaled by 65536 / (65536 - threshold), which
// keeps the expectation exact for the probability that is really used.
//
// Attention: the keys of sixteen share two calls by quads, 0-3 and 8-11, and 4-7
// and 12-15, which is how a 32x32 matrix tile spreads them over lanes: key j of
// (head, packed query row) takes value ((j >> 3) & 1) * 4 + (j & 3) of the call with
// counter ((j >> 4) * 2 + ((j >> 2) & 1), row, head, offset).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "transformer_kernels.h"

struct BfKey {
  uint32_t k0, k1;
};

__device__ __forceinline__ BfKey bf_key(const BfDropout& d) {
  const uint64_t s = d.seed_ptr ? static_cast<uint64_t>(*d.seed_ptr) : d.seed;
  return {static_cast<uint32_t>(s), static_cast<uint32_t>(s >> 32)};
}

// one instruction; 0x96 is the truth table of the exclusive or of three
__device__ __forceinline__ uint32_t bf_xor3(uint32_t a, uint32_t b, uint32_t c) {
  return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96);
}

__device__ __forceinline__ uint4 bf_philox(uint32_t c0, uint32_t c1,
                                           uint32_t c2, uint32_t c3, BfKey k) {
#pragma unroll
  for (int i = 0; i < 7; ++i) {
    const uint64_t a = static_cast<uint64_t>(c0) * 0xD2511F53u;
    const uint64_t b = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
    c0 = bf_xor3(static_cast<uint32_t>(b >> 32), c1, k.k0);
    c1 = static_cast<uint32_t>(b);
    c2 = bf_xor3(static_cast<uint32_t>(a >> 32), c3, k.k1);
    c3 = static_cast<uint32_t>(a);
    k.k0 += 0x9E3779B9u;
    k.k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

// value u (0..7) of a call
__device__ __forceinline__ uint32_t bf_half(const uint4& w, int u) {
  const uint32_t x = u < 4 ? (u < 2 ? w.x : w.y) : (u < 6 ? w.z : w.w);
  return u & 1 ? x >> 16 : x & 0xFFFFu;
}

// the eight values of elements 8*block .. 8*block+7 of a tensor in row-major
// order
__device__ __forceinline__ uint4 bf_flat_bits(uint64_t block,
                                              const BfDropout& d, BfKey k) {
  return bf_philox(static_cast<uint32_t>(block),
                   static_cast<uint32_t>(block >> 32), 0u, d.offset, k);
}
