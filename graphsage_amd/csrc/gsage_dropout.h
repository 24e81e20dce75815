// The counter hash behind every dropout mask: an element is kept or not by (seed, element index) alone,
// so a mask is never stored, a backward pass draws it again, and two kernels that see the same element
// of the same table under the same seed agree about it.
#pragma once
#include "gsage_common.h"

// ------------------------------------------------------------------ dropout hash RNG
// keep(seed, idx) with idx = row*F + col; mirrored in graphsage_amd/rng.py for tests.
// 32-bit arithmetic only (64-bit multiplies are emulated on the VALU): a bijective scramble
// of the element index keyed by the seed, then murmur3's fmix32 avalanche.
__device__ __forceinline__ bool dropout_keep(uint64_t seed, uint64_t idx, float p) {
  uint32_t lo = (uint32_t)idx, hi = (uint32_t)(idx >> 32);
  uint32_t h = (uint32_t)seed ^ (lo * 0x9E3779B1u);
  h ^= (uint32_t)(seed >> 32) + hi * 0x85EBCA77u;
  h ^= h >> 16;
  h *= 0x85EBCA6Bu;
  h ^= h >> 13;
  h *= 0xC2B2AE35u;
  h ^= h >> 16;
  float u = (float)(h >> 8) * (1.0f / 16777216.0f);  // 24 random bits -> [0,1)
  return u >= p;
}

// The hash in two parts for many elements of one upper index word: the key (once per 2^32 elements) and the draw, given
// lo(idx) * DROPOUT_STEP (of a run's followers: the first product plus multiples of the step; v_mul_lo_u32 is a
// quarter-rate instruction).  u >= p on u = k 2^-24 is k >= ceil(p 2^24) on the integer k = h >> 8, i.e.
// h >= ceil(p 2^24) << 8 (p < 1, so the threshold fits): kept where dropout_draw(..) >= dropout_threshold(p), bit for
// bit the masks of dropout_keep.
constexpr uint32_t DROPOUT_STEP = 0x9E3779B1u;
__device__ __forceinline__ uint32_t dropout_threshold(float p) { return ((uint32_t)ceilf(p * 16777216.0f)) << 8; }
__device__ __forceinline__ uint32_t dropout_word(uint64_t seed, uint32_t hi) {
  return (uint32_t)seed ^ ((uint32_t)(seed >> 32) + hi * 0x85EBCA77u);
}
__device__ __forceinline__ uint32_t dropout_draw(uint32_t word, uint32_t m) {
  uint32_t h = word ^ m;
  h ^= h >> 16;
  h *= 0x85EBCA6Bu;
  h ^= h >> 13;
  h *= 0xC2B2AE35u;
  h ^= h >> 16;
  return h;
}

// four consecutive elements whose indices fit 32 bits (idx + 3 < 2^32), at about half the instructions
__device__ __forceinline__ void dropout_keep4_lo(uint64_t seed, uint32_t idx, uint32_t thr, bool (&k)[4]) {
  const uint32_t word = dropout_word(seed, 0), m0 = idx * DROPOUT_STEP;
#pragma unroll
  for (int i = 0; i < 4; ++i) k[i] = dropout_draw(word, m0 + (uint32_t)i * DROPOUT_STEP) >= thr;
}
