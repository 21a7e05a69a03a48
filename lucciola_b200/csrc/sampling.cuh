// The samplers' random numbers: a counter-based hash of (key of the request, index of the generated token, vocabulary index).
#pragma once

#include "common.cuh"

namespace lb {

__host__ __device__ __forceinline__ unsigned long long mix64(unsigned long long x) {
  x ^= x >> 30; x *= 0xBF58476D1CE4E5B9ull;
  x ^= x >> 27; x *= 0x94D049BB133111EBull;
  x ^= x >> 31;
  return x;
}

// The top 23 bits of a hash as a number strictly inside (0, 1): (b + 0.5) / 2^23.  b + 0.5 has at most 24
// significant bits, so every value is exact in float32; the smallest is 2^-24 and the largest 1 - 2^-24.  (With
// 24 bits the largest sum, 16777215.5, would round to 2^24 and give exactly 1, whose score is +infinity.)
__host__ __device__ __forceinline__ float bits_to_uniform(unsigned int bits23) {
  return ((float)bits23 + 0.5f) * (1.0f / 8388608.0f);
}

// What all of a row's numbers have in common, and the 23 bits of vocabulary index i.
__host__ __device__ __forceinline__ unsigned long long hash_row(unsigned long long key, unsigned int counter) {
  return mix64(key + 0x9E3779B97F4A7C15ull * (unsigned long long)(counter + 1u));
}
// (mix64 without its last step, which changes the low 33 bits alone)
__host__ __device__ __forceinline__ unsigned int hash_bits(unsigned long long row, unsigned int i) {
  unsigned long long x = row ^ (0xD6E8FEB86659FD93ull * (unsigned long long)(i + 1u));
  x ^= x >> 30; x *= 0xBF58476D1CE4E5B9ull;
  x ^= x >> 27; x *= 0x94D049BB133111EBull;
  return (unsigned int)(x >> 41);
}

// Uniform in (0, 1) with 23 bits.
__host__ __device__ __forceinline__ float hash_uniform(unsigned long long key, unsigned int counter, unsigned int i) {
  return bits_to_uniform(hash_bits(hash_row(key, counter), i));
}

// The score of temperature sampling without filters: logit / T - log(-log(u)).
__device__ __forceinline__ float gumbel_score(float logit, float inv_t, float u) { return __fmaf_rn(logit, inv_t, -logf(-logf(u))); }

}  // namespace lb
