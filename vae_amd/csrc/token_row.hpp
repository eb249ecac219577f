// What the token kernels (token.hip, distill.hip) share: a row of logits over a vocabulary, its softmax statistics and
// the ids that index it.  No reference counterpart: the reference's likelihoods are Bernoulli, Gaussian and the
// discretized logistic (abstract_vae.py:461-471); this is the categorical one.
//
// Statistics of a row x[V] at scale c = log2(e) / temperature:  m = max x,  s = sum 2^((x - m) c).
//   p_j = 2^((x_j - m) c) / s,   ln p_j = ln2 ((x_j - m) c - log2 s).
// The difference is formed before it is scaled: x = m gives exactly 1, and a row whose maximum is the type's lowest
// value (a mask written with it) does not overflow.  An all -inf row has s = 0 and no distribution: log p = -inf,
// entropy 0, gradient 0.  A NaN or +inf logit makes s NaN and with it everything the row returns.
#pragma once
#include "common.hpp"

namespace vae {

// ids come as int32 or int64
__device__ __forceinline__ int64_t load_id(const void* __restrict__ ids, int id_bytes, int64_t i) {
  return id_bytes == 4 ? (int64_t) reinterpret_cast<const int32_t*>(ids)[i] : reinterpret_cast<const int64_t*>(ids)[i];
}

// the largest finite-or-minus-infinite value a statistic is taken against: -inf would make x - m NaN
constexpr float kLowest = -3.402823466e38f;

__device__ __forceinline__ float nan_f() { return __builtin_nanf(""); }

// ln p of a value with statistics (m, s); s == 0: an empty row.  In natural units: x - m of the type's range does not
// overflow here, times log2(e) it could.
__device__ __forceinline__ float row_log_prob(float x, float m, float s, float inv_tau) {
  return s == 0.f ? -INFINITY : (x - m) * inv_tau - kLn2 * log2f(s);
}

// (value, index) as one sortable integer: larger value first, then the lower index; a NaN is below everything
__device__ __forceinline__ uint32_t order_bits(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);  // -0 and +0 are one value
  return x != x ? 0u : ((b & 0x80000000u) ? ~b : (b | 0x80000000u));
}
__device__ __forceinline__ float order_value(uint32_t o) {
  return __uint_as_float((o & 0x80000000u) ? (o ^ 0x80000000u) : ~o);
}
__device__ __forceinline__ uint64_t order_key(float x, uint32_t index) {
  return ((uint64_t)order_bits(x) << 32) | (uint32_t)(~index);
}

// sum / max over a workgroup of 256 in a fixed order; every thread gets the result
__device__ __forceinline__ uint64_t block_max_u64(uint64_t v) {
  __shared__ uint64_t lds_k[kBlock / 64];
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    const uint64_t w = __shfl_xor(v, o, 64);
    v = w > v ? w : v;
  }
  lds_barrier();
  if ((threadIdx.x & 63) == 0) lds_k[threadIdx.x >> 6] = v;
  lds_barrier();
  uint64_t r = lds_k[0];
#pragma unroll
  for (int w = 1; w < kBlock / 64; ++w) r = lds_k[w] > r ? lds_k[w] : r;
  return r;
}

}  // namespace vae
