// Rows of words brought to 8 bits, each by its own scale.
#pragma once
#include <stdint.h>

#include "field.h"
#include "gemm.h"

namespace gkr {

// round(c(x) levels / a), halves away from zero, for |c(x)| <= a: the quotient of
// 2 levels |c| + a (below 2^38) by 2 a.  The product with a rounded reciprocal is
// off by one at most; the rest, exact in 53 bits, says which way.
struct Quantizer {
  double inv, den, twice, half;
  __device__ __forceinline__ Quantizer(uint32_t a, uint32_t levels)
      : inv(a ? 0.5 / a : 0.0), den(2.0 * a), twice(2.0 * levels), half(a) {}
  __device__ __forceinline__ int32_t operator()(uint32_t x) const {
    const int32_t v = center_m31(x), sign = v >> 31;
    const double num = __builtin_fma((double)((v ^ sign) - sign), twice, half);
    const double q = __builtin_floor(num * inv), rest = __builtin_fma(-q, den, num);
    const int32_t r = (int32_t)q + (rest < 0 ? -1 : rest >= den && den > 0 ? 1 : 0);
    return (r ^ sign) - sign;
  }
};
__device__ __forceinline__ uint32_t word_of(int32_t v) { return (uint32_t)v + ((uint32_t)(v >> 31) & P); }

// A workgroup a row: the largest magnitude, then the words.
static __global__ void __launch_bounds__(256) k_quantize_rows(const uint32_t* __restrict__ X, uint64_t k, uint32_t levels,
                                                              uint32_t* __restrict__ out, uint32_t* __restrict__ scales) {
  __shared__ uint32_t most[4];
  const uint32_t* const row = X + blockIdx.x * k;
  uint32_t a = 0;
  for (uint64_t i = threadIdx.x; i < k; i += 256) {
    const int32_t v = center_m31(row[i]);
    a = max(a, (uint32_t)(v < 0 ? -v : v));
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) a = max(a, (uint32_t)__shfl_xor(a, off));
  if ((threadIdx.x & 63) == 0) most[threadIdx.x >> 6] = a;
  __syncthreads();
  a = max(max(most[0], most[1]), max(most[2], most[3]));
  const Quantizer q(a, levels);
  for (uint64_t i = threadIdx.x; i < k; i += 256) out[blockIdx.x * k + i] = word_of(q(row[i]));
  if (threadIdx.x == 0) scales[blockIdx.x] = a;
}

}  // namespace gkr
