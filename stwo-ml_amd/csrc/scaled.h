// Rows of words brought to 8 bits, each by its own scale.
#pragma once
#include <stdint.h>

#include "field.h"
#include "gemm.h"
#include "witness.h"

namespace gkr {

// A workgroup a row: the largest magnitude, then the words.  Where the launch that
// multiplies or packs the rows does not do it.
static __global__ void __launch_bounds__(1024) k_quantize_rows(const uint32_t* __restrict__ X, uint64_t k, uint32_t levels,
                                                               uint32_t* __restrict__ out, uint32_t* __restrict__ scales) {
  __shared__ uint32_t most[16];
  const uint32_t* const row = X + blockIdx.x * k;
  uint32_t a = 0;
#pragma unroll 4
  for (uint64_t i = threadIdx.x; i < k; i += 1024) a = max(a, size_of_word(row[i]));
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) a = max(a, (uint32_t)__shfl_xor(a, off));
  if ((threadIdx.x & 63) == 0) most[threadIdx.x >> 6] = a;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 16; w++) a = max(a, most[w]);
  const Quantizer q(a, levels);
#pragma unroll 4
  for (uint64_t i = threadIdx.x; i < k; i += 1024) out[blockIdx.x * k + i] = word_of(q(row[i]));
  if (threadIdx.x == 0) scales[blockIdx.x] = a;
}

}  // namespace gkr
