// The witness operators' element-wise end: bias, activation, residual and the
// gate's product, over canonical M31 words.
#pragma once
#include <stdint.h>

#include "field.h"

namespace gkr {

// act(z): table == nullptr and relu == 0 is z itself; the table's entry at
// z mod 2^log is what the LogUp layer proves (mask = 2^log - 1).
struct ActArg {
  const uint32_t* table;
  uint32_t mask, relu;
};
__device__ __forceinline__ uint32_t activate(const ActArg& a, uint32_t z) {
  if (a.table) return a.table[z & a.mask];
  return a.relu && z > (P >> 1) ? 0u : z;
}

// What happens to a sum of the product (fused) or a pair of sums (gated).
struct FusedEnd {
  ActArg act;
  const uint32_t* bias;      // n
  const uint32_t* residual;  // m x n; may be out (read by the thread that writes the element)
  uint32_t* pre;
  uint32_t* out;
};
__device__ __forceinline__ void fused_end(const FusedEnd& e, uint64_t at, uint64_t col, uint32_t z) {
  if (e.bias) z = m31_add(z, e.bias[col]);
  if (e.pre) e.pre[at] = z;
  uint32_t y = activate(e.act, z);
  if (e.residual) y = m31_add(y, e.residual[at]);
  e.out[at] = y;
}
struct GatedEnd {
  ActArg act;
  uint32_t *gate, *act_out, *up, *out;
};
__device__ __forceinline__ void gated_end(const GatedEnd& e, uint64_t at, uint32_t g, uint32_t u) {
  const uint32_t a = activate(e.act, g);
  if (e.gate) e.gate[at] = g;
  if (e.act_out) e.act_out[at] = a;
  if (e.up) e.up[at] = u;
  e.out[at] = m31_mul(a, u);
}

// One thread per element, behind the products.
static __global__ void k_fused_end(const uint32_t* __restrict__ z, uint64_t count, uint64_t n, FusedEnd e) {
  for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < count; i += (uint64_t)gridDim.x * blockDim.x)
    fused_end(e, i, i % n, z[i]);
}
static __global__ void k_gated_end(const uint32_t* __restrict__ g, const uint32_t* __restrict__ u, uint64_t count,
                                   GatedEnd e) {
  for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < count; i += (uint64_t)gridDim.x * blockDim.x)
    gated_end(e, i, g[i], u[i]);
}

}  // namespace gkr
