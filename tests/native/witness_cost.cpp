// Test-only host build of the rule that chooses a packed product's kernel (stwo-ml_amd/csrc/witness_cost.h).
#include "../../stwo-ml_amd/csrc/witness_cost.h"

// 0 tiles, 1 mixed, 2 wide, 3 blocks
extern "C" int wc_kernel(uint64_t m, uint64_t k, uint64_t n, int gated, int quant) {
  const uint32_t nsteps = (uint32_t)((k + 31) / 32);
  return (int)gkr::PackedCost(m, n, nsteps, gated != 0, false, quant != 0).kernel(m, n, nsteps, gated != 0, quant != 0);
}
