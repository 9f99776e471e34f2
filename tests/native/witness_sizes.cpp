// Test-only host build of the witness operators' size limits (stwo-ml_amd/csrc/witness_sizes.h).
#include "../../stwo-ml_amd/csrc/witness_sizes.h"

extern "C" {
uint32_t ws_outside() { return gkr::kOutside; }
uint32_t ws_row_lds() { return gkr::kRowLds; }
uint64_t ws_max_inner() { return gkr::kMaxInner; }
int ws_few_rows_fit(uint64_t m, uint64_t k, uint64_t n, int one_plane) {
  return gkr::few_rows_fit(m, k, n, one_plane != 0);
}
uint64_t ws_pack_groups(uint64_t m, uint64_t k) { return gkr::pack_groups(m, k); }
int ws_packable(uint64_t m, uint64_t k, uint64_t n) { return gkr::packable(m, k, n); }
}
