// Which sizes the witness operators' kernels take (host only where it is not
// a constant): what they address in 32 bits, and what a launch's grid holds.
#pragma once
#include <stdint.h>

namespace gkr {

// Bytes that a buffer descriptor covers at most here, and the offset behind
// them all that stands for "no such place" (witness.h).
constexpr uint32_t kOutside = 0xfffffff0u;
constexpr uint32_t kRowLds = 65536;  // digits of a few rows' products in LDS at a time
// Longest inner size of the kernels here: a digit sum stays below 2^31.
// Beyond it (no model's layer) the forward product's passes of K are used,
// with the element-wise work in a launch behind.
constexpr uint64_t kMaxInner = 131071;

// Whether k_rows takes an m x k by k x n product: up to four rows; five to
// sixteen by weights of one plane while their digits fit in LDS at once (every
// workgroup makes them again, which takes it longer beyond than a launch that
// packs them).  It writes the output through one buffer, byte offsets 4 (r n + c).
inline bool few_rows_fit(uint64_t m, uint64_t k, uint64_t n, bool one_plane) {
  if (k > kMaxInner || n > 1ull << 26 || m > 16 || 4 * m * n > kOutside) return false;
  if (m <= 4) return true;
  return one_plane && (m <= 8 ? 8 : 16) * 4 * ((k + 63) / 64 * 64) <= kRowLds;
}

constexpr uint64_t kProductStep = 32;     // K per operand block (gemm.h)
constexpr uint64_t kPackThreads = 256;    // of k_wit_pack, a block of eight rows a wave
inline uint64_t pack_groups(uint64_t m, uint64_t k) {
  return ((m + 7) / 8 * ((k + kProductStep - 1) / kProductStep) + 3) / 4;
}
// Whether the packed product takes it: its grids (the packing's has fewer than
// 2^32 threads, as any dimension), its 32-bit counts of blocks and its offsets
// of steps and of a workgroup's rows (256 of 2^21 words).
inline bool packable(uint64_t m, uint64_t k, uint64_t n) {
  return k <= kMaxInner && m <= 1ull << 22 && n <= 1ull << 21 && pack_groups(m, k) * kPackThreads < 1ull << 32 &&
         (m / 64 + 1) * (n / 128 + 1) <= 1ull << 21;
}

}  // namespace gkr
