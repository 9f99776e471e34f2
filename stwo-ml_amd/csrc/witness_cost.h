// What the kernels of a packed product (witness.h) take, in us, and which of them is
// taken for it (host only).
#pragma once
#include <stdint.h>

#include <algorithm>

namespace gkr {

// What the two kinds of kernel take, in us, to choose between them; fitted to 27
// products of 40 to 512 rows, k 100 to 13824, n 900 to 13824, rows and weights
// of one plane and of four, which each kind took 10 to 330 us for: within a
// quarter, and the better one taken in all but two (by 1.1 and 1.2 times).
// k_wit_tiles: 8 us for each round of the workgroups that fit at once (`slots`),
// and the operands' way from the second-level cache, 17 GB/ms; kb is a
// workgroup's K step.
inline double tiles_us(uint64_t groups, uint32_t slots, uint32_t nsteps, uint32_t kb) {
  return 8.0 * (double)((groups + slots - 1) / slots) + (double)groups * nsteps * kb / 17000.0;
}
// k_wit_blocks: a workgroup fills a CU; a K step takes it 0.27 us where few run
// and 0.5 on all 256 (the matrix cores slow down).  K splits fill the last
// round, against the parts' way through memory and a launch to join them.
inline double blocks_us(uint64_t groups, uint32_t nsteps, uint64_t elements, uint32_t* splits) {
  double best = 0;
  for (uint32_t s = 1; s <= 16 && (s == 1 || nsteps / s >= 16); s++) {
    const uint64_t rounds = (groups * s + 255) / 256, steps = (nsteps + s - 1) / s;
    const double step = 0.27 + 0.23 * std::min(1.0, (double)(groups * s) / 256);
    const double us = 12.0 + step * (double)(rounds * steps) + (s > 1 ? 5.0 + (double)s * (double)elements * 2e-6 : 0.0);
    if (s == 1 || us < best) {
      best = us;
      *splits = s;
    }
  }
  return best;
}

// k_wit_wide, 128 x 96 a workgroup: fitted to 24 products of 300 to 2048 rows, k 576 to
// 13824, n 1024 to 8000, 8 to 228 us without the packing, within a seventh; a quarter
// more, as the others' times are only that well known.  Beyond two rounds the rows and
// weights no longer lie in the second-level caches (5000 x 13824 x 5120 in nine rounds
// 640 us, k_wit_blocks 440).
inline double wide_us(uint64_t groups, uint32_t nsteps) {
  return groups > 512 ? 1e30 : 1.25 * (2.0 + (double)((groups + 255) / 256) * (9.0 + 0.09 * nsteps));
}

// The kernel of more than 64 rows by weights of one plane.  Whether the rows have one
// plane or four is found out on the device, by a launch that holds both ways of its
// kernel: the sum of the two is compared, with `quant` that of one plane alone.
enum class PackedKernel { kTiles, kMixed, kWide, kBlocks };
struct PackedCost {
  double blocks[2] = {0, 0};      // k_wit_blocks, for rows of one plane and of four
  uint32_t splits[2] = {1, 1};    // of K, there
  PackedCost(uint64_t m, uint64_t n, uint32_t nsteps, bool gated, bool general, bool quant) {
    const uint64_t ctiles = (n + 31) / 32, elements = m * n * (gated ? 2 : 1);
    const uint64_t bgroups = (ctiles * (gated ? 2 : 1) * (general ? 4 : 1) + 7) / 8;
    blocks[0] = blocks_us(((m + 31) / 32 + 7) / 8 * bgroups, nsteps, elements, &splits[0]);
    if (!quant) blocks[1] = blocks_us(((m + 7) / 8 + 7) / 8 * bgroups, nsteps, elements, &splits[1]);
  }
  PackedKernel kernel(uint64_t m, uint64_t n, uint32_t nsteps, bool gated, bool quant) const {
    const uint64_t ctiles = (n + 31) / 32, rows64 = (m + 63) / 64;
    const uint32_t nw = gated ? 2 : 1, down = m <= 128 ? nw : 2 * nw;  // waves down the rows of k_wit_mixed
    const double tiles = tiles_us(rows64 * ctiles, 512, nsteps, 2 + nw) +
                         (quant ? 0 : tiles_us(rows64 * ctiles, 512, nsteps, 4 * (2 + nw)));
    const double mixed =
        m <= 256 ? tiles_us(ctiles, 256, nsteps, down * ((gated ? 2 : 4) + nw)) + blocks[1] : 1e30;
    // k_wit_wide where it leads by what these times are known to, rows and weights from
    // memory (the fit's were in the caches): by a tenth where it leaves CUs idle that
    // splits of K fill, and against the streams by a launch to join splits of rows of four
    // planes, which has nothing to do for rows of one.  Of 570 products of 129 to 2048
    // rows, k 256 to 13824, n 512 to 13824 it takes 286, 0.57 to 1.07 times what they take
    // without it; with neither margin 35 took 1.03 to 1.23 times as long (330 x 4643 x
    // 2277: 29.7 us, 24.2 without).
    const uint64_t groups = (m + 127) / 128 * ((ctiles + 2) / 3);
    const double wide = gated ? 1e30 : wide_us(groups, nsteps), join = splits[1] > 1 ? 6.0 : 0.0;
    if (wide * (splits[0] > 1 && groups <= 200 ? 1.1 : 1.0) < blocks[0] && wide + join + blocks[1] < std::min(mixed, tiles))
      return PackedKernel::kWide;
    if (tiles <= std::min(mixed, blocks[0] + blocks[1])) return PackedKernel::kTiles;
    return mixed <= blocks[0] + blocks[1] ? PackedKernel::kMixed : PackedKernel::kBlocks;
  }
};

}  // namespace gkr
