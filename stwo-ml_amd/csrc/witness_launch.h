// Launches of the witness products' kernels (witness.h), for any end of them:
// which kernel takes a product, in how many workgroups.
#pragma once
#include "gemm.h"
#include "internal.h"
#include "witness.h"

// The m x k words that the weights are multiplied by.
struct WitRows {
  const uint32_t* x;
  uint64_t m, k;
};
inline WitRows wit_rows(const gkr_matrix* a) { return WitRows{a->dev, a->rows, a->cols}; }
inline bool overlap(const gkr_matrix* x, const gkr_matrix* y) {
  const uint32_t *x1 = x->dev + x->rows * x->cols, *y1 = y->dev + y->rows * y->cols;
  return x->dev < y1 && y->dev < x1;
}
// The contents of an output change; a residual may be the same memory by another
// handle, whose derived copies go too.
inline int drop_output(gkr_ctx* c, gkr_matrix* out, const gkr_matrix* residual) {
  if (residual && residual != out && residual->dev == out->dev) TRY(drop_derived(c, const_cast<gkr_matrix*>(residual)));
  return drop_derived(c, out);
}
static WitWeight wit_weight(const gkr_matrix* w) { return WitWeight{w->bplanes, (uint32_t)w->bnplanes}; }

static dim3 end_grid(uint64_t count) { return dim3((uint32_t)std::min<uint64_t>((count + 255) / 256, 1u << 20)); }
// Few rows (k_rows); with QUANT they are quantized_rows_fit.
template <bool GATED, bool QUANT = false, class End>
static int rows_product(gkr_ctx* c, const WitRows& a, const gkr_matrix* w0, const gkr_matrix* w1, const End& end,
                        const WitQuant& quant = {}) {
  const uint32_t m = (uint32_t)a.m, k = (uint32_t)a.k;
  const uint64_t n = w0->cols, ctiles = (n + kGemmTile - 1) / kGemmTile;
  const bool one = w0->bnplanes == 1 && w1->bnplanes == 1;
  auto launch = [&](auto kernel, uint32_t mr, uint32_t waves) {
    const uint32_t lds = std::min<uint32_t>(kRowLds, 4 * mr * ((k + 63) / 64 * 64));
    GKR_LAUNCH(c, kernel, dim3((uint32_t)ctiles), dim3(64 * waves), lds, a.x, wit_weight(w0), wit_weight(w1), m, k,
               (uint32_t)n, end, quant);
  };
  const bool many = ctiles > 256;
  // two matrices of general weights: eight waves of twice the registers
#define GKR_ROWS_ONE(MR) \
  (many ? launch(k_rows<MR, 1, GATED, 8, QUANT, End>, MR, 8) : launch(k_rows<MR, 1, GATED, 16, QUANT, End>, MR, 16))
#define GKR_ROWS(MR)                                                                                     \
  do {                                                                                                   \
    if constexpr (QUANT) GKR_ROWS_ONE(MR);                                                               \
    else if (one) GKR_ROWS_ONE(MR);                                                                      \
    else if (many || GATED) launch(k_rows<MR, 4, GATED, 8, QUANT, End>, MR, 8);                          \
    else launch(k_rows<MR, 4, GATED, GATED ? 8 : 16, QUANT, End>, MR, 16);                               \
  } while (0)
  if (m == 1) GKR_ROWS(1);
  else if (m == 2) GKR_ROWS(2);
  else if (m <= 4) GKR_ROWS(4);
  else if (m <= 8) GKR_ROWS_ONE(8);
  else GKR_ROWS_ONE(16);
#undef GKR_ROWS_ONE
#undef GKR_ROWS
  return check_launch(c);
}
static bool few_rows(const WitRows& a, const gkr_matrix* w0, const gkr_matrix* w1) {
  return few_rows_fit(a.m, a.k, w0->cols, w0->bnplanes == 1 && w1->bnplanes == 1);
}

static bool quantized_rows_fit(const WitRows& a, const gkr_matrix* w) {
  const uint64_t mr = a.m == 1 ? 1 : a.m == 2 ? 2 : a.m <= 4 ? 4 : a.m <= 8 ? 8 : 16;
  static_assert(4 * kQuantFew <= kRowLds, "one fill");
  return w->bnplanes == 1 && few_rows(a, w, w) && mr * ((a.k + 63) / 64 * 64) <= kQuantFew;
}

// Two masks of the packing, used in turn: the packing of one product clears the
// other's.  A mask that is set says that rows may have four planes, which is right
// for all rows: a captured product may find its own from the last replay.  A prompt
// zeroes its own too (k_prompt), as there the kernel of general words costs more.
static int wit_masks(gkr_ctx* c, uint32_t** mask, uint32_t** next_mask) {
  constexpr uint32_t words = kMaskWords * kMaskStride;
  if (!c->wit_mask) {
    drain(c);
    uint32_t* w = nullptr;
    HIP_TRY(hipMalloc(&w, 2 * words * sizeof(uint32_t)));
    c->wit_mask = w;
    const uint64_t count = 2 * words * sizeof(uint32_t) / 16;
    GKR_LAUNCH(c, k_extend, extend_grid(count), dim3(256), 0, nullptr, 0, (uint4*)w, count);
    TRY(check_launch(c));
  }
  *mask = c->wit_mask + (c->wit_turn & 1) * words;
  *next_mask = c->wit_mask + (~c->wit_turn & 1) * words;
  c->wit_turn++;
  return GKR_OK;
}

// What the two kinds of kernel take, in us, to choose between them; fitted to 27
// products of 40 to 512 rows, k 100 to 13824, n 900 to 13824, rows and weights
// of one plane and of four, which each kind took 10 to 330 us for: within a
// quarter, and the better one taken in all but two (by 1.1 and 1.2 times).
// k_wit_tiles: 8 us for each round of the workgroups that fit at once (`slots`),
// and the operands' way from the second-level cache, 17 GB/ms; kb is a
// workgroup's K step.
static double tiles_us(uint64_t groups, uint32_t slots, uint32_t nsteps, uint32_t kb) {
  return 8.0 * (double)((groups + slots - 1) / slots) + (double)groups * nsteps * kb / 17000.0;
}
// k_wit_blocks: a workgroup fills a CU; a K step takes it 0.27 us where few run
// and 0.5 on all 256 (the matrix cores slow down).  K splits fill the last
// round, against the parts' way through memory and a launch to join them.
static double blocks_us(uint64_t groups, uint32_t nsteps, uint64_t elements, uint32_t* splits) {
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
static double wide_us(uint64_t groups, uint32_t nsteps) {
  return groups > 512 ? 1e30 : 1.25 * (2.0 + (double)((groups + 255) / 256) * (9.0 + 0.09 * nsteps));
}

// More rows: packed, multiplied (k_wit_tiles) and, where K is split, joined.  With
// `quant` they are brought to 8 bits as they are packed, and have one plane.
template <bool GATED, class End>
static int packed_product(gkr_ctx* c, const WitRows& a, const gkr_matrix* w0, const gkr_matrix* w1, const End& end,
                          const WitQuant* quant = nullptr) {
  const uint64_t m = a.m, k = a.k, n = w0->cols;
  WitProduct g{};
  g.m = m;
  g.n = n;
  g.nsteps = (uint32_t)((k + kGemmK - 1) / kGemmK);
  const uint64_t ctiles = (n + kGemmTile - 1) / kGemmTile;
  g.ctiles = (uint32_t)ctiles;
  g.w[0] = wit_weight(w0);
  g.w[1] = wit_weight(w1);
  const uint64_t one_tiles = (m + 31) / 32, four_tiles = (m + 7) / 8;
  int8_t* packed;
  TRY(ensureT(c, S_GEMMA, (one_tiles + (quant ? 0 : four_tiles)) * g.nsteps * kGemmBlockBytes, &packed));
  g.one = packed;
  g.four = packed + one_tiles * g.nsteps * kGemmBlockBytes;
  uint32_t *mask, *next_mask;
  TRY(wit_masks(c, &mask, &next_mask));
  g.mask = mask;
  static_assert(kProductStep == kGemmK, "packable");
  if (quant) {
    GKR_LAUNCH(c, k_wit_quantize, dim3((uint32_t)((m + kQuantRows - 1) / kQuantRows)), dim3(256 * kQuantRows), 0, a.x, m, k,
               g.nsteps, packed, *quant, mask, next_mask);
  } else {
    const dim3 pack_grid((uint32_t)pack_groups(m, k));
    GKR_LAUNCH(c, k_wit_pack, pack_grid, dim3(kPackThreads), 0, a.x, m, k, g.nsteps, packed,
               const_cast<int8_t*>(g.four), mask, next_mask);
  }
  TRY(check_launch(c));

  uint32_t max_splits = 1, max_rgroups = 1;
  // group: row tiles of a workgroup, for rows of one plane and of four
  auto plan = [&](int four, uint32_t group, uint32_t splits) -> int {
    WitPlan& p = g.plan[four];
    if (four && quant) {  // there are none; a mask that is set all the same (a refused packing) finds nothing to do
      p = WitPlan{1, 1, 0, 0};
      return GKR_OK;
    }
    const uint64_t tiles = four ? four_tiles : one_tiles;
    p.rtiles = (uint32_t)tiles;
    p.rgroups = (uint32_t)((tiles + group - 1) / group);
    p.splits = splits;
    p.steps = (g.nsteps + p.splits - 1) / p.splits;
    p.splits = (g.nsteps + p.steps - 1) / p.steps;
    max_splits = std::max(max_splits, p.splits);
    max_rgroups = std::max(max_rgroups, p.rgroups);
    if (p.splits > 1) TRY(ensureT(c, S_GEMMP, (uint64_t)max_splits * (GATED ? 2 : 1) * m * n, &g.part));
    return GKR_OK;
  };
  auto launch_tiles = [&](auto kernel, uint32_t rt, uint32_t waves, uint32_t wr1, uint32_t wr4) -> int {
    g.cgroups = g.ctiles;
    TRY(plan(0, rt * wr1, 1));
    TRY(plan(1, rt * wr4, 1));
    uint32_t rg;
    const dim3 grid = gemm_group_grid(max_rgroups, g.cgroups, 1, &rg, kGemmMaxGroups / 4);
    GKR_LAUNCH(c, kernel, grid, dim3(64 * waves), 0, g, rg, end);
    return check_launch(c);
  };
  // the block kernels' column groups, and what they take (splits[]) for rows of one plane and of four
  constexpr uint32_t NW = GATED ? 2 : 1;
  const bool general = w0->bnplanes > 1 || w1->bnplanes > 1;
  const uint64_t bgroups = (ctiles * NW * (general ? 4 : 1) + 7) / 8, elements = m * n * NW;
  uint32_t splits[2] = {1, 1};
  const double blocks[2] = {blocks_us((one_tiles + 7) / 8 * bgroups, g.nsteps, elements, &splits[0]),
                            quant ? 0 : blocks_us((four_tiles + 7) / 8 * bgroups, g.nsteps, elements, &splits[1])};
  // rows1: row tiles a workgroup has of rows of one plane that it streams the weights for; 0: blocks as for four
  auto launch_blocks = [&](auto kernel, uint32_t rows1) -> int {
    g.cgroups = (uint32_t)bgroups;
    TRY(plan(0, rows1 ? rows1 : 8, rows1 ? 1 : splits[0]));
    TRY(plan(1, 8, splits[1]));
    uint64_t grid = 0;
    for (int i = 0; i < 2; i++) {
      const uint64_t groups = (uint64_t)g.plan[i].rgroups * (i == 0 && rows1 ? g.ctiles : g.cgroups);
      grid = std::max(grid, (groups + 7) / 8 * 8 * g.plan[i].splits);
    }
    GKR_LAUNCH(c, kernel, dim3((uint32_t)grid), dim3(512), 0, g, end);
    return check_launch(c);
  };
  auto launch_wide = [&](auto kernel, uint32_t rt, uint32_t ct) -> int {
    g.cgroups = (uint32_t)bgroups;
    TRY(plan(0, rt, 1));
    TRY(plan(1, 8, splits[1]));
    const uint64_t wide = (uint64_t)g.plan[0].rgroups * ((g.ctiles + ct - 1) / ct);
    const uint64_t other = ((uint64_t)g.plan[1].rgroups * g.cgroups + 7) / 8 * 8 * g.plan[1].splits;
    GKR_LAUNCH(c, kernel, dim3((uint32_t)std::max((wide + 7) / 8 * 8, other)), dim3(512), 0, g, end);
    return check_launch(c);
  };
#define GKR_WIT_TILES(RT, PB, W, WR1, WR4) launch_tiles(k_wit_tiles<RT, PB, GATED, W, WR1, WR4, End>, RT, W, WR1, WR4)
  // sixteen waves a workgroup for one matrix, eight for two: the registers of
  // sixteen hold no more accumulators
  constexpr int W = GATED ? 8 : 16;
  if (general) {
    const double tiles = tiles_us(one_tiles * ctiles, 256, g.nsteps, 1 + 4 * NW) +
                         (quant ? 0 : tiles_us((four_tiles + 1) / 2 * ctiles, 256, g.nsteps, 2 * (1 + 4 * NW)));
    if (GATED || tiles <= blocks[0] + blocks[1]) {
      TRY(GKR_WIT_TILES(1, 4, W, 1, 2));
    } else if constexpr (!GATED) {
      TRY(launch_blocks(k_wit_blocks<4, false, End>, 0));
    }
  } else if (m <= 8) TRY(GKR_WIT_TILES(1, 1, W, 1, 1));
  else if (m <= 16) TRY(GKR_WIT_TILES(1, 1, W, 1, 2));
  else if (m <= 32) TRY(GKR_WIT_TILES(1, 1, W, 1, 4));
  else if (m <= 64) TRY(GKR_WIT_TILES(2, 1, W, 1, 4));
  else {
    const uint64_t rows64 = (m + 63) / 64;
    const double tiles = tiles_us(rows64 * ctiles, 512, g.nsteps, 2 + NW) +
                         (quant ? 0 : tiles_us(rows64 * ctiles, 512, g.nsteps, 4 * (2 + NW)));
    constexpr uint32_t RT = GATED ? 2 : 4, WR = GATED ? 2 : 1;
    const uint32_t down = m <= 128 ? WR : 2 * WR;  // waves down the rows of k_wit_mixed
    const double mixed = m <= 256 ? tiles_us(ctiles, 256, g.nsteps, down * (RT + NW)) + blocks[1] : 1e30;
    const double wide = GATED ? 1e30 : wide_us((m + 127) / 128 * ((ctiles + 2) / 3), g.nsteps);
    const double most = std::min(wide, blocks[0]) + blocks[1];
    if (tiles <= std::min(mixed, most)) TRY(GKR_WIT_TILES(2, 1, W, 1, 4));
    else if (mixed > most && wide < blocks[0]) {
      if constexpr (!GATED) TRY(launch_wide(k_wit_wide<4, 3, End>, 4, 3));
    } else if (mixed > most) TRY(launch_blocks(k_wit_blocks<1, GATED, End>, 0));
    else if (m <= 128) TRY(launch_blocks(k_wit_mixed<RT, WR, GATED, End>, RT * WR));
    else TRY(launch_blocks(k_wit_mixed<RT, 2 * WR, GATED, End>, 2 * RT * WR));
  }
#undef GKR_WIT_TILES
  if (max_splits > 1) {
    auto join = k_wit_join<GATED, End>;
    GKR_LAUNCH(c, join, end_grid((m * n + 3) / 4), dim3(256), 0, g, end);
    TRY(check_launch(c));
  }
  return GKR_OK;
}
