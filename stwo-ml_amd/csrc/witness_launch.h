// Launches of the witness products' kernels (witness.h), for any end of them:
// which kernel takes a product, in how many workgroups.
#pragma once
#include "gemm.h"
#include "internal.h"
#include "witness.h"
#include "witness_cost.h"

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
  // the block kernels' column groups, and what they take for rows of one plane and of four
  constexpr uint32_t NW = GATED ? 2 : 1;
  const bool general = w0->bnplanes > 1 || w1->bnplanes > 1;
  const uint64_t bgroups = (ctiles * NW * (general ? 4 : 1) + 7) / 8;
  const PackedCost cost(m, n, g.nsteps, GATED, general, quant != nullptr);
  // rows1: row tiles a workgroup has of rows of one plane that it streams the weights for; 0: blocks as for four
  auto launch_blocks = [&](auto kernel, uint32_t rows1) -> int {
    g.cgroups = (uint32_t)bgroups;
    TRY(plan(0, rows1 ? rows1 : 8, rows1 ? 1 : cost.splits[0]));
    TRY(plan(1, 8, cost.splits[1]));
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
    TRY(plan(1, 8, cost.splits[1]));
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
    if (GATED || tiles <= cost.blocks[0] + cost.blocks[1]) {
      TRY(GKR_WIT_TILES(1, 4, W, 1, 2));
    } else if constexpr (!GATED) {
      TRY(launch_blocks(k_wit_blocks<4, false, End>, 0));
    }
  } else if (m <= 8) TRY(GKR_WIT_TILES(1, 1, W, 1, 1));
  else if (m <= 16) TRY(GKR_WIT_TILES(1, 1, W, 1, 2));
  else if (m <= 32) TRY(GKR_WIT_TILES(1, 1, W, 1, 4));
  else if (m <= 64) TRY(GKR_WIT_TILES(2, 1, W, 1, 4));
  else {
    constexpr uint32_t RT = GATED ? 2 : 4, WR = GATED ? 2 : 1;  // k_wit_mixed: row tiles of a wave, waves down the rows
    switch (cost.kernel(m, n, g.nsteps, GATED, quant != nullptr)) {
      case PackedKernel::kTiles: TRY(GKR_WIT_TILES(2, 1, W, 1, 4)); break;
      case PackedKernel::kWide:
        if constexpr (!GATED) TRY(launch_wide(k_wit_wide<4, 3, End>, 4, 3));
        break;
      case PackedKernel::kBlocks: TRY(launch_blocks(k_wit_blocks<1, GATED, End>, 0)); break;
      case PackedKernel::kMixed:
        if (m <= 128) TRY(launch_blocks(k_wit_mixed<RT, WR, GATED, End>, RT * WR));
        else TRY(launch_blocks(k_wit_mixed<RT, 2 * WR, GATED, End>, 2 * RT * WR));
    }
  }
#undef GKR_WIT_TILES
  if (max_splits > 1) {
    auto join = k_wit_join<GATED, End>;
    GKR_LAUNCH(c, join, end_grid((m * n + 3) / 4), dim3(256), 0, g, end);
    TRY(check_launch(c));
  }
  return GKR_OK;
}
