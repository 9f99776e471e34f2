// Witness operators: the forward product with its epilogue, and the gated
// feed-forward block (kernels in witness.h).
#include "internal.h"
#include "activations.h"
#include "gemm.h"
#include "witness.h"

static bool overlap(const gkr_matrix* x, const gkr_matrix* y) {
  const uint32_t *x1 = x->dev + x->rows * x->cols, *y1 = y->dev + y->rows * y->cols;
  return x->dev < y1 && y->dev < x1;
}
// Every given matrix is alive on c, every output has rows x cols and shares
// no memory with an input or another output.
int check_operands(gkr_ctx* c, const char* what, std::initializer_list<const gkr_matrix*> ins,
                   std::initializer_list<const gkr_matrix*> outs) {
  for (auto& list : {ins, outs})
    for (const gkr_matrix* m : list)
      if (m && (m->ctx != c || !m->dev))
        return fail(GKR_ERR_INVALID, "%s: a matrix belongs to another (or a destroyed) context", what);
  for (auto o = outs.begin(); o != outs.end(); o++) {
    if (!*o) continue;
    for (const gkr_matrix* m : ins)
      if (m && overlap(m, *o)) return fail(GKR_ERR_INVALID, "%s: an output shares memory with an input", what);
    for (auto p = outs.begin(); p != o; p++)
      if (*p && overlap(*p, *o)) return fail(GKR_ERR_INVALID, "%s: two outputs share memory", what);
  }
  return GKR_OK;
}
int check_shape(const char* what, const char* name, const gkr_matrix* m, uint64_t rows, uint64_t cols) {
  if (m && (m->rows != rows || m->cols != cols))
    return fail(GKR_ERR_INVALID, "%s: %s is %llux%llu, not %llux%llu", what, name, (unsigned long long)m->rows,
                (unsigned long long)m->cols, (unsigned long long)rows, (unsigned long long)cols);
  return GKR_OK;
}
static int activation_arg(gkr_ctx* c, const char* what, uint32_t tag, uint32_t log_size, ActArg* arg) {
  *arg = ActArg{nullptr, 0, 0};
  if (tag == 0) return GKR_OK;
  if (!act_valid(tag)) return fail(GKR_ERR_INVALID, "%s: unknown activation type %u", what, tag);
  if (log_size > 24) return fail(GKR_ERR_INVALID, "%s: a table of 2^%u entries (at most 2^24)", what, log_size);
  if (tag == ACT_RELU) {
    arg->relu = 1;
    return GKR_OK;
  }
  if (log_size == 0) log_size = act_default_log_size(tag);
  uint32_t* table;
  TRY(device_table(c, tag, log_size, &table));
  arg->table = table;
  arg->mask = (1u << log_size) - 1;
  return GKR_OK;
}
static WitWeight wit_weight(const gkr_matrix* w) { return WitWeight{w->bplanes, (uint32_t)w->bnplanes}; }

static dim3 end_grid(uint64_t count) { return dim3((uint32_t)std::min<uint64_t>((count + 255) / 256, 1u << 20)); }
// Few rows (k_rows).
template <bool GATED, class End>
static int rows_product(gkr_ctx* c, const gkr_matrix* a, const gkr_matrix* w0, const gkr_matrix* w1, const End& end) {
  const uint32_t m = (uint32_t)a->rows, k = (uint32_t)a->cols;
  const uint64_t n = w0->cols, ctiles = (n + kGemmTile - 1) / kGemmTile;
  const bool one = w0->bnplanes == 1 && w1->bnplanes == 1;
  auto launch = [&](auto kernel, uint32_t mr, uint32_t waves) {
    const uint32_t lds = std::min<uint32_t>(kRowLds, 4 * mr * ((k + 63) / 64 * 64));
    GKR_LAUNCH(c, kernel, dim3((uint32_t)ctiles), dim3(64 * waves), lds, a->dev, wit_weight(w0), wit_weight(w1), m, k,
               (uint32_t)n, end);
  };
  const bool many = ctiles > 256;
  // two matrices of general weights: eight waves of twice the registers
#define GKR_ROWS(MR)                                                                \
  do {                                                                              \
    if (!one && (many || GATED)) launch(k_rows<MR, 4, GATED, 8, End>, MR, 8);       \
    else if (!one) launch(k_rows<MR, 4, GATED, GATED ? 8 : 16, End>, MR, 16);       \
    else if (many) launch(k_rows<MR, 1, GATED, 8, End>, MR, 8);                     \
    else launch(k_rows<MR, 1, GATED, 16, End>, MR, 16);                             \
  } while (0)
  if (m == 1) GKR_ROWS(1);
  else if (m == 2) GKR_ROWS(2);
  else if (m <= 4) GKR_ROWS(4);
  else if (m <= 8) many ? launch(k_rows<8, 1, GATED, 8, End>, 8, 8) : launch(k_rows<8, 1, GATED, 16, End>, 8, 16);
  else many ? launch(k_rows<16, 1, GATED, 8, End>, 16, 8) : launch(k_rows<16, 1, GATED, 16, End>, 16, 16);
#undef GKR_ROWS
  return check_launch(c);
}
static bool few_rows(const gkr_matrix* a, const gkr_matrix* w0, const gkr_matrix* w1) {
  return few_rows_fit(a->rows, a->cols, w0->cols, w0->bnplanes == 1 && w1->bnplanes == 1);
}

// Two masks of the packing, used in turn: the packing of one product clears the
// other's.  A mask that is set says that rows may have four planes, which is right
// for all rows: a captured product may find its own from the last replay.
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

// More rows: packed, multiplied (k_wit_tiles) and, where K is split, joined.
template <bool GATED, class End>
static int packed_product(gkr_ctx* c, const gkr_matrix* a, const gkr_matrix* w0, const gkr_matrix* w1, const End& end) {
  const uint64_t m = a->rows, k = a->cols, n = w0->cols;
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
  TRY(ensureT(c, S_GEMMA, (one_tiles + four_tiles) * g.nsteps * kGemmBlockBytes, &packed));
  g.one = packed;
  g.four = packed + one_tiles * g.nsteps * kGemmBlockBytes;
  uint32_t *mask, *next_mask;
  TRY(wit_masks(c, &mask, &next_mask));
  g.mask = mask;
  static_assert(kProductStep == kGemmK, "packable");
  const dim3 pack_grid((uint32_t)pack_groups(m, k));
  GKR_LAUNCH(c, k_wit_pack, pack_grid, dim3(kPackThreads), 0, a->dev, m, k, g.nsteps, packed,
             const_cast<int8_t*>(g.four), mask, next_mask);
  TRY(check_launch(c));

  uint32_t max_splits = 1, max_rgroups = 1;
  // group: row tiles of a workgroup, for rows of one plane and of four
  auto plan = [&](int four, uint32_t group, uint32_t splits) -> int {
    const uint64_t tiles = four ? four_tiles : one_tiles;
    WitPlan& p = g.plan[four];
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
                            blocks_us((four_tiles + 7) / 8 * bgroups, g.nsteps, elements, &splits[1])};
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
#define GKR_WIT_TILES(RT, PB, W, WR1, WR4) launch_tiles(k_wit_tiles<RT, PB, GATED, W, WR1, WR4, End>, RT, W, WR1, WR4)
  // sixteen waves a workgroup for one matrix, eight for two: the registers of
  // sixteen hold no more accumulators
  constexpr int W = GATED ? 8 : 16;
  if (general) {
    const double tiles = tiles_us(one_tiles * ctiles, 256, g.nsteps, 1 + 4 * NW) +
                         tiles_us((four_tiles + 1) / 2 * ctiles, 256, g.nsteps, 2 * (1 + 4 * NW));
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
    const double tiles = tiles_us(rows64 * ctiles, 512, g.nsteps, 2 + NW) + tiles_us(rows64 * ctiles, 512, g.nsteps, 4 * (2 + NW));
    constexpr uint32_t RT = GATED ? 2 : 4, WR = GATED ? 2 : 1;
    const uint32_t down = m <= 128 ? WR : 2 * WR;  // waves down the rows of k_wit_mixed
    const double mixed = m <= 256 ? tiles_us(ctiles, 256, g.nsteps, down * (RT + NW)) + blocks[1] : 1e30;
    if (tiles <= std::min(mixed, blocks[0] + blocks[1])) TRY(GKR_WIT_TILES(2, 1, W, 1, 4));
    else if (mixed > blocks[0] + blocks[1]) TRY(launch_blocks(k_wit_blocks<1, GATED, End>, 0));
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

static int fused_forward(gkr_ctx* c, const gkr_matrix* a, const gkr_matrix* b, const gkr_matrix* bias, uint32_t tag,
                         uint32_t table_log, const gkr_matrix* residual, gkr_matrix* pre, gkr_matrix* out) {
  static const char what[] = "fused product";
  if (!c || !a || !b || !out) return fail(GKR_ERR_INVALID, "null argument");
  TRY(check_operands(c, what, {a, b, bias}, {pre, out}));
  if (a->cols != b->rows)
    return fail(GKR_ERR_INVALID, "%s: A is %llux%llu, B is %llux%llu", what, (unsigned long long)a->rows,
                (unsigned long long)a->cols, (unsigned long long)b->rows, (unsigned long long)b->cols);
  const uint64_t m = a->rows, n = b->cols;
  TRY(check_shape(what, "the bias", bias, 1, n));
  TRY(check_shape(what, "the residual", residual, m, n));
  TRY(check_shape(what, "pre", pre, m, n));
  TRY(check_shape(what, "the output", out, m, n));
  if (residual && (residual->ctx != c || !residual->dev))
    return fail(GKR_ERR_INVALID, "%s: a matrix belongs to another (or a destroyed) context", what);
  if (residual && ((residual->dev != out->dev && overlap(residual, out)) || (pre && overlap(residual, pre))))
    return fail(GKR_ERR_INVALID, "%s: the residual shares part of an output's memory", what);
  HIP_TRY(hipSetDevice(c->device));
  FusedEnd e{};
  TRY(activation_arg(c, what, tag, table_log, &e.act));
  e.bias = bias ? bias->dev : nullptr;
  e.residual = residual ? residual->dev : nullptr;
  e.pre = pre ? pre->dev : nullptr;
  e.out = out->dev;
  TRY(drop_derived(c, out));
  if (pre) TRY(drop_derived(c, pre));
  TRY(weight_planes(c, const_cast<gkr_matrix*>(b)));
  if (few_rows(a, b, b)) return rows_product<false>(c, a, b, b, e);
  if (packable(m, a->cols, n)) return packed_product<false>(c, a, b, b, e);
  uint32_t* z;
  TRY(ensureT(c, S_WITG, m * n, &z));
  TRY(matmul_forward(c, a, const_cast<gkr_matrix*>(b), z));
  auto end = k_wit_end<false, FusedEnd>;
  GKR_LAUNCH(c, end, end_grid(m * n), dim3(256), 0, z, z, m * n, n, e);
  return check_launch(c);
}

static int gated_forward(gkr_ctx* c, const gkr_matrix* a, const gkr_matrix* wg, const gkr_matrix* wu, uint32_t tag,
                         uint32_t table_log, gkr_matrix* gate, gkr_matrix* act, gkr_matrix* up, gkr_matrix* out) {
  static const char what[] = "gated block";
  if (!c || !a || !wg || !wu || !out) return fail(GKR_ERR_INVALID, "null argument");
  TRY(check_operands(c, what, {a, wg, wu}, {gate, act, up, out}));
  if (a->cols != wg->rows || wg->rows != wu->rows || wg->cols != wu->cols)
    return fail(GKR_ERR_INVALID, "%s: A is %llux%llu, the weights %llux%llu and %llux%llu", what,
                (unsigned long long)a->rows, (unsigned long long)a->cols, (unsigned long long)wg->rows,
                (unsigned long long)wg->cols, (unsigned long long)wu->rows, (unsigned long long)wu->cols);
  const uint64_t m = a->rows, n = wg->cols;
  TRY(check_shape(what, "gate", gate, m, n));
  TRY(check_shape(what, "act", act, m, n));
  TRY(check_shape(what, "up", up, m, n));
  TRY(check_shape(what, "the output", out, m, n));
  HIP_TRY(hipSetDevice(c->device));
  GatedEnd e{};
  TRY(activation_arg(c, what, tag, table_log, &e.act));
  e.gate = gate ? gate->dev : nullptr;
  e.act_out = act ? act->dev : nullptr;
  e.up = up ? up->dev : nullptr;
  e.out = out->dev;
  for (gkr_matrix* w : {gate, act, up, out})
    if (w) TRY(drop_derived(c, w));
  TRY(weight_planes(c, const_cast<gkr_matrix*>(wg)));
  TRY(weight_planes(c, const_cast<gkr_matrix*>(wu)));
  if (few_rows(a, wg, wu)) return rows_product<true>(c, a, wg, wu, e);
  if (packable(m, a->cols, n)) return packed_product<true>(c, a, wg, wu, e);
  uint32_t *g, *u;
  TRY(ensureT(c, S_WITG, m * n, &g));
  TRY(ensureT(c, S_WITU, m * n, &u));
  TRY(matmul_forward(c, a, const_cast<gkr_matrix*>(wg), g));
  TRY(matmul_forward(c, a, const_cast<gkr_matrix*>(wu), u));
  auto end = k_wit_end<true, GatedEnd>;
  GKR_LAUNCH(c, end, end_grid(m * n), dim3(256), 0, g, u, m * n, n, e);
  return check_launch(c);
}

extern "C" int gkr_matmul_forward_fused(gkr_ctx* c, const gkr_matrix* a, const gkr_matrix* b, const gkr_matrix* bias,
                                        uint32_t tag, uint32_t table_log, const gkr_matrix* residual, gkr_matrix* pre,
                                        gkr_matrix* out) {
  return guarded([&] { return fused_forward(c, a, b, bias, tag, table_log, residual, pre, out); });
}
extern "C" int gkr_gated_forward(gkr_ctx* c, const gkr_matrix* a, const gkr_matrix* wg, const gkr_matrix* wu,
                                 uint32_t tag, uint32_t table_log, gkr_matrix* gate, gkr_matrix* act, gkr_matrix* up,
                                 gkr_matrix* out) {
  return guarded([&] { return gated_forward(c, a, wg, wu, tag, table_log, gate, act, up, out); });
}
