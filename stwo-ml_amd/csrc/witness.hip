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
// Longest inner size of the kernels here: a digit sum stays below 2^31.
// Beyond it (no model's layer) the forward product's passes of K are used,
// with the element-wise work in a launch behind.
constexpr uint64_t kMaxInner = 131071;

static WitWeight wit_weight(const gkr_matrix* w) { return WitWeight{w->bplanes, (uint32_t)w->bnplanes}; }

// One to four rows (k_rows).
template <bool GATED, class End>
static int rows_product(gkr_ctx* c, const gkr_matrix* a, const gkr_matrix* w0, const gkr_matrix* w1, const End& end) {
  const uint32_t m = (uint32_t)a->rows, k = (uint32_t)a->cols;
  const uint64_t n = w0->cols, ctiles = (n + kGemmTile - 1) / kGemmTile;
  const bool one = w0->bnplanes == 1 && w1->bnplanes == 1;
  auto launch = [&](auto kernel, uint32_t mr) {
    const uint32_t lds = std::min<uint32_t>(kRowLds, 4 * mr * ((k + 63) / 64 * 64));
    GKR_LAUNCH(c, kernel, dim3((uint32_t)ctiles), dim3(64 * kRowWaves), lds, a->dev, wit_weight(w0), wit_weight(w1), m, k,
               (uint32_t)n, end);
  };
  if (m == 1) one ? launch(k_rows<1, 1, GATED, End>, 1) : launch(k_rows<1, 4, GATED, End>, 1);
  else if (m == 2) one ? launch(k_rows<2, 1, GATED, End>, 2) : launch(k_rows<2, 4, GATED, End>, 2);
  else one ? launch(k_rows<4, 1, GATED, End>, 4) : launch(k_rows<4, 4, GATED, End>, 4);
  return check_launch(c);
}
// A grid of kernels with 1024 threads takes this many column tiles.
constexpr uint64_t kRowMaxTiles = 1ull << 21;
static bool few_rows(uint64_t m, uint64_t k, uint64_t n) {
  return m <= 4 && k <= kMaxInner && n <= kRowMaxTiles * kGemmTile;
}

static dim3 end_grid(uint64_t count) { return dim3((uint32_t)std::min<uint64_t>((count + 255) / 256, 1u << 20)); }

extern "C" int gkr_matmul_forward_fused(gkr_ctx* c, const gkr_matrix* a, const gkr_matrix* b, const gkr_matrix* bias,
                                        uint32_t tag, uint32_t table_log, const gkr_matrix* residual, gkr_matrix* pre,
                                        gkr_matrix* out) {
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
  if (few_rows(m, a->cols, n)) return rows_product<false>(c, a, b, b, e);
  uint32_t* z;
  TRY(ensureT(c, S_WITG, m * n, &z));
  TRY(matmul_forward(c, a, const_cast<gkr_matrix*>(b), z));
  GKR_LAUNCH(c, k_fused_end, end_grid(m * n), dim3(256), 0, z, m * n, n, e);
  return check_launch(c);
}

extern "C" int gkr_gated_forward(gkr_ctx* c, const gkr_matrix* a, const gkr_matrix* wg, const gkr_matrix* wu,
                                 uint32_t tag, uint32_t table_log, gkr_matrix* gate, gkr_matrix* act, gkr_matrix* up,
                                 gkr_matrix* out) {
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
  if (few_rows(m, a->cols, n)) return rows_product<true>(c, a, wg, wu, e);
  uint32_t *g, *u;
  TRY(ensureT(c, S_WITG, m * n, &g));
  TRY(ensureT(c, S_WITU, m * n, &u));
  TRY(matmul_forward(c, a, const_cast<gkr_matrix*>(wg), g));
  TRY(matmul_forward(c, a, const_cast<gkr_matrix*>(wu), u));
  GKR_LAUNCH(c, k_gated_end, end_grid(m * n), dim3(256), 0, g, u, m * n, e);
  return check_launch(c);
}
