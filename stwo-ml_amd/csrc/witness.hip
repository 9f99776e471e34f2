// Witness operators: the forward product with its epilogue, and the gated
// feed-forward block (kernels in witness.h).
#include "internal.h"
#include "activations.h"
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
  uint32_t *g, *u;
  TRY(ensureT(c, S_WITG, m * n, &g));
  TRY(ensureT(c, S_WITU, m * n, &u));
  TRY(matmul_forward(c, a, const_cast<gkr_matrix*>(wg), g));
  TRY(matmul_forward(c, a, const_cast<gkr_matrix*>(wu), u));
  GKR_LAUNCH(c, k_gated_end, end_grid(m * n), dim3(256), 0, g, u, m * n, e);
  return check_launch(c);
}
