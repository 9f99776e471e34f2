// Products of 8-bit integers with scales for each row and column (kernels in
// witness.h and scaled.h).
#include "witness_launch.h"
#include "scaled.h"

// The operands that both forms have, checked, and the end of the product.
static int scaled_end(gkr_ctx* c, const char* what, const gkr_matrix* a, const gkr_matrix* b, const gkr_matrix* col_scales,
                      uint32_t shift, uint32_t limit, const gkr_matrix* bias, const gkr_matrix* residual, gkr_matrix* pre,
                      gkr_matrix* out, ScaledEnd* e) {
  if (a->cols != b->rows)
    return fail(GKR_ERR_INVALID, "%s: A is %llux%llu, B is %llux%llu", what, (unsigned long long)a->rows,
                (unsigned long long)a->cols, (unsigned long long)b->rows, (unsigned long long)b->cols);
  const uint64_t m = a->rows, n = b->cols;
  if (m > 0xffffffffull) return fail(GKR_ERR_INVALID, "%s: %llu rows (at most 2^32 - 1)", what, (unsigned long long)m);
  TRY(check_shape(what, "the columns' scales", col_scales, 1, n));
  TRY(check_shape(what, "the bias", bias, 1, n));
  TRY(check_shape(what, "the residual", residual, m, n));
  TRY(check_shape(what, "pre", pre, m, n));
  TRY(check_shape(what, "the output", out, m, n));
  if (shift > 63) return fail(GKR_ERR_INVALID, "%s: a shift of %u bits (at most 63)", what, shift);
  if (limit > P / 2) return fail(GKR_ERR_INVALID, "%s: a limit of %u (at most 2^30 - 1)", what, limit);
  if (residual && (residual->ctx != c || !residual->dev))
    return fail(GKR_ERR_INVALID, "%s: a matrix belongs to another (or a destroyed) context", what);
  if (residual && ((residual->dev != out->dev && overlap(residual, out)) || (pre && overlap(residual, pre))))
    return fail(GKR_ERR_INVALID, "%s: the residual shares part of an output's memory", what);
  *e = ScaledEnd{};
  e->col_scales = col_scales ? col_scales->dev : nullptr;
  e->bias = bias ? bias->dev : nullptr;
  e->residual = residual ? residual->dev : nullptr;
  e->pre = pre ? pre->dev : nullptr;
  e->out = out->dev;
  e->shift = shift;
  e->limit = (int32_t)(limit ? limit : P / 2);
  e->last_row = (uint32_t)(m - 1);
  return GKR_OK;
}
// A product that neither kind of kernel takes: the forward product's passes,
// with the end in a launch behind.
static int long_product(gkr_ctx* c, const gkr_matrix* a, const gkr_matrix* b, const ScaledEnd& e) {
  const uint64_t m = a->rows, n = b->cols;
  uint32_t* z;
  TRY(ensureT(c, S_WITG, m * n, &z));
  TRY(matmul_forward(c, a, const_cast<gkr_matrix*>(b), z));
  auto end = k_wit_end<false, ScaledEnd>;
  GKR_LAUNCH(c, end, end_grid(m * n), dim3(256), 0, z, z, m * n, n, e);
  return check_launch(c);
}
static int scaled_product(gkr_ctx* c, const gkr_matrix* a, const gkr_matrix* b, const ScaledEnd& e) {
  const WitRows rows = wit_rows(a);
  if (few_rows(rows, b, b)) return rows_product<false>(c, rows, b, b, e);
  if (packable(a->rows, a->cols, b->cols)) return packed_product<false>(c, rows, b, b, e);
  return long_product(c, a, b, e);
}

static int scaled_forward(gkr_ctx* c, const gkr_matrix* a, const gkr_matrix* b, const gkr_matrix* row_scales,
                          const gkr_matrix* col_scales, uint32_t shift, uint32_t limit, const gkr_matrix* bias,
                          const gkr_matrix* residual, gkr_matrix* pre, gkr_matrix* out) {
  static const char what[] = "scaled product";
  if (!c || !a || !b || !out) return fail(GKR_ERR_INVALID, "null argument");
  TRY(check_operands(c, what, {a, b, row_scales, col_scales, bias}, {pre, out}));
  ScaledEnd e;
  TRY(scaled_end(c, what, a, b, col_scales, shift, limit, bias, residual, pre, out, &e));
  TRY(check_shape(what, "the rows' scales", row_scales, a->rows, 1));
  e.row_scales = row_scales ? row_scales->dev : nullptr;
  HIP_TRY(hipSetDevice(c->device));
  if (pre) TRY(drop_derived(c, pre));
  TRY(drop_output(c, out, residual));
  TRY(weight_planes(c, const_cast<gkr_matrix*>(b)));
  return scaled_product(c, a, b, e);
}

static int quantized_forward(gkr_ctx* c, const gkr_matrix* a, const gkr_matrix* b, uint32_t levels,
                             const gkr_matrix* col_scales, uint32_t shift, uint32_t limit, const gkr_matrix* bias,
                             const gkr_matrix* residual, gkr_matrix* quantized, gkr_matrix* row_scales, gkr_matrix* pre,
                             gkr_matrix* out) {
  static const char what[] = "quantized product";
  if (!c || !a || !b || !out) return fail(GKR_ERR_INVALID, "null argument");
  TRY(check_operands(c, what, {a, b, col_scales, bias}, {quantized, row_scales, pre, out}));
  if (levels == 0 || levels > 127) return fail(GKR_ERR_INVALID, "%s: %u levels (1 .. 127)", what, levels);
  ScaledEnd e;
  TRY(scaled_end(c, what, a, b, col_scales, shift, limit, bias, residual, pre, out, &e));
  const uint64_t m = a->rows, k = a->cols;
  TRY(check_shape(what, "the quantized rows", quantized, m, k));
  TRY(check_shape(what, "the rows' scales", row_scales, m, 1));
  for (gkr_matrix* w : {quantized, row_scales})
    if (residual && w && overlap(residual, w))
      return fail(GKR_ERR_INVALID, "%s: the residual shares part of an output's memory", what);
  HIP_TRY(hipSetDevice(c->device));
  for (gkr_matrix* w : {quantized, row_scales, pre})
    if (w) TRY(drop_derived(c, w));
  TRY(drop_output(c, out, residual));
  TRY(weight_planes(c, const_cast<gkr_matrix*>(b)));
  uint32_t* scales;
  if (row_scales) scales = row_scales->dev;
  else TRY(ensureT(c, S_QSCALE, m, &scales));
  const WitRows rows = wit_rows(a);
  const WitQuant quant{levels, quantized ? quantized->dev : nullptr, scales};
  if (quantized_rows_fit(rows, b)) return rows_product<false, true>(c, rows, b, b, e, quant);
  e.row_scales = scales;
  if (!few_rows(rows, b, b) && packable(m, k, b->cols)) return packed_product<false>(c, rows, b, b, e, &quant);
  gkr_matrix q{c, nullptr, m, k, false};
  if (quantized) q.dev = quantized->dev;
  else TRY(ensureT(c, S_QUANT, m * k, &q.dev));
  for (uint64_t row = 0; row < m; row += 1u << 21) {  // as many workgroups as one grid dimension holds
    const uint64_t some = std::min<uint64_t>(m - row, 1u << 21);
    GKR_LAUNCH(c, k_quantize_rows, dim3((uint32_t)some), dim3(1024), 0, a->dev + row * k, k, levels, q.dev + row * k,
               scales + row);
    TRY(check_launch(c));
  }
  return scaled_product(c, &q, b, e);
}

extern "C" int gkr_matmul_forward_scaled(gkr_ctx* c, const gkr_matrix* a, const gkr_matrix* b,
                                         const gkr_matrix* row_scales, const gkr_matrix* col_scales, uint32_t shift,
                                         uint32_t limit, const gkr_matrix* bias, const gkr_matrix* residual,
                                         gkr_matrix* pre, gkr_matrix* out) {
  return guarded([&] { return scaled_forward(c, a, b, row_scales, col_scales, shift, limit, bias, residual, pre, out); });
}
extern "C" int gkr_matmul_forward_quantized(gkr_ctx* c, const gkr_matrix* a, const gkr_matrix* b, uint32_t levels,
                                            const gkr_matrix* col_scales, uint32_t shift, uint32_t limit,
                                            const gkr_matrix* bias, const gkr_matrix* residual, gkr_matrix* quantized,
                                            gkr_matrix* row_scales, gkr_matrix* pre, gkr_matrix* out) {
  return guarded([&] {
    return quantized_forward(c, a, b, levels, col_scales, shift, limit, bias, residual, quantized, row_scales, pre, out);
  });
}
