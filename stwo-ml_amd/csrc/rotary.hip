// Rotary positions (kernels in rotary.h).
#include <math.h>

#include "internal.h"
#include "rotary.h"

struct gkr_rotary {
  gkr_ctx* ctx;
  int2* table = nullptr;  // [position][pair]
  uint32_t pairs = 0, shift = 0, positions = 0;
};
void release_rotary(gkr_rotary* r) {
  if (r->table) (void)hipFree(r->table);
  r->table = nullptr;
  r->ctx = nullptr;
}

extern "C" int gkr_rotary_frequencies(uint32_t turned, double base, const gkr_rotary_scaling* scaling, uint64_t* out) {
  if (!out) return fail(GKR_ERR_INVALID, "null argument");
  if (turned == 0 || turned % 2 || turned > 65536)
    return fail(GKR_ERR_INVALID, "rotary frequencies: %u turned dims (an even number up to 65536)", turned);
  if (!(base > 0) || !isfinite(base)) return fail(GKR_ERR_INVALID, "rotary frequencies: a base of %g", base);
  gkr_rotary_scaling s{};
  if (scaling) s = *scaling;
  if (s.kind > GKR_ROTARY_WAVES) return fail(GKR_ERR_INVALID, "rotary frequencies: unknown scaling %u", s.kind);
  if (s.kind != GKR_ROTARY_PLAIN && (!(s.factor > 0) || !isfinite(s.factor)))
    return fail(GKR_ERR_INVALID, "rotary frequencies: a factor of %g", s.factor);
  if (s.kind == GKR_ROTARY_WAVES && (!(s.positions > 0) || !isfinite(s.positions) || !(s.low >= 0) ||
                                     !(s.high > s.low) || !isfinite(s.high)))
    return fail(GKR_ERR_INVALID, "rotary frequencies: %g positions, waves between %g and %g", s.positions, s.low, s.high);
  if (s.kind == GKR_ROTARY_BASE && turned > 2) base *= pow(s.factor, turned / (turned - 2.0));
  if (!(base > 0) || !isfinite(base))
    return fail(GKR_ERR_INVALID, "rotary frequencies: a base changed by a factor of %g to %g", s.factor, base);
  for (uint32_t i = 0; i < turned / 2; i++) {
    double f = pow(base, -2.0 * i / turned) / 6.283185307179586476925;  // turns a position
    if (s.kind == GKR_ROTARY_LINEAR) f /= s.factor;
    if (s.kind == GKR_ROTARY_WAVES) {
      const double keep = fmin(fmax((s.positions * f - s.low) / (s.high - s.low), 0.0), 1.0);
      f *= keep + (1 - keep) / s.factor;
    }
    if (!isfinite(f)) return fail(GKR_ERR_INVALID, "rotary frequencies: a base of %g and a factor of %g", base, s.factor);
    f -= floor(f);  // whole turns are none
    out[i] = f < 1 ? (uint64_t)(f * 18446744073709551616.0) : 0;
  }
  return GKR_OK;
}

extern "C" int gkr_rotary_new(gkr_ctx* c, const uint64_t* freqs, uint32_t turned, uint32_t amplitude, uint32_t shift,
                              uint32_t positions, gkr_rotary** out) {
  if (!c || !freqs || !out) return fail(GKR_ERR_INVALID, "null argument");
  if (turned == 0 || turned % 2 || turned > 65536)
    return fail(GKR_ERR_INVALID, "rotary positions: %u turned dims (an even number up to 65536)", turned);
  if (amplitude == 0 || amplitude > 1u << 30 || shift > 30)
    return fail(GKR_ERR_INVALID, "rotary positions: an amplitude of %u and a shift of %u (1 .. 2^30, at most 30)", amplitude, shift);
  if (positions == 0 || positions > 1u << 31)
    return fail(GKR_ERR_INVALID, "rotary positions: %u positions (1 .. 2^31)", positions);
  HIP_TRY(hipSetDevice(c->device));
  const uint32_t pairs = turned / 2;
  const uint64_t count = (uint64_t)positions * pairs;
  gkr_rotary* r = nullptr;
  const int rc = guarded([&]() -> int {
    r = new gkr_rotary{c};
    r->pairs = pairs;
    r->shift = shift;
    r->positions = positions;
    c->rotaries.insert(r);
    return GKR_OK;
  });
  if (rc != GKR_OK) {
    delete r;
    return rc;
  }
  drain(c);
  uint64_t* f = nullptr;
  auto failed = [&](int code, const char* what, hipError_t e) {
    (void)hipGetLastError();
    if (f) (void)hipFree(f);
    gkr_rotary_free(r);
    return fail(code, "rotary positions: %s: %s", what, hipGetErrorString(e));
  };
  hipError_t e = hipMalloc(&r->table, count * sizeof(int2));
  if (e != hipSuccess) {
    r->table = nullptr;
    return failed(GKR_ERR_NOMEM, "the table", e);
  }
  e = hipMalloc(&f, pairs * sizeof(uint64_t));
  if (e != hipSuccess) {
    f = nullptr;
    return failed(GKR_ERR_NOMEM, "the frequencies", e);
  }
  e = hipMemcpyAsync(f, freqs, pairs * sizeof(uint64_t), hipMemcpyHostToDevice, c->stream);
  if (e != hipSuccess) return failed(GKR_ERR_DEVICE, "the frequencies", e);
  GKR_LAUNCH(c, k_turns, dim3((uint32_t)std::min<uint64_t>((count + 255) / 256, 1u << 16)), dim3(256), 0, f, pairs, count,
             (double)amplitude, r->table);
  int made = check_launch(c);
  if (made == GKR_OK) made = sync(c);
  (void)hipFree(f);
  if (made != GKR_OK) {
    gkr_rotary_free(r);
    return made;
  }
  *out = r;
  return GKR_OK;
}
extern "C" void gkr_rotary_free(gkr_rotary* r) {
  if (!r) return;
  if (r->ctx) {
    drain(r->ctx);
    (void)hipStreamSynchronize(r->ctx->stream);
    r->ctx->rotaries.erase(r);
    release_rotary(r);
  }
  delete r;
}

static int rotary_forward(gkr_ctx* c, const gkr_rotary* r, uint32_t head_dim, int interleaved, const uint32_t* starts,
                          const uint32_t* counts, size_t n, uint32_t limit, const gkr_matrix* q, gkr_matrix* q_out,
                          const gkr_matrix* k, gkr_matrix* k_out) {
  static const char what[] = "rotary positions";
  if (!c || !r || !q || !q_out || (n && !counts) || !k != !k_out) return fail(GKR_ERR_INVALID, "null argument");
  if (r->ctx != c) return fail(GKR_ERR_INVALID, "%s of another (or a destroyed) context", what);
  // an output may be its own input's memory, and shares none else
  auto apart = [](const gkr_matrix* in, const gkr_matrix* o) { return in && in->dev != o->dev ? in : nullptr; };
  TRY(check_operands(c, what, {q, k}, {}));
  TRY(check_operands(c, what, {apart(q, q_out), k}, {q_out}));
  if (k) TRY(check_operands(c, what, {q, apart(k, k_out)}, {k_out}));
  if (k) TRY(check_operands(c, what, {}, {q_out, k_out}));
  if (head_dim == 0 || head_dim > 1u << 20 || 2 * r->pairs > head_dim)
    return fail(GKR_ERR_INVALID, "%s: %u turned dims of heads of %u", what, 2 * r->pairs, head_dim);
  if (limit > P / 2) return fail(GKR_ERR_INVALID, "%s: a limit of %u (at most 2^30 - 1)", what, limit);
  uint64_t rows = 0;
  for (size_t i = 0; i < n; i++) {
    const uint32_t start = starts ? starts[i] : 0;
    if (start > r->positions || counts[i] > r->positions - start)
      return fail(GKR_ERR_INVALID, "%s: %u tokens from position %u on (of %u)", what, counts[i], start, r->positions);
    rows += counts[i];
  }
  uint64_t units = 0;
  const uint32_t a_head = (r->pairs + 3) / 4 + (head_dim - 2 * r->pairs + 7) / 8;
  for (const gkr_matrix* m : {q, k}) {
    if (!m) continue;
    const char* const name = m == q ? "q" : "k";
    if (m->cols % head_dim) return fail(GKR_ERR_INVALID, "%s: %s has %llu columns, not whole heads of %u", what, name,
                                        (unsigned long long)m->cols, head_dim);
    if (m->cols > 1u << 30) return fail(GKR_ERR_INVALID, "%s: %s has %llu columns (at most 2^30)", what, name,
                                        (unsigned long long)m->cols);
    TRY(check_shape(what, name, m, rows, m->cols));
    units += m->cols / head_dim * a_head;
  }
  TRY(check_shape(what, "q's output", q_out, rows, q->cols));
  if (k) TRY(check_shape(what, "k's output", k_out, rows, k->cols));
  if ((units + 255) / 256 > 65535) return fail(GKR_ERR_INVALID, "%s: rows of %llu and %llu columns", what,
                                               (unsigned long long)q->cols, (unsigned long long)(k ? k->cols : 0));
  HIP_TRY(hipSetDevice(c->device));
  for (const gkr_matrix* m : {q, (const gkr_matrix*)q_out, k, (const gkr_matrix*)k_out})
    if (m && (m == q_out || m == k_out || m->dev == q_out->dev || (k_out && m->dev == k_out->dev)))
      TRY(drop_derived(c, const_cast<gkr_matrix*>(m)));
  TurnArgs a{};
  a.table = r->table;
  a.head_dim = head_dim;
  a.pairs = r->pairs;
  a.shift = r->shift;
  a.limit = (int32_t)limit;
  a.m[0] = {q->dev, q_out->dev, (uint32_t)(q->cols / head_dim)};
  if (k) a.m[1] = {k->dev, k_out->dev, (uint32_t)(k->cols / head_dim)};
  uint64_t base = 0;
  uint32_t some = 0;  // rows of the launch that is being put together
  auto launch = [&]() -> int {
    if (some == 0) return GKR_OK;
    const dim3 grid(some, (uint32_t)((units + 255) / 256));
    if (interleaved) GKR_LAUNCH(c, k_turn<true>, grid, dim3(256), 0, a, base);
    else GKR_LAUNCH(c, k_turn<false>, grid, dim3(256), 0, a, base);
    base += some;
    some = a.n = 0;
    return check_launch(c);
  };
  for (size_t i = 0; i < n; i++) {
    for (uint32_t done = 0; done < counts[i];) {
      const uint32_t take = std::min(counts[i] - done, kTurnRows - some);
      a.e[a.n].row0 = some;
      a.e[a.n].position = (starts ? starts[i] : 0) + done;
      a.n++;
      some += take;
      done += take;
      if (a.n == kTurnSeqs || some == kTurnRows) TRY(launch());
    }
  }
  return launch();
}
extern "C" int gkr_rotary_forward(gkr_ctx* c, const gkr_rotary* r, uint32_t head_dim, int interleaved,
                                  const uint32_t* starts, const uint32_t* counts, size_t n, uint32_t limit,
                                  const gkr_matrix* q, gkr_matrix* q_out, const gkr_matrix* k, gkr_matrix* k_out) {
  return guarded([&] { return rotary_forward(c, r, head_dim, interleaved, starts, counts, n, limit, q, q_out, k, k_out); });
}
