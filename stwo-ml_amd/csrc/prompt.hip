// Causal attention of whole prompts (kernels in prompt.h).
#include <algorithm>
#include <vector>

#include "activations.h"
#include "prompt.h"
#include "witness_launch.h"

static int attention_prompt(gkr_ctx* c, const gkr_matrix* q, const gkr_matrix* k, const gkr_matrix* v,
                            const uint32_t* counts, size_t n_seqs, uint32_t heads, uint32_t kv_heads, uint32_t offset,
                            uint32_t table_log, gkr_matrix* weighted, gkr_matrix* sums, gkr_matrix* scores,
                            gkr_matrix* out) {
  static const char what[] = "prompt attention";
  if (!c || !q || !k || !v || !out || (n_seqs && !counts)) return fail(GKR_ERR_INVALID, "null argument");
  TRY(check_operands(c, what, {q, k, v}, {weighted, sums, scores, out}));
  if (kv_heads == 0 || kv_heads > 4096 || heads == 0 || heads % kv_heads || heads > 65535)
    return fail(GKR_ERR_INVALID, "%s: %u query heads on %u kv heads (at most 65535 on 4096)", what, heads, kv_heads);
  if (q->cols % heads || q->cols / heads > 256)
    return fail(GKR_ERR_INVALID, "%s: q has %llu columns, not %u heads of at most 256", what,
                (unsigned long long)q->cols, heads);
  if (offset >= P) return fail(GKR_ERR_INVALID, "%s: the offset %u is not a canonical M31", what, offset);
  if (table_log > 24) return fail(GKR_ERR_INVALID, "%s: a table of 2^%u entries (at most 2^24)", what, table_log);
  if (table_log == 0) table_log = act_default_log_size(ACT_SOFTMAX);
  const uint32_t dim = (uint32_t)(q->cols / heads), chunks = (dim + 15) / 16, group = heads / kv_heads;
  uint64_t rows = 0, blocks = 0, longest = 0;
  for (size_t i = 0; i < n_seqs; i++) {
    if (counts[i] > kMaxPrompt || (uint64_t)counts[i] * group > 0x7fffffffull)
      return fail(GKR_ERR_INVALID, "%s: a sequence of %u tokens of %u heads each (at most %u, and 2^31 rows)", what, counts[i],
                  group, kMaxPrompt);
    rows += counts[i];
    blocks += (counts[i] + kAttBlock - 1) / kAttBlock;
    longest = std::max<uint64_t>(longest, counts[i]);
  }
  TRY(check_shape(what, "q", q, rows, (uint64_t)heads * dim));
  TRY(check_shape(what, "k", k, rows, (uint64_t)kv_heads * dim));
  TRY(check_shape(what, "v", v, rows, (uint64_t)kv_heads * dim));
  TRY(check_shape(what, "the output", out, rows, (uint64_t)heads * dim));
  TRY(check_shape(what, "weighted", weighted, rows, (uint64_t)heads * dim));
  TRY(check_shape(what, "sums", sums, rows, heads));
  if (scores) {
    TRY(check_shape(what, "scores", scores, rows * heads, scores->cols));
    if (scores->cols < longest || scores->cols > kMaxTokens)
      return fail(GKR_ERR_INVALID, "%s: scores of %llu columns for sequences of up to %llu tokens (at most 2^21)", what,
                  (unsigned long long)scores->cols, (unsigned long long)longest);
  }
  if (rows > 0xffffffffull || blocks > 0xffffffffull) return fail(GKR_ERR_INVALID, "%s: too many tokens", what);
  HIP_TRY(hipSetDevice(c->device));
  for (gkr_matrix* m : {weighted, sums, scores, out})
    if (m) TRY(drop_derived(c, m));
  const uint64_t pool = blocks * (4 * 1024 * chunks) * kv_heads;
  int8_t *kd, *vd;
  uint32_t* upper;
  TRY(ensureT(c, S_PROMPTK, pool, &kd));
  TRY(ensureT(c, S_PROMPTV, pool, &vd));
  TRY(ensureT(c, S_PROMPTU, blocks * kv_heads, &upper));
  uint32_t *mask, *next_mask;
  TRY(wit_masks(c, &mask, &next_mask));

  auto pack_all = [&](uint32_t* counter, uint32_t counters) -> int {
    PromptPack pack{};
    pack.kv_heads = kv_heads;
    pack.dim = dim;
    pack.chunks = chunks;
    pack.blocks = (uint32_t)blocks;
    pack.counter = counter;
    pack.counters = counters;
    uint32_t in_launch = 0;
    uint64_t row = 0, at = 0;
    auto launch = [&]() -> int {
      if (in_launch == 0) return GKR_OK;
      pack.n_blocks = in_launch;
      const dim3 grid((in_launch + 7) / 8 * 8 * std::min(kv_heads, kPackHeads), (kv_heads + kPackHeads - 1) / kPackHeads);
      auto one = [&](auto kernel) {
        GKR_LAUNCH(c, kernel, grid, dim3(64 * std::min(kPackWaves, 2 * chunks)), 0, pack, k->dev, v->dev, kd, vd, upper, mask, next_mask);
      };
      if (2 * chunks <= kPackWaves) one(k_prompt_pack<1>);
      else one(k_prompt_pack<2>);
      pack.n = in_launch = pack.counters = 0;  // cleared by the first
      return check_launch(c);
    };
    for (size_t i = 0; i < n_seqs; i++) {
      if (counts[i] == 0) continue;
      const uint32_t some = (counts[i] + kAttBlock - 1) / kAttBlock;
      auto& e = pack.e[pack.n++];
      e.block0 = in_launch;
      e.len = counts[i];
      e.at = (uint32_t)at;
      e.row = (uint32_t)row;
      in_launch += some;
      at += some;
      row += counts[i];
      if (pack.n == kPromptSeqs || in_launch > 1u << 14) TRY(launch());
    }
    return launch();
  };

  PromptArgs a{};
  a.k = kd;
  a.v = vd;
  a.q = q->dev;
  a.mask = mask;
  a.o = AttOut{out->dev, weighted ? weighted->dev : nullptr, sums ? sums->dev : nullptr, scores ? scores->dev : nullptr,
               scores ? scores->cols : 0};
  a.blocks = (uint32_t)blocks;
  a.upper = upper;
  a.kv_heads = kv_heads;
  a.group = group;
  a.dim = dim;
  a.chunks = chunks;
  a.offset = offset;
  a.table_mask = (1u << table_log) - 1;
  // Long sequences first: the last workgroups have little to do (16 prompts of 0 to 1024
  // tokens: the int8 kernel 99 us in the order they came in, 90 so).
  std::vector<uint32_t> order, first_row(n_seqs), first_block(n_seqs);
  for (size_t i = 0, row = 0, block = 0; i < n_seqs; i++) {
    first_row[i] = (uint32_t)row;
    first_block[i] = (uint32_t)block;
    row += counts[i];
    block += (counts[i] + kAttBlock - 1) / kAttBlock;
    if (counts[i]) order.push_back((uint32_t)i);
  }
  std::stable_sort(order.begin(), order.end(), [&](uint32_t x, uint32_t y) { return counts[x] > counts[y]; });
  // The sequences' items, in workgroups of `tile` rows: the packing, then for up to
  // kPromptSeqs sequences and 2^22 items (and one sequence's more, at most 2^23, so
  // that a grid has fewer than 2^32 threads) the int8 kernel's launch and the
  // other's, one of which finds nothing to do.
  auto launch_all = [&](uint32_t tile, uint32_t per, auto kernels) -> int {
    uint64_t all = 0;
    for (size_t i = 0; i < n_seqs; i++) {
      const uint64_t items = ((uint64_t)counts[i] * group + tile - 1) / tile * kv_heads;
      if (items > 1u << 23) return fail(GKR_ERR_INVALID, "%s: too many tokens and heads for one launch", what);
      all += items;
    }
    const uint64_t launches = n_seqs / kPromptSeqs + (all >> 22) + 2, room = std::min<uint64_t>(all, (1u << 22) + (1u << 23));
    TRY(ensureT(c, S_PROMPTQ, room + kPromptCounters * launches, &a.todo));
    a.counter = a.todo + room;
    TRY(pack_all(a.counter, (uint32_t)(kPromptCounters * launches)));
    auto launch = [&]() -> int {
      TRY(kernels());
      a.n = a.items = a.general_items = 0;
      a.counter += kPromptCounters;
      return GKR_OK;
    };
    for (size_t i : order) {
      auto& e = a.e[a.n++];
      e.item0 = a.items;
      e.general0 = a.general_items;
      e.tiles = (counts[i] * group + tile - 1) / tile;
      e.len = counts[i];
      e.at = first_block[i];
      e.row = first_row[i];
      a.items += e.tiles * kv_heads;
      a.general_items += (e.tiles + per - 1) / per * kv_heads;
      const bool last = i == order.back();
      if (last) a.clear = mask;
      if (last || a.n == kPromptSeqs || a.items > 1u << 22) TRY(launch());
    }
    return GKR_OK;
  };
  // R1 and W1 of the int8 kernel, R4 and W4 of the other: tiles of 16 rows a wave, waves
#define GKR_PROMPT(DT, R1, W1, OCC1, R4, W4, OCC4)                                                                    \
  return launch_all(16 * R1 * W1, R4 * W4 / (R1 * W1), [&]() -> int {                                                  \
    constexpr uint32_t PER = R4 * W4 / (R1 * W1);                                                                      \
    static_assert(PER * R1 * W1 == R4 * W4, "whole items");                                                            \
    if (scores || weighted) GKR_LAUNCH(c, (k_prompt_int8<DT, R1, W1, OCC1, true>), dim3(a.items), dim3(64 * W1), 0, a); \
    else GKR_LAUNCH(c, (k_prompt_int8<DT, R1, W1, OCC1, false>), dim3(a.items), dim3(64 * W1), 0, a);                  \
    TRY(check_launch(c));                                                                                              \
    const dim3 grid(std::min(a.general_items, 256u * (OCC4 * 4 / W4)));                                                \
    if (scores || weighted) GKR_LAUNCH(c, (k_prompt<DT, R4, W4, OCC4, PER, true>), grid, dim3(64 * W4), 0, a);         \
    else GKR_LAUNCH(c, (k_prompt<DT, R4, W4, OCC4, PER, false>), grid, dim3(64 * W4), 0, a);                           \
    return check_launch(c);                                                                                            \
  })
  if (dim <= 64) GKR_PROMPT(1, 1, 4, 4, 1, 8, 2);
  if (dim <= 128) GKR_PROMPT(2, 1, 4, 4, 1, 8, 2);
  GKR_PROMPT(4, 1, 4, 2, 1, 4, 1);
#undef GKR_PROMPT
}
extern "C" int gkr_attention_prompt(gkr_ctx* c, const gkr_matrix* q, const gkr_matrix* k, const gkr_matrix* v,
                                    const uint32_t* counts, size_t n_seqs, uint32_t heads, uint32_t kv_heads,
                                    uint32_t offset, uint32_t table_log, gkr_matrix* weighted, gkr_matrix* sums,
                                    gkr_matrix* scores, gkr_matrix* out) {
  return guarded([&] {
    return attention_prompt(c, q, k, v, counts, n_seqs, heads, kv_heads, offset, table_log, weighted, sums, scores, out);
  });
}
