// The paged key-value cache and attention over it (kernels in attend.h).
#include "internal.h"
#include "activations.h"
#include "attend.h"

struct gkr_kv_cache {
  gkr_ctx* ctx;
  KvPool pool{};
  uint32_t* table = nullptr;  // device: pool.pages
  uint32_t* bad = nullptr;    // coherent host word: an append met a word outside the int8 range
  std::unique_ptr<KvBook> book;
};

void release_cache(gkr_kv_cache* k) {
  if (k->pool.k) (void)hipFree(k->pool.k);
  if (k->pool.v) (void)hipFree(k->pool.v);
  if (k->table) (void)hipFree(k->table);
  if (k->bad) (void)hipHostFree(k->bad);
  k->pool.k = k->pool.v = nullptr;
  k->table = k->bad = nullptr;
  k->ctx = nullptr;
}

extern "C" int gkr_kv_cache_new(gkr_ctx* c, uint32_t kv_heads, uint32_t dim, uint32_t n_pages, uint32_t page_tokens,
                                uint32_t max_seqs, uint32_t max_tokens, int int8, gkr_kv_cache** out) {
  if (!c || !out) return fail(GKR_ERR_INVALID, "null argument");
  if (kv_heads == 0 || kv_heads > 4096 || dim == 0 || dim > 256)
    return fail(GKR_ERR_INVALID, "key-value cache: %u heads of %u values (1 .. 4096 of 1 .. 256)", kv_heads, dim);
  if (page_tokens == 0 || page_tokens % kAttBlock || page_tokens > 65536)
    return fail(GKR_ERR_INVALID, "key-value cache: pages of %u tokens (a multiple of %u up to 65536)", page_tokens,
                kAttBlock);
  if (n_pages == 0 || max_seqs == 0 || max_seqs > 1u << 20 || max_tokens == 0 || max_tokens > kMaxTokens)
    return fail(GKR_ERR_INVALID, "key-value cache: %u pages, %u sequences of up to %u tokens (at most 2^20 of 2^21)",
                n_pages, max_seqs, max_tokens);
  const uint32_t width = (max_tokens + page_tokens - 1) / page_tokens, chunks = (dim + 15) / 16;
  if ((uint64_t)max_seqs * width > 1ull << 32)
    return fail(GKR_ERR_INVALID, "key-value cache: a page table of %u x %u", max_seqs, width);
  uint64_t bytes;
  if (!kv_pool_bytes(n_pages, page_tokens, kv_heads, dim, int8 ? 1 : 4, &bytes))
    return fail(GKR_ERR_INVALID, "key-value cache: %u pages of %u tokens, %u heads of %u values: pools of more than 2^48 bytes",
                n_pages, page_tokens, kv_heads, dim);
  HIP_TRY(hipSetDevice(c->device));
  gkr_kv_cache* k = nullptr;
  const int rc = guarded([&]() -> int {
    k = new gkr_kv_cache{c};
    k->pool.width = width;
    k->pool.page_blocks = page_tokens / kAttBlock;
    k->pool.kv_heads = kv_heads;
    k->pool.dim = dim;
    k->pool.chunks = chunks;
    k->pool.planes = int8 ? 1 : 4;
    c->caches.insert(k);
    return GKR_OK;
  });
  if (rc != GKR_OK) {
    delete k;
    return rc;
  }
  drain(c);
  if (hipMalloc(&k->pool.k, bytes) != hipSuccess || hipMalloc(&k->pool.v, bytes) != hipSuccess ||
      hipMalloc(&k->table, (uint64_t)max_seqs * width * sizeof(uint32_t)) != hipSuccess ||
      hipHostMalloc((void**)&k->bad, 64, hipHostMallocCoherent | hipHostMallocMapped) != hipSuccess) {
    (void)hipGetLastError();
    gkr_kv_cache_free(k);
    return fail(GKR_ERR_NOMEM, "key-value cache: two pools of %llu bytes", (unsigned long long)bytes);
  }
  // after the pools: four bytes a page on the host, 16 GB for the most that can be asked for
  const int booked = guarded([&]() -> int {
    k->book.reset(new KvBook(n_pages, page_tokens, max_seqs, max_tokens));
    return GKR_OK;
  });
  if (booked != GKR_OK) {
    gkr_kv_cache_free(k);
    return booked;
  }
  k->pool.pages = k->table;
  *k->bad = 0;
  // entries that no append has set name a page that there is
  const hipError_t e = hipMemsetAsync(k->table, 0, (uint64_t)max_seqs * width * sizeof(uint32_t), c->stream);
  if (e != hipSuccess) {
    gkr_kv_cache_free(k);
    return fail(GKR_ERR_DEVICE, "key-value cache: clear of the page table: %s", hipGetErrorString(e));
  }
  *out = k;
  return GKR_OK;
}
extern "C" void gkr_kv_cache_free(gkr_kv_cache* k) {
  if (!k) return;
  if (k->ctx) {
    drain(k->ctx);
    (void)hipStreamSynchronize(k->ctx->stream);
    k->ctx->caches.erase(k);
    release_cache(k);
  }
  delete k;
}
static int check_seq(const gkr_kv_cache* k, uint32_t seq) {
  if (!k) return fail(GKR_ERR_INVALID, "null argument");
  if (!k->ctx) return fail(GKR_ERR_INVALID, "key-value cache of a destroyed context");
  if (!k->book->live(seq)) return fail(GKR_ERR_INVALID, "no sequence %u in this cache", seq);
  return GKR_OK;
}
extern "C" int gkr_kv_cache_new_sequence(gkr_kv_cache* k, uint32_t* seq) {
  if (!k || !seq) return fail(GKR_ERR_INVALID, "null argument");
  if (!k->ctx) return fail(GKR_ERR_INVALID, "key-value cache of a destroyed context");
  if (!k->book->open(seq)) return fail(GKR_ERR_NOMEM, "key-value cache: all %u sequences in use", k->book->max_seqs());
  return GKR_OK;
}
extern "C" int gkr_kv_cache_truncate(gkr_kv_cache* k, uint32_t seq, uint32_t n_tokens) {
  TRY(check_seq(k, seq));
  if (n_tokens > k->book->seq(seq).len)
    return fail(GKR_ERR_INVALID, "sequence %u has %u tokens, not %u", seq, k->book->seq(seq).len, n_tokens);
  k->book->cut(seq, n_tokens);
  return GKR_OK;
}
extern "C" int gkr_kv_cache_free_sequence(gkr_kv_cache* k, uint32_t seq) {
  TRY(check_seq(k, seq));
  k->book->close(seq);
  return GKR_OK;
}
extern "C" int gkr_kv_cache_length(const gkr_kv_cache* k, uint32_t seq, uint32_t* n) {
  if (!n) return fail(GKR_ERR_INVALID, "null argument");
  TRY(check_seq(k, seq));
  *n = k->book->seq(seq).len;
  return GKR_OK;
}
extern "C" int gkr_kv_cache_free_pages(const gkr_kv_cache* k, uint32_t* n) {
  if (!k || !n) return fail(GKR_ERR_INVALID, "null argument");
  *n = k->book->free_pages();
  return GKR_OK;
}

static int append_launches(gkr_ctx* c, gkr_kv_cache* k, const uint32_t* counts,
                           const std::vector<KvBook::Before>& before, const uint32_t* kw, const uint32_t* vw) {
  KvSlots slots{};
  // the tokens' stores go by the table: an entry that was not set names another sequence's page, so none is
  // launched before the runtime has taken these launches
  auto set_pages = [&]() -> int {
    if (slots.n == 0) return GKR_OK;
    GKR_LAUNCH(c, k_kv_pages, dim3(1), dim3(256), 0, k->table, slots);
    slots.n = 0;
    drain(c);
    return check_launch(c);
  };
  for (size_t i = 0; i < before.size(); i++) {
    const KvBook::Before& was = before[i];
    const auto& pages = k->book->seq(was.seq).pages;
    for (uint32_t p = was.pages; p < k->book->pages_of(was.len + counts[i]); p++) {
      slots.e[slots.n++] = {was.seq * k->pool.width + p, pages[p]};
      if (slots.n == 256) TRY(set_pages());
    }
  }
  TRY(set_pages());
  KvAppend a{};
  uint32_t quads = 0;
  auto store = [&]() -> int {
    if (quads && k->pool.dim % 4 == 0)
      GKR_LAUNCH(c, k_kv_append<4>, dim3(quads), dim3(256), 0, k->pool, a, kw, vw, k->bad);
    else if (quads)
      GKR_LAUNCH(c, k_kv_append<1>, dim3(quads), dim3(256), 0, k->pool, a, kw, vw, k->bad);
    a.n = quads = 0;
    return check_launch(c);
  };
  uint64_t row = 0;
  for (size_t i = 0; i < before.size(); i++) {
    if (counts[i] == 0) continue;
    const uint32_t pos = before[i].len;
    a.e[a.n++] = {before[i].seq, pos, counts[i], quads, row};
    quads += (pos + counts[i] + 3) / 4 - pos / 4;
    row += counts[i];
    if (a.n == kAttRows || quads > 1u << 22) TRY(store());  // at most 2^22 + 2^19 workgroups
  }
  return store();
}
static int append(gkr_ctx* c, gkr_kv_cache* k, const uint32_t* seqs, const uint32_t* counts, size_t n,
                  const gkr_matrix* km, const gkr_matrix* vm) {
  TRY(check_operands(c, "cache append", {km, vm}, {}));
  const uint64_t width = (uint64_t)k->pool.kv_heads * k->pool.dim;
  uint64_t total = 0;
  for (size_t i = 0; i < n; i++) {
    TRY(check_seq(k, seqs[i]));
    total += counts[i];
  }
  TRY(check_shape("cache append", "k", km, total, width));
  TRY(check_shape("cache append", "v", vm, total, width));
  std::vector<KvBook::Before> before;  // lengths and pages first; taken back if anything fails
  std::string why;
  if (!k->book->extend(seqs, counts, n, &before, &why)) return fail(GKR_ERR_NOMEM, "cache append: %s", why.c_str());
  struct Undo {
    KvBook& book;
    const std::vector<KvBook::Before>& before;
    bool kept = false;
    ~Undo() {
      if (!kept) book.back(before);
    }
  } undo{*k->book, before};
  int rc = append_launches(c, k, counts, before, km->dev, vm->dev);
  if (rc == GKR_OK) {  // a launcher thread's refusal is there once it has issued them all
    drain(c);
    rc = check_launch(c);
  }
  if (k->pool.planes == 1) {
    if (rc != GKR_OK) {  // a launch was refused: one before it may still set the word
      drain(c);
      (void)hipStreamSynchronize(c->stream);
    } else {
      rc = sync(c);
      if (rc == GKR_OK && *(volatile uint32_t*)k->bad)
        rc = fail(GKR_ERR_INVALID, "cache append: a word outside -128 .. 127 for an int8 cache");
    }
    *(volatile uint32_t*)k->bad = 0;
  }
  undo.kept = rc == GKR_OK;
  return rc;
}
extern "C" int gkr_kv_cache_append(gkr_ctx* c, gkr_kv_cache* k, const uint32_t* seqs, const uint32_t* counts, size_t n,
                                   const gkr_matrix* km, const gkr_matrix* vm) {
  if (!c || !k || !km || !vm || (n && (!seqs || !counts))) return fail(GKR_ERR_INVALID, "null argument");
  if (k->ctx != c) return fail(GKR_ERR_INVALID, "key-value cache belongs to another (or a destroyed) context");
  HIP_TRY(hipSetDevice(c->device));
  return guarded([&] { return append(c, k, seqs, counts, n, km, vm); });
}

static int attention_forward(gkr_ctx* c, const gkr_kv_cache* k, const gkr_matrix* q, const uint32_t* seqs,
                             const uint32_t* lens, size_t n_rows, uint32_t heads, uint32_t offset, uint32_t table_log,
                             gkr_matrix* weighted, gkr_matrix* sums, gkr_matrix* scores, gkr_matrix* out) {
  static const char what[] = "attention";
  if (!c || !k || !q || !out || !seqs) return fail(GKR_ERR_INVALID, "null argument");
  if (k->ctx != c) return fail(GKR_ERR_INVALID, "key-value cache belongs to another (or a destroyed) context");
  TRY(check_operands(c, what, {q}, {weighted, sums, scores, out}));
  const KvPool& pool = k->pool;
  if (heads == 0 || heads % pool.kv_heads || heads > 65535)
    return fail(GKR_ERR_INVALID, "%s: %u query heads on %u kv heads", what, heads, pool.kv_heads);
  if (offset >= P) return fail(GKR_ERR_INVALID, "%s: the offset %u is not a canonical M31", what, offset);
  if (table_log > 24) return fail(GKR_ERR_INVALID, "%s: a table of 2^%u entries (at most 2^24)", what, table_log);
  if (table_log == 0) table_log = act_default_log_size(ACT_SOFTMAX);
  const uint64_t width = (uint64_t)heads * pool.dim;
  TRY(check_shape(what, "q", q, n_rows, width));
  TRY(check_shape(what, "the output", out, n_rows, width));
  TRY(check_shape(what, "weighted", weighted, n_rows, width));
  TRY(check_shape(what, "sums", sums, n_rows, heads));
  uint32_t longest = 0;
  for (size_t i = 0; i < n_rows; i++) {
    TRY(check_seq(k, seqs[i]));
    const uint32_t have = k->book->seq(seqs[i]).len;
    if (lens && lens[i] > have)
      return fail(GKR_ERR_INVALID, "%s: row %zu sees %u tokens of a sequence of %u", what, i, lens[i], have);
    longest = std::max(longest, lens ? lens[i] : have);
  }
  if (scores) {
    TRY(check_shape(what, "scores", scores, n_rows * heads, scores->cols));
    if (scores->cols < longest || scores->cols > kMaxTokens)
      return fail(GKR_ERR_INVALID, "%s: scores of %llu columns for rows of up to %u tokens (at most 2^21)", what,
                  (unsigned long long)scores->cols, longest);
  }
  HIP_TRY(hipSetDevice(c->device));
  for (gkr_matrix* m : {weighted, sums, scores, out})
    if (m) TRY(drop_derived(c, m));
  AttOut o{out->dev, weighted ? weighted->dev : nullptr, sums ? sums->dev : nullptr, scores ? scores->dev : nullptr,
           scores ? scores->cols : 0};
  const uint32_t tiles = (heads / pool.kv_heads + kAttHeads - 1) / kAttHeads, wide = pool.kv_heads * tiles;
  const uint32_t mask = (1u << table_log) - 1;
  for (size_t row0 = 0; row0 < n_rows; row0 += kAttRows) {
    const uint32_t n = (uint32_t)std::min<size_t>(kAttRows, n_rows - row0);
    AttRowArgs rows{};
    rows.n = n;
    rows.wide = wide;
    uint64_t all_steps = 0, longest_steps = 0;
    for (uint32_t i = 0; i < n; i++) {
      const uint32_t seq = seqs[row0 + i], len = lens ? lens[row0 + i] : k->book->seq(seq).len;
      const uint64_t tokens = scores ? scores->cols : len;  // the scores behind the last token are cleared
      rows.e[i].step0 = all_steps;
      rows.e[i].seq = seq;
      rows.e[i].len = len;
      const uint64_t row_steps = std::max<uint64_t>(1, (tokens + 4 * kAttBlock - 1) / (4 * kAttBlock));
      rows.e[i].steps = (uint32_t)row_steps;
      all_steps += wide * row_steps;
      longest_steps = std::max(longest_steps, row_steps);
    }
    // as many workgroups as fit at once, with equal shares; more where a share would be too long
    const uint32_t fit = kAttWaveGroups[pool.planes == 1 ? 0 : 1];
    const uint64_t groups = std::max<uint64_t>(std::min<uint64_t>(fit, all_steps),
                                               (all_steps + kAttMaxSteps - 2) / (kAttMaxSteps - 1));
    if (groups > 1u << 23) return fail(GKR_ERR_INVALID, "%s: too many tokens and heads for one launch", what);
    rows.share = all_steps / groups;
    rows.extra = all_steps % groups;
    const uint64_t segments = (uint64_t)n * wide, part_heads = std::min(kAttHeads, heads / pool.kv_heads);
    int64_t* part = nullptr;
    uint32_t* part_z = nullptr;
    const bool join = groups > 1 && all_steps > segments;  // with one step a segment none is shared
    if (join) {
      TRY(ensureT(c, S_ATTP, (segments + groups) * part_heads * (pool.dim + 1), &part));
      part_z = reinterpret_cast<uint32_t*>(part + (segments + groups) * part_heads * pool.dim);
    }
    auto launch = [&](auto kernel) {
      GKR_LAUNCH(c, kernel, dim3((uint32_t)groups), dim3(256), 0, pool, pool.pages, rows, q->dev, heads, (uint32_t)row0, offset, mask,
                 part, part_z, o);
    };
    const uint32_t steps = (pool.dim + 63) / 64;
    if (pool.planes == 1) {
      if (steps == 1) launch(k_attend<1, 1>);
      else if (steps == 2) launch(k_attend<1, 2>);
      else launch(k_attend<1, 4>);
    } else {
      if (steps == 1) launch(k_attend<4, 1>);
      else if (steps == 2) launch(k_attend<4, 2>);
      else launch(k_attend<4, 4>);
    }
    TRY(check_launch(c));
    if (join) {
      auto launch_join = [&](auto kernel, uint32_t threads) {
        GKR_LAUNCH(c, kernel, dim3((uint32_t)segments, (uint32_t)part_heads), dim3(threads), 0, rows, heads,
                   pool.kv_heads, pool.dim, (uint32_t)row0, part, part_z, o);
      };
      if (longest_steps * groups <= 6 * all_steps) launch_join(k_attend_join<1>, steps * 64);
      else launch_join(k_attend_join<8>, 512);
      TRY(check_launch(c));
    }
  }
  return GKR_OK;
}

extern "C" int gkr_attention_forward(gkr_ctx* c, const gkr_kv_cache* k, const gkr_matrix* q, const uint32_t* seqs,
                                     const uint32_t* lens, size_t n_rows, uint32_t heads, uint32_t offset,
                                     uint32_t table_log, gkr_matrix* weighted, gkr_matrix* sums, gkr_matrix* scores,
                                     gkr_matrix* out) {
  return guarded([&] {
    return attention_forward(c, k, q, seqs, lens, n_rows, heads, offset, table_log, weighted, sums, scores, out);
  });
}
