// Test-only host build of the key-value cache's page book (stwo-ml_amd/csrc/kv_book.h).
#include "../../stwo-ml_amd/csrc/kv_book.h"

using namespace gkr;

extern "C" {
KvBook* kvb_new(uint32_t pages, uint32_t page_tokens, uint32_t seqs, uint32_t max_tokens) {
  return new KvBook(pages, page_tokens, seqs, max_tokens);
}
void kvb_free(KvBook* b) { delete b; }
int kvb_open(KvBook* b, uint32_t* seq) { return b->open(seq); }
void kvb_close(KvBook* b, uint32_t seq) { b->close(seq); }
void kvb_cut(KvBook* b, uint32_t seq, uint32_t n) { b->cut(seq, n); }
int kvb_live(KvBook* b, uint32_t seq) { return b->live(seq); }
uint32_t kvb_free_pages(KvBook* b) { return b->free_pages(); }
uint32_t kvb_len(KvBook* b, uint32_t seq) { return b->seq(seq).len; }
uint32_t kvb_pages(KvBook* b, uint32_t seq, uint32_t* out) {
  const auto& p = b->seq(seq).pages;
  for (size_t i = 0; i < p.size(); i++) out[i] = p[i];
  return (uint32_t)p.size();
}
// undo != 0: extended and taken back, as when the launch behind it fails
int kvb_extend(KvBook* b, const uint32_t* seqs, const uint32_t* counts, size_t n, int undo) {
  std::vector<KvBook::Before> before;
  std::string why;
  if (!b->extend(seqs, counts, n, &before, &why)) return why.empty() ? -1 : 0;
  if (undo) b->back(before);
  return 1;
}
uint32_t kvb_key_byte(uint32_t token, uint32_t dim, uint32_t plane, uint32_t planes) {
  return kv_key_byte(token, dim, plane, planes);
}
int kvb_pool_bytes(uint32_t n_pages, uint32_t page_tokens, uint32_t kv_heads, uint32_t dim, uint32_t planes,
                   uint64_t* bytes) {
  return kv_pool_bytes(n_pages, page_tokens, kv_heads, dim, planes, bytes);
}
uint32_t kvb_value_byte(uint32_t token, uint32_t dim, uint32_t plane, uint32_t planes) {
  return kv_value_byte(token, dim, plane, planes);
}
}
