// Which pages of a paged key-value cache hold which sequence's tokens (host
// only), and where in a block a value's byte lies.
#pragma once
#include <stdint.h>
#include <stdio.h>

#include <stdexcept>
#include <string>
#include <vector>

#ifdef __HIPCC__
#define KV_HD __host__ __device__ __forceinline__
#else
#define KV_HD inline
#endif

namespace gkr {

constexpr uint32_t kAttBlock = 64;         // tokens per block
constexpr uint32_t kMaxTokens = 1u << 21;  // per sequence: sums of weights below 2^31, weighted sums below 2^61

// Byte of a plane's digit of (token in the block, dim), among the block's keys
// and among its values (attend.h: the matrix cores' operand orders).
KV_HD uint32_t kv_key_byte(uint32_t token, uint32_t dim, uint32_t plane, uint32_t planes) {
  return (dim / 16 * planes + plane) * 1024 + 16 * token + dim % 16;
}
KV_HD uint32_t kv_value_byte(uint32_t token, uint32_t dim, uint32_t plane, uint32_t planes) {
  return (dim / 16 * planes + plane) * 1024 + 256 * (token / 4 % 4) + 16 * (dim % 16) + 4 * (token / 16) + token % 4;
}

// Bytes of one of a cache's two pools: 1 KB per page, kv head, block of 64
// tokens, plane and 16 dims.  False if it is more than 2^48, beyond any device;
// the product of the sizes that a cache takes can pass 2^64.
inline bool kv_pool_bytes(uint32_t n_pages, uint32_t page_tokens, uint32_t kv_heads, uint32_t dim, uint32_t planes,
                          uint64_t* bytes) {
  const uint64_t page = (uint64_t)kv_heads * (page_tokens / kAttBlock) * planes * ((dim + 15) / 16) * 1024;  // <= 2^38
  if (n_pages > (1ull << 48) / page) return false;
  *bytes = n_pages * page;
  return true;
}

class KvBook {
 public:
  struct Seq {
    bool live = false;
    uint32_t len = 0;
    std::vector<uint32_t> pages;
  };
  // What extend() found: to set page table entries from, or to go back to.
  struct Before {
    uint32_t seq, len, pages;
  };

  KvBook(uint32_t n_pages, uint32_t page_tokens, uint32_t max_seqs, uint32_t max_tokens)
      : page_tokens_(page_tokens), max_tokens_(max_tokens), seqs_(max_seqs) {
    free_seqs_.reserve(max_seqs);
    for (uint32_t s = max_seqs; s-- > 0;) free_seqs_.push_back(s);
    free_pages_.reserve(n_pages);  // room for all: giving pages back never allocates
    for (uint32_t p = n_pages; p-- > 0;) free_pages_.push_back(p);
  }
  bool live(uint32_t seq) const { return seq < seqs_.size() && seqs_[seq].live; }
  const Seq& seq(uint32_t s) const { return seqs_[s]; }
  uint32_t free_pages() const { return (uint32_t)free_pages_.size(); }
  uint32_t max_seqs() const { return (uint32_t)seqs_.size(); }
  uint32_t pages_of(uint32_t tokens) const { return tokens / page_tokens_ + (tokens % page_tokens_ != 0); }

  bool open(uint32_t* seq) {
    if (free_seqs_.empty()) return false;
    *seq = free_seqs_.back();
    free_seqs_.pop_back();
    seqs_[*seq].live = true;
    return true;
  }
  void close(uint32_t seq) {
    cut(seq, 0);
    seqs_[seq].live = false;
    free_seqs_.push_back(seq);
  }
  // Keeps the first n tokens; the pages behind them go back.  A later append
  // may overwrite those at once: it runs behind the calls that read them.
  void cut(uint32_t seq, uint32_t n) {
    Seq& s = seqs_[seq];
    while (s.pages.size() > pages_of(n)) {
      free_pages_.push_back(s.pages.back());
      s.pages.pop_back();
    }
    s.len = n;
  }
  // counts[i] tokens more for each of n sequences (live; one may come twice), all or none: *why says what was
  // missing.  Throws std::bad_alloc, also with nothing done.
  bool extend(const uint32_t* seqs, const uint32_t* counts, size_t n, std::vector<Before>* before, std::string* why) {
    before->clear();
    before->reserve(n);
    try {
      for (size_t i = 0; i < n; i++) {
        Seq& s = seqs_[seqs[i]];
        char text[160];
        if (counts[i] > max_tokens_ - s.len) {
          snprintf(text, sizeof text, "sequence %u has %u tokens and %u more are too many (at most %u)", seqs[i], s.len,
                   counts[i], max_tokens_);
          *why = text;
          back(*before);
          return false;
        }
        const uint32_t pages = pages_of(s.len + counts[i]);
        if (pages - s.pages.size() > free_pages_.size()) {
          snprintf(text, sizeof text, "sequence %u needs %u more pages and %u are free", seqs[i],
                   (uint32_t)(pages - s.pages.size()), free_pages());
          *why = text;
          back(*before);
          return false;
        }
        if (s.pages.capacity() < pages) s.pages.reserve(pages + pages / 2);
        before->push_back({seqs[i], s.len, (uint32_t)s.pages.size()});
        while (s.pages.size() < pages) {
          s.pages.push_back(free_pages_.back());
          free_pages_.pop_back();
        }
        s.len += counts[i];
      }
    } catch (...) {
      back(*before);
      throw;
    }
    return true;
  }
  void back(const std::vector<Before>& before) {
    for (size_t i = before.size(); i-- > 0;) cut(before[i].seq, before[i].len);
  }

 private:
  uint32_t page_tokens_, max_tokens_;
  std::vector<Seq> seqs_;
  std::vector<uint32_t> free_pages_, free_seqs_;
};

}  // namespace gkr
