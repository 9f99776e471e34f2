// Attention of new tokens over a paged key-value cache, exact over the field.
//
// For a query head and the tokens j that it sees
//   x_j = q . k_j + offset (mod P),  e_j = 2^16 2^g_j,  g_j = min((x_j mod 2^log) >> 16, 10),
//   out = round(sum_j 2^g_j c(v_j) / sum_j 2^g_j)
// The softmax table is a power of two in 0 .. 10, so no running maximum is
// needed: the sums stay whole numbers (below 2^10 2^30 tokens) and are joined
// in any order.
//
// Cache.  A page holds page_tokens / 64 blocks of 64 tokens for each kv head,
// a block's keys and values each as `planes` planes of balanced base-256
// digits (gemm.h; one plane in an int8 cache), 1 KB per 16 dims and plane (the
// planes of the same dims next to each other, so that a lane's loads of a block
// differ by constants), in the operand order of v_mfma_i32_16x16x64_i8:
//   keys    [dim / 16][plane][token][dim % 16]: lane l of the score product
//           reads token 16 t + l % 16, dims 16 (4 s + l / 16) .. + 15;
//   values  [dim / 16][plane][c][dim % 16][4 t + v] holds token 16 t + 4 c + v:
//           lane l of the value product reads dim l % 16, chunk c = l / 16.
// The score product K Q^T leaves lane l with head l % 16 and the tokens 16 t +
// 4 (l / 16) + v, which is the value product's operand order for the weights:
// they go from one product to the next without a shuffle.
#pragma once
#include <stdint.h>

#include "field.h"
#include "gemm.h"
#include "kv_book.h"

namespace gkr {

constexpr uint32_t kAttHeads = 16;   // query heads of one kv head per workgroup
constexpr uint32_t kAttRows = 128;   // rows (or sequences) per launch
constexpr uint32_t kAttMaxSteps = 256;  // a workgroup's: 65536 tokens keep the digit sums below 2^31

struct KvPool {
  int8_t *k, *v;
  const uint32_t* pages;  // [seq][width]: the pages of a sequence's tokens
  uint32_t width, page_blocks, kv_heads, dim, chunks, planes;
};
__device__ __forceinline__ uint64_t kv_block(const KvPool& p, uint32_t seq, uint32_t block, uint32_t head) {
  const uint32_t at = p.page_blocks == 1 ? block : block / p.page_blocks;  // uniform: a division less
  const uint32_t page = p.pages[(uint64_t)seq * p.width + at];
  return (((uint64_t)page * p.kv_heads + head) * p.page_blocks + (block - at * p.page_blocks)) * p.planes * p.chunks * 1024;
}

struct KvSlots {  // entries of the page table to set
  uint32_t n;
  struct {
    uint32_t slot, page;
  } e[256];
};
static __global__ void k_kv_pages(uint32_t* table, KvSlots s) {
  if (threadIdx.x < s.n) table[s.e[threadIdx.x].slot] = s.e[threadIdx.x].page;
}

struct KvAppend {
  uint32_t n;
  struct {
    uint32_t seq, pos, count, quad0;  // quad0: groups of four token positions before this entry's
    uint64_t row;                     // its first row of k and v
  } e[kAttRows];
};
// A workgroup takes four token positions 4 i .. 4 i + 3 of a sequence; tokens
// that were there stay.  A word outside an int8 cache's range sets *bad (host
// memory).  DIMS = 4 (dims a multiple of 4): a thread takes four dims of the
// four tokens, whose digits are four bytes next to each other a token among the
// keys and, where all four tokens are new, a dim among the values (65537 tokens
// of 8 x 128 general values: 982 us a value and byte at a time, 567 so);
// DIMS = 1: a value at a time.
template <int DIMS>
static __global__ void __launch_bounds__(256) k_kv_append(KvPool p, KvAppend a, const uint32_t* __restrict__ k,
                                                          const uint32_t* __restrict__ v, uint32_t* bad) {
  uint32_t i = 0;
  for (uint32_t up = a.n; up - i > 1;) {  // the last entry that begins at or before this group
    const uint32_t mid = (i + up) / 2;
    if (a.e[mid].quad0 <= blockIdx.x) i = mid;
    else up = mid;
  }
  const uint32_t pos = a.e[i].pos, end = pos + a.e[i].count;
  const uint32_t t0 = (pos / 4 + (blockIdx.x - a.e[i].quad0)) * 4;  // never crosses a block
  const uint32_t width = p.kv_heads * p.dim, block = t0 / kAttBlock, in = t0 % kAttBlock;
  uint32_t high = 0;
  for (uint32_t w = threadIdx.x * DIMS; w < width; w += blockDim.x * DIMS) {
    const uint32_t head = w / p.dim, d = w % p.dim;
    const uint64_t base = kv_block(p, a.e[i].seq, block, head);
    uint32_t kx[4][DIMS], vx[4][DIMS];  // places that are not new read a new one's, unused
#pragma unroll
    for (uint32_t t = 0; t < 4; t++) {
      const uint32_t token = t0 + t < pos ? pos : t0 + t < end ? t0 + t : end - 1;
      const uint64_t at = (a.e[i].row + (token - pos)) * width + w;
      if constexpr (DIMS == 4) {
        const v4i_word kq = *(const v4i_word*)(k + at), vq = *(const v4i_word*)(v + at);
#pragma unroll
        for (int j = 0; j < 4; j++) {
          kx[t][j] = (uint32_t)kq[j];
          vx[t][j] = (uint32_t)vq[j];
        }
      } else {
        kx[t][0] = k[at];
        vx[t][0] = v[at];
      }
    }
    uint32_t vd[DIMS][4];  // [dim][token]: digits
#pragma unroll
    for (uint32_t t = 0; t < 4; t++) {
      uint32_t kd[4] = {}, out[4];
#pragma unroll
      for (int j = 0; j < DIMS; j++) {
        kd[j] = digit_bytes(kx[t][j]);
        vd[j][t] = digit_bytes(vx[t][j]);
      }
      transpose_bytes(kd, out);
      high |= out[1] | out[2] | out[3];
      if (t0 + t < pos || t0 + t >= end) continue;
#pragma unroll
      for (uint32_t q = 0; q < 4; q++) {
        if (q >= p.planes) break;
        int8_t* const to = p.k + base + kv_key_byte(in + t, d, q, p.planes);
        if constexpr (DIMS == 4) *(uint32_t*)to = out[q];
        else *to = (int8_t)out[q];
      }
    }
    const bool whole = t0 >= pos && t0 + 4 <= end;
#pragma unroll
    for (uint32_t j = 0; j < DIMS; j++) {
      uint32_t out[4];
      transpose_bytes(vd[j], out);
      high |= out[1] | out[2] | out[3];
#pragma unroll
      for (uint32_t q = 0; q < 4; q++) {
        if (q >= p.planes) break;
        int8_t* const to = p.v + base + kv_value_byte(in, d + j, q, p.planes);
        if (whole) {
          *(uint32_t*)to = out[q];
        } else {
#pragma unroll
          for (uint32_t t = 0; t < 4; t++)
            if (t0 + t >= pos && t0 + t < end) to[t] = (int8_t)(out[q] >> (8 * t));
        }
      }
    }
  }
  if (p.planes == 1 && high) *(volatile uint32_t*)bad = 1;
}

// The rows of a launch.  Their work lies on a line: row by row, kv head (and
// tile of 16 query heads) by kv head, step by step (four blocks); a segment is
// one row's and head tile's steps, at least one.  Workgroup w takes `share`
// steps of the line, the first `extra` of them one more; where its stretch
// begins or ends inside a segment it leaves its sums of that segment in slot
// (segment + w) of the parts.
struct AttRowArgs {
  uint32_t n, wide;  // rows; segments per row
  uint64_t share, extra;
  struct {
    uint64_t step0;  // steps of the rows before it
    uint32_t seq, len, steps, pad;
  } e[kAttRows];
  __device__ __forceinline__ uint64_t begin(uint64_t w) const { return w * share + (w < extra ? w : extra); }
  // the workgroup that has step x
  __device__ __forceinline__ uint64_t owner(uint64_t x) const {
    const uint64_t longer = extra * (share + 1);
    return x < longer ? x / (share + 1) : extra + (x - longer) / share;
  }
};
struct AttOut {
  uint32_t *out, *weighted, *sums, *scores;
  uint64_t score_cols;
};

// Byte B of each of four words.
template <int B>
__device__ __forceinline__ uint32_t pick_bytes(const uint32_t (&w)[4]) {
  constexpr uint32_t sel = 0x0c0c0400u + 0x101u * B;  // byte B of the first, of the second, zeros
  return __builtin_amdgcn_perm(w[1], w[0], sel) | __builtin_amdgcn_perm(w[3], w[2], sel) << 16;
}
// A signed 32-bit number above -P mod P.
__device__ __forceinline__ uint32_t signed32_mod_p(int32_t x) { return umin32((uint32_t)x, (uint32_t)x + P); }
// A signed whole number mod P.
__device__ __forceinline__ uint32_t signed_mod_p(int64_t x) {
  const uint32_t r = m31_reduce64((uint64_t)(x < 0 ? -x : x));
  return x < 0 ? m31_neg(r) : r;
}
// 2^16 r mod P.
__device__ __forceinline__ uint32_t shift16(uint32_t r) { return m31_reduce62((uint64_t)r << 16); }
__device__ __forceinline__ void att_finish(const AttOut& o, uint64_t at, int64_t total, uint32_t z) {
  uint32_t mean = 0;
  if (z) {
    // floor((2 |total| + z) / 2 z): |c(v)| <= 2^30, so at most 2^30; the quotient in
    // 53 bits is off by one at most
    const uint64_t num = 2 * (uint64_t)(total < 0 ? -total : total) + z, den = 2 * (uint64_t)z;
    uint32_t r = (uint32_t)((double)num / (double)den);
    const int64_t rest = (int64_t)(num - (uint64_t)r * den);
    r += rest < 0 ? -1 : rest >= (int64_t)den ? 1 : 0;
    mean = total < 0 ? m31_neg(r) : r;
  }
  o.out[at] = mean;
  if (o.weighted) o.weighted[at] = shift16(signed_mod_p(total));
}

// A block of the pool as a buffer: loads add a 32-bit lane offset to its scalar
// descriptor, and those of a block of no bytes return without touching memory.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t kv_buffer(const int8_t* at, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)at, 0, (int)bytes, 0x00027000);
}
__device__ __forceinline__ v4i kv_load(__amdgpu_buffer_rsrc_t block, uint32_t at, uint32_t more) {
  constexpr int kNonTemporal = 2;
  return __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(block, (int)at + (int)more, 0, kNonTemporal));
}

// A stretch of steps, segment by segment: up to 16 query heads of one kv head.
// In a step wave w forms the scores and weights of block w, all waves read the
// four blocks' weights from LDS (two buffers, one barrier a step), and wave w
// takes the dims 16 (w + 4 i) .. + 15 of the values.  The loads run ahead: a
// wave holds NS of its four token tiles of keys and NS of the step's four
// blocks of values, and refills each as it has used it, across steps and into
// the next segment (values are loaded before their weights are known).
// What is done once a segment (the query's digits, the sums' end) goes through
// LDS in small loops: unrolled over registers, the code of a short segment took
// longer to fetch than to run.
// Bound by the cache's bytes: 64 rows of up to 4096 int8 tokens, 8 kv heads of
// 128, 56 us and 5 us of k_attend_join (4.7 TB/s; one workgroup per row, head
// and 20 blocks, whatever the lengths, 82 us); one row of 65537 general tokens
// 94 us and 7 (5.7 TB/s), 10 more with its 2.6 M scores.  Here 1024 workgroups
// for int8 caches (512: 72 us, 2048: 93), 256 of a wave per SIMD for general
// ones (512 at half the registers: 149 us).
// NP planes of the cache; DT = dims / 64 rounded up.
constexpr uint32_t kAttWaveGroups[2] = {1024, 256};  // workgroups that fit the chip at once: int8 caches, others
template <int NP, int DT>
static __global__ void __launch_bounds__(256, NP * DT <= 2 ? 2 : 1)
    k_attend(KvPool p, const uint32_t* __restrict__ pages, AttRowArgs rows, const uint32_t* __restrict__ q,
             uint32_t heads, uint32_t row0, uint32_t offset, uint32_t mask, int64_t* __restrict__ part,
             uint32_t* __restrict__ part_z, AttOut o) {
  constexpr int NG = NP + 3, NV = NP + 1;  // digit groups of the scores and of the weighted sums
  constexpr int NS = NP * DT <= 4 ? 4 : NP * DT <= 8 ? 2 : 1;
  constexpr uint32_t D = 64 * DT;
  union Shared {
    v4i weights[2][4][2][64];
    int64_t totals[kAttHeads][D];
  };
  __shared__ Shared sh;
  __shared__ v4i digits[DT][4][64];  // the query's: [dims / 64][plane][16 chunk + head]
  __shared__ uint32_t zsum[4][16];
  const uint32_t lane = threadIdx.x & 63, col = lane & 15, quarter = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t group = heads / p.kv_heads, tiles = (group + kAttHeads - 1) / kAttHeads;
  const uint32_t part_heads = group < kAttHeads ? group : kAttHeads;
  uint32_t koff[DT], voff[DT];  // this lane's bytes of a block: dims past the last read the last's again
#pragma unroll
  for (int s = 0; s < DT; s++) {
    const uint32_t chunk = 4 * s + quarter, tile = wave + 4 * s, end = p.chunks - 1;
    koff[s] = (chunk < end ? chunk : end) * (NP * 1024) + 16 * col;  // (the query's digits are zero there)
    voff[s] = (tile < end ? tile : end) * (NP * 1024) + 16 * lane;   // (not stored)
  }
  p.pages = pages;
  const uint64_t end = rows.begin((uint64_t)blockIdx.x + 1);
  struct Piece {  // of a segment: row r, kv head and tile y, steps s0 .. s1 of n, blocks .. seen_end
    uint32_t r, y, s0, s1, n, seq, kvh, seen_end;
  };
  auto piece_at = [&](uint32_t r, uint64_t pos) {
    while (r + 1 < rows.n && rows.e[r + 1].step0 <= pos) r++;
    Piece c;
    c.r = r;
    c.n = rows.e[r].steps;
    c.seq = rows.e[r].seq;
    const uint32_t in = (uint32_t)(pos - rows.e[r].step0), nblocks = (rows.e[r].len + kAttBlock - 1) / kAttBlock;
    c.y = in / c.n;
    c.s0 = in % c.n;
    c.s1 = end - pos < c.n - c.s0 ? c.s0 + (uint32_t)(end - pos) : c.n;
    c.kvh = c.y / tiles;
    c.seen_end = 4 * c.s1 < nblocks ? 4 * c.s1 : nblocks;
    return c;
  };
  auto has_data = [](const Piece& c) { return 4 * c.s0 < c.seen_end; };

  v4i kd[NS][DT][NP], vd[NS][DT][NP];
  const uint32_t bytes = NP * 1024 * p.chunks;  // of a block
  __amdgpu_buffer_rsrc_t kbase = kv_buffer(p.k, 0), vbase[4] = {kbase, kbase, kbase, kbase};
  // blocks past the end have no bytes here: their tokens have no weight
  auto key_block = [&](uint32_t seq, uint32_t kvh, uint32_t b, uint32_t seen_end) {
    const bool in = b + wave < seen_end;
    kbase = kv_buffer(p.k + (in ? kv_block(p, seq, b + wave, kvh) : 0), in ? bytes : 0);
  };
  auto load_keys = [&](int slot, int t) {
#pragma unroll
    for (int s = 0; s < DT; s++)
#pragma unroll
      for (int pk = 0; pk < NP; pk++)
        kd[slot][s][pk] = kv_load(kbase, koff[s], 256 * t + 1024 * pk);
  };
  auto value_blocks = [&](uint32_t seq, uint32_t kvh, uint32_t b, uint32_t seen_end, int j0, int j1) {
#pragma unroll
    for (int j = j0; j < j1; j++) {
      const bool in = b + j < seen_end;
      vbase[j] = kv_buffer(p.v + (in ? kv_block(p, seq, b + j, kvh) : 0), in ? bytes : 0);
    }
  };
  auto load_values = [&](int slot, int j) {
#pragma unroll
    for (int i = 0; i < DT; i++)
#pragma unroll
      for (int pv = 0; pv < NP; pv++)
        vd[slot][i][pv] = kv_load(vbase[j], voff[i], 1024 * pv);
  };

  uint64_t pos = rows.begin(blockIdx.x);
  uint32_t turn = 0, r0 = 0;
  for (uint32_t up = rows.n; up - r0 > 1;) {  // the last row that begins at or before pos
    const uint32_t mid = (r0 + up) / 2;
    if (rows.e[mid].step0 <= pos) r0 = mid;
    else up = mid;
  }
  Piece cur = piece_at(r0, pos);
  bool loaded = false;  // the first loads of `cur` went out with the piece before
#pragma unroll 1
  for (;;) {
    const uint32_t len = rows.e[cur.r].len, h0 = cur.y % tiles * kAttHeads;
    const uint32_t mine = group - h0 < kAttHeads ? group - h0 : kAttHeads, head0 = cur.kvh * group + h0;
    const uint64_t row = row0 + cur.r;
    pos += cur.s1 - cur.s0;
    const bool last = pos == end;
    const Piece next = last ? cur : piece_at(cur.r, pos);
    uint32_t words[DT][4];  // the query's, four of a head a thread and 64 dims
#pragma unroll
    for (int k = 0; k < DT; k++) {
      const uint32_t i = threadIdx.x + 256 * k, h = i / (D / 4), d0 = i % (D / 4) * 4;
      const uint32_t* const from = q + (row * heads + head0 + (h < mine ? h : 0)) * p.dim;
#pragma unroll
      for (int j = 0; j < 4; j++) words[k][j] = from[d0 + j < p.dim ? d0 + j : 0];
    }
    if (!loaded && has_data(cur)) {
      key_block(cur.seq, cur.kvh, 4 * cur.s0, cur.seen_end);
      value_blocks(cur.seq, cur.kvh, 4 * cur.s0, cur.seen_end, 0, NS);
#pragma unroll
      for (int t = 0; t < NS; t++) load_keys(t, t);
#pragma unroll
      for (int j = 0; j < NS; j++) load_values(j, j);
    }
    loaded = !last && has_data(cur) && has_data(next);
#pragma unroll
    for (int k = 0; k < DT; k++) {
      const uint32_t i = threadIdx.x + 256 * k, h = i / (D / 4), d0 = i % (D / 4) * 4;
      uint32_t d[4], out[4];
#pragma unroll
      for (int j = 0; j < 4; j++) d[j] = digit_bytes(h < mine && d0 + j < p.dim ? words[k][j] : 0u);
      transpose_bytes(d, out);
#pragma unroll
      for (int g = 0; g < 4; g++) ((uint32_t*)&digits[d0 / 64][g][d0 % 64 / 16 * 16 + h])[d0 % 16 / 4] = out[g];
    }
    __syncthreads();
    v4i qd[DT][4], acc[DT][NV];  // head col, dims 16 (4 s + quarter) .. + 15
#pragma unroll
    for (int s = 0; s < DT; s++)
#pragma unroll
      for (int g = 0; g < 4; g++) qd[s][g] = digits[s][g][lane];
#pragma unroll
    for (int i = 0; i < DT; i++)
#pragma unroll
      for (int g = 0; g < NV; g++) acc[i][g] = v4i{0, 0, 0, 0};
    uint32_t z = 0, b = 4 * cur.s0;
    uint32_t* const scores = o.scores + (row * heads + head0) * o.score_cols;  // used where given
#pragma unroll 1
    for (; b < cur.seen_end; b += 4, turn ^= 1) {
      const uint32_t block = b + wave, first = block * kAttBlock + 4 * quarter;
      // the step whose loads go out during this one: none at the end
      const bool same = b + 4 < cur.seen_end;
      const uint32_t n_seq = same ? cur.seq : next.seq, n_kvh = same ? cur.kvh : next.kvh;
      const uint32_t n_b = same ? b + 4 : 4 * next.s0, n_end = same ? cur.seen_end : loaded ? next.seen_end : 0;
      // tokens of the block that are seen, from this lane's first on
      const int left = block < cur.seen_end ? (int)(len - first) : 0;
      v4i w0, w1, x[4];
#pragma unroll
      for (int t = 0; t < 4; t++) {
        v4i sc[NG];
#pragma unroll
        for (int g = 0; g < NG; g++) sc[g] = v4i{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < DT; s++)
#pragma unroll
          for (int pk = 0; pk < NP; pk++)
#pragma unroll
            for (int g = 0; g < 4; g++)
              sc[pk + g] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kd[t % NS][s][pk], qd[s][g], sc[pk + g], 0, 0, 0);
        if (t + NS == 4) key_block(n_seq, n_kvh, n_b, n_end);
        load_keys(t % NS, (t + NS) % 4);
        uint32_t e[4], e8[4];
#pragma unroll
        for (int v = 0; v < 4; v++) {
          uint32_t xv;
          if constexpr (NP == 1) {
            // |sc[g]| <= 2^22: pairs in 32 bits, the upper one turned by 16 of 31 bits
            const uint32_t low = signed32_mod_p(sc[0][v] + (sc[1][v] << 8)), high = signed32_mod_p(sc[2][v] + (sc[3][v] << 8));
            xv = m31_add(m31_add(low, ((high << 16) & P) | (high >> 15)), offset);
          } else {
            // sum_g 256^g sc[g], below 2^52, with 2^32 = 2 (mod P)
            int64_t sum = (int64_t)sc[0][v] + ((int64_t)sc[1][v] << 8) + ((int64_t)sc[2][v] << 16) + ((int64_t)sc[3][v] << 24);
            if constexpr (NP > 1)
              sum += ((int64_t)sc[4][v] << 1) + ((int64_t)sc[5][v] << 9) + ((int64_t)sc[6][v] << 17);
            xv = m31_add(m31_reduce64((uint64_t)(sum + ((int64_t)P << 24))), offset);
          }
          x[t][v] = (int)xv;
          uint32_t g = (xv & mask) >> 16;
          g = g < 10 ? g : 10;
          e[v] = 16 * t + v < left ? 1u << g : 0u;
          e8[v] = e[v] + 0x80u;  // digits base 256, balanced: 128 is 256 - 128
          z += e[v];
        }
        const uint32_t lo = pick_bytes<0>(e), hi = pick_bytes<1>(e8);
        w0[t] = (int)lo;
        w1[t] = (int)hi;
      }
      sh.weights[turn][wave][0][lane] = w0;
      sh.weights[turn][wave][1][lane] = w1;
      if (o.scores && block < 4 * cur.s1 && col < mine) {
        const uint64_t tok = first;
        uint32_t* const out = scores + col * o.score_cols + tok;
        if ((uint64_t)block * kAttBlock + kAttBlock <= o.score_cols) {
#pragma unroll
          for (int t = 0; t < 4; t++) {
            v4i_word seen;
#pragma unroll
            for (int v = 0; v < 4; v++) seen[v] = 16 * t + v < left ? x[t][v] : 0;
            *(v4i_word*)(out + 16 * t) = seen;
          }
        } else {
#pragma unroll
          for (int t = 0; t < 4; t++)
#pragma unroll
            for (int v = 0; v < 4; v++)
              if (tok + 16 * t + v < o.score_cols) out[16 * t + v] = 16 * t + v < left ? (uint32_t)x[t][v] : 0u;
        }
      }
      __syncthreads();
      value_blocks(n_seq, n_kvh, n_b, n_end, 0, NS);
      value_blocks(cur.seq, cur.kvh, b, cur.seen_end, NS, 4);  // the rest of this step's are still to come
#pragma unroll
      for (int j = 0; j < 4; j++) {  // blocks past the end have no weight
        const v4i e0 = sh.weights[turn][j][0][lane], e1 = sh.weights[turn][j][1][lane];
#pragma unroll
        for (int i = 0; i < DT; i++)
#pragma unroll
          for (int pv = 0; pv < NP; pv++) {
            acc[i][pv] = __builtin_amdgcn_mfma_i32_16x16x64_i8(e0, vd[j % NS][i][pv], acc[i][pv], 0, 0, 0);
            acc[i][pv + 1] = __builtin_amdgcn_mfma_i32_16x16x64_i8(e1, vd[j % NS][i][pv], acc[i][pv + 1], 0, 0, 0);
          }
        load_values(j % NS, (j + NS) % 4);
      }
    }
    if (o.scores)  // behind the last token they are cleared
#pragma unroll 1
      for (uint64_t tok = (uint64_t)b * kAttBlock + threadIdx.x; tok < (uint64_t)4 * cur.s1 * kAttBlock; tok += 256)
#pragma unroll 1
        for (uint32_t h = 0; h < mine && tok < o.score_cols; h++) scores[h * o.score_cols + tok] = 0;
    z += __shfl_xor(z, 16);
    z += __shfl_xor(z, 32);
    if (lane < 16) zsum[wave][lane] = z;
    __syncthreads();  // the steps' LDS has been read
#pragma unroll
    for (int i = 0; i < DT; i++)
#pragma unroll
      for (int v = 0; v < 4; v++) {
        int64_t total = 0;
#pragma unroll
        for (int g = 0; g < NV; g++) total += (int64_t)acc[i][g][v] << (8 * g);
        sh.totals[4 * quarter + v][16 * (wave + 4 * i) + col] = total;
      }
    __syncthreads();
    const bool whole = cur.s0 == 0 && cur.s1 == cur.n;
    const uint64_t slot = (uint64_t)cur.r * rows.wide + cur.y + blockIdx.x;
#pragma unroll 1
    for (uint32_t i = threadIdx.x; i < mine * p.dim; i += 256) {
      const uint32_t h = i / p.dim, d = i - h * p.dim;
      const uint32_t zh = zsum[0][h] + zsum[1][h] + zsum[2][h] + zsum[3][h];
      const int64_t total = sh.totals[h][d];
      if (whole)
        att_finish(o, (row * heads + head0) * p.dim + i, total, zh);
      else
        part[slot * part_heads * p.dim + i] = total;
      if (d == 0) {
        if (!whole) part_z[slot * part_heads + h] = zh;
        else if (o.sums) o.sums[row * heads + head0 + h] = shift16(m31_from_u32(zh));
      }
    }
    if (last) break;
    cur = next;
    __syncthreads();  // LDS is written again
  }
}

// Joins the parts of segments that several workgroups had: workgroup (segment,
// head).  SLICES waves per 64 dims take the parts in turn: one where a segment
// has few parts, eight where it has many (one row's 64 parts, 8 heads of 128:
// 7 us with eight; 512 segments of two parts: 11 us with eight, 5 with one).
template <int SLICES>
static __global__ void __launch_bounds__(256 * (SLICES > 1 ? 2 : 1))
    k_attend_join(AttRowArgs rows, uint32_t heads, uint32_t kv_heads, uint32_t dim, uint32_t row0,
                  const int64_t* __restrict__ part, const uint32_t* __restrict__ part_z, AttOut o) {
  const uint32_t r = blockIdx.x / rows.wide, y = blockIdx.x % rows.wide, h = blockIdx.y, tid = threadIdx.x;
  const uint32_t group = heads / kv_heads, tiles = (group + kAttHeads - 1) / kAttHeads;
  const uint32_t part_heads = group < kAttHeads ? group : kAttHeads, h0 = y % tiles * kAttHeads;
  if (h0 + h >= group) return;
  const uint64_t n = rows.e[r].steps, begin = rows.e[r].step0 + y * n;
  const uint64_t w0 = rows.owner(begin), w1 = rows.owner(begin + n - 1);
  if (w0 == w1) return;  // finished where it was computed
  const uint64_t first = blockIdx.x + w0, last = blockIdx.x + w1;
  const uint64_t at = (uint64_t)(row0 + r) * heads + y / tiles * group + h0 + h;
  if constexpr (SLICES == 1) {
    uint32_t z = 0;
    int64_t t = 0;
    for (uint64_t i = first; i <= last; i++) {
      z += part_z[i * part_heads + h];
      if (tid < dim) t += part[(i * part_heads + h) * dim + tid];
    }
    if (tid < dim) att_finish(o, at * dim + tid, t, z);
    if (tid == 0 && o.sums) o.sums[at] = shift16(m31_from_u32(z));
    return;
  }
  __shared__ unsigned long long total[256];
  __shared__ uint32_t z;
  if (tid < 256) total[tid] = 0;
  if (tid == 0) z = 0;
  __syncthreads();
  for (uint32_t d = tid & 63; d < dim; d += 64) {
    int64_t t = 0;
#pragma unroll 8
    for (uint64_t i = first + (tid >> 6); i <= last; i += SLICES) t += part[(i * part_heads + h) * dim + d];
    atomicAdd(&total[d], (unsigned long long)t);
  }
  uint32_t mine = 0;
  for (uint64_t i = first + tid; i <= last; i += 64 * SLICES) mine += part_z[i * part_heads + h];
  if (mine) atomicAdd(&z, mine);
  __syncthreads();
  if (tid < dim) att_finish(o, at * dim + tid, (int64_t)total[tid], z);
  if (tid == 0 && o.sums) o.sums[at] = shift16(m31_from_u32(z));
}

}  // namespace gkr
