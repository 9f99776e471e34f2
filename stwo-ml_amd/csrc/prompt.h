// Causal attention of whole prompts, exact over the field: the weights and means
// of attend.h, for packed sequences whose every token sees itself and those
// before it.
//
// The rows of a kv head are its tokens' query heads, token by token (row r of a
// sequence: token r / group, head r % group of the kv head's), so a tile of rows
// has the same keys and almost the same end.  Keys and values are packed first
// into blocks of 64 tokens per kv head, four planes of balanced base-256 digits
// each, in the operand order of v_mfma_i32_16x16x64_i8 (kv_book.h gives a plane's
// bytes): the score product leaves a lane with the tokens that the value product
// takes from it.
#pragma once
#include <stdint.h>

#include "attend.h"
#include "field.h"
#include "gemm.h"
#include "kv_book.h"
#include "witness.h"

namespace gkr {

constexpr uint32_t kPromptSeqs = 128;      // sequences per launch
constexpr uint32_t kMaxPrompt = 131071;    // tokens of one: digit sums stay below 2^31
// Words of the mask (witness.h) that the packing sets: every wave of the products
// reads them all, a line each.
constexpr uint32_t kPromptWords = 16;
__device__ __forceinline__ uint32_t prompt_mask(const uint32_t* mask) {  // this lane's
  return mask[kMaskStride * (threadIdx.x & (kPromptWords - 1))];
}

struct PromptPack {
  uint32_t n, kv_heads, dim, chunks;
  uint32_t n_blocks, blocks, counters;  // blocks of this launch; blocks of a kv head, all sequences'; launches of the products to come
  uint32_t* counter;
  struct {
    uint32_t block0, len, at;  // its first block in this launch; tokens; its first block of all
    uint32_t row;              // its first row of k and v
  } e[kPromptSeqs];
};
// Bytes of plane p of a block begin at p * chunks * 1024.
__device__ __forceinline__ uint32_t prompt_key(uint32_t token, uint32_t chunk) { return chunk * 1024 + 16 * token; }
__device__ __forceinline__ uint32_t prompt_value(uint32_t quarter, uint32_t dim) {
  return dim / 16 * 1024 + 256 * quarter + 16 * (dim % 16);
}
// A workgroup packs a block of 64 tokens of one kv head, a wave 16 dims of its keys
// or of its values at a time (so that all words are asked for at once).
// A digit above plane 0 is rare: the three upper planes are stored only where the
// block's keys, or values, have such a digit, which its word of `upper` tells the
// products (bit 0 keys, bit 1 values); then a word of the mask is set too, as in
// k_wit_pack, and `clear`, the mask of the next operator on the stream, is zeroed.
// Places behind a sequence's last token get its words again: they have no weight.
// The workgroups of an XCD (blockIdx 8 apart) take the heads of a block one after
// another, so that it reads whole rows.  All of a wave's loads go out before a branch on
// a dim's place in its head (heads of a multiple of four dims: whole 16 bytes, and one
// branch for all; 7599 tokens of 8 x 128 62 -> 36 us), and a lane stores the 16 bytes
// that it holds of a plane (36 -> 23 us, 4096 tokens 9.3).
constexpr uint32_t kPackHeads = 64;  // along one grid dimension
constexpr uint32_t kPackWaves = 16;
template <uint32_t PIECES>  // a wave's: of 32 there are at most
static __global__ void __launch_bounds__(64 * kPackWaves) k_prompt_pack(PromptPack a, const uint32_t* __restrict__ k,
                                                             const uint32_t* __restrict__ v, int8_t* __restrict__ ko,
                                                             int8_t* __restrict__ vo, uint32_t* __restrict__ upper,
                                                             uint32_t* __restrict__ mask, uint32_t* __restrict__ clear) {
  __shared__ uint32_t highs[kPackWaves];  // of the waves: bit 0 keys, bit 1 values
  const uint32_t waves = blockDim.x / 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (blockIdx.x == 0 && blockIdx.y == 0) {
    if (threadIdx.x < kMaskWords) clear[kMaskStride * threadIdx.x] = 0;
    for (uint32_t c = threadIdx.x; c < a.counters; c += blockDim.x) a.counter[c] = 0;
  }
  const uint32_t wide = a.kv_heads < kPackHeads ? a.kv_heads : kPackHeads;
  const uint32_t head = blockIdx.x / 8 % wide + blockIdx.y * kPackHeads, at = blockIdx.x / 8 / wide * 8 + blockIdx.x % 8;
  if (at >= a.n_blocks || head >= a.kv_heads) return;  // uniform
  uint32_t i = 0;
  for (uint32_t up = a.n; up - i > 1;) {  // the last sequence that begins at or before this block
    const uint32_t mid = (i + up) / 2;
    if (a.e[mid].block0 <= at) i = mid;
    else up = mid;
  }
  const uint32_t in = at - a.e[i].block0, first = in * kAttBlock, last = a.e[i].len - 1;
  const uint64_t width = (uint64_t)a.kv_heads * a.dim, block = (uint64_t)head * a.blocks + a.e[i].at + in;
  const uint32_t lane = threadIdx.x & 63, q = lane & 3, plane = 1024 * a.chunks;
  const uint64_t to = block * (4 * plane);
  uint32_t d[PIECES][4][4];  // digits: keys [16 tokens][plane], values [dim][plane]: a word each
#pragma unroll
  for (uint32_t j = 0; j < PIECES; j++) {
    // keys: lane 4 t + q has dims 4 q .. + 3 of tokens t, 16 + t ..;
    // values: lane 16 c + 4 g + t has tokens 16 t + 4 c .. + 3 of dims 4 g .. + 3
    const uint32_t piece = wave + j * waves, chunk = piece / 2, values = piece & 1;
    if (piece >= 2 * a.chunks) break;  // uniform
    const uint32_t dim0 = 16 * chunk + 4 * (values ? lane / 4 % 4 : q);
    uint32_t x[4][4];
    const uint32_t* from[4];
#pragma unroll
    for (uint32_t t = 0; t < 4; t++) {
      const uint32_t token = first + (values ? 16 * q + 4 * (lane / 16) + t : 16 * t + lane / 4);
      from[t] = (values ? v : k) + ((uint64_t)a.e[i].row + (token < last ? token : last)) * width + (uint64_t)head * a.dim;
    }
    if (a.dim % 4 == 0) {  // uniform
      const uint32_t at0 = dim0 < a.dim ? dim0 : 0;
      v4i_word w[4];
#pragma unroll
      for (uint32_t t = 0; t < 4; t++) w[t] = *(const v4i_word*)(from[t] + at0);
#pragma unroll
      for (uint32_t t = 0; t < 4; t++)
#pragma unroll
        for (int e = 0; e < 4; e++) x[t][e] = (uint32_t)w[t][e];
    } else {
#pragma unroll
      for (uint32_t t = 0; t < 4; t++)
#pragma unroll
        for (uint32_t e = 0; e < 4; e++) x[t][e] = from[t][dim0 + e < a.dim ? dim0 + e : 0];
    }
#pragma unroll
    for (uint32_t t = 0; t < 4; t++)
#pragma unroll
      for (uint32_t e = 0; e < 4; e++) x[t][e] = dim0 + e < a.dim ? digit_bytes(x[t][e]) : 0u;
    uint32_t high = 0;
#pragma unroll
    for (uint32_t t = 0; t < 4; t++) {
      const uint32_t of[4] = {values ? x[0][t] : x[t][0], values ? x[1][t] : x[t][1], values ? x[2][t] : x[t][2],
                              values ? x[3][t] : x[t][3]};
      transpose_bytes(of, d[j][t]);
      high |= d[j][t][1] | d[j][t][2] | d[j][t][3];
    }
    const uint32_t any = (uint32_t)__any(high != 0) << values;
    if (lane == 0) highs[wave] = j ? highs[wave] | any : any;
  }
  __syncthreads();
  uint32_t all = 0;
  if (lane < waves) all = highs[lane];  // every wave has a piece
  all = (uint32_t)__any(all & 1) | (uint32_t)__any(all >> 1) << 1;
#pragma unroll
  for (uint32_t j = 0; j < PIECES; j++) {
    const uint32_t piece = wave + j * waves, chunk = piece / 2, values = piece & 1;
    if (piece >= 2 * a.chunks) break;  // uniform
    const uint32_t planes = all >> values & 1 ? 4 : 1;
    // of a quad lane q takes the 16 bytes of token 16 q + lane / 4, or of dim 4 g + q
    int8_t* const out = (values ? vo + prompt_value(lane / 16, 16 * chunk + 4 * (lane / 4 % 4) + q)
                                : ko + prompt_key(16 * q + lane / 4, chunk)) + to;
#pragma unroll
    for (uint32_t p = 0; p < 4; p++) {
      if (p >= planes) break;
      uint32_t w[4] = {d[j][0][p], d[j][1][p], d[j][2][p], d[j][3][p]};
      quad_transpose(w);
      *(uint4*)(out + p * plane) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  if (threadIdx.x == 0) {
    upper[block] = all;
    volatile uint32_t* const word = mask + kMaskStride * (blockIdx.x % kPromptWords);
    if (all && !*word) *word = 1;
  }
}

// sum_g 256^g s[g] + offset (mod P) of a general score's digit sums, with 2^32 = 2.
// SHORT, up to 128 dims: the top digit of a balanced word is at most 64, so |s[0]|
// <= 2^21, |s[1]| <= 2^22, |s[2]| <= 3 2^21, |s[3]| <= 3 2^21, |s[4]| <= 2^22, |s[5]|
// <= 2^21, |s[6]| <= 2^19, and each of three 32-bit sums holds what has its unit
// (64-bit sums take twice the instructions).  Otherwise each by itself.
template <bool SHORT, class S>
__device__ __forceinline__ uint32_t prompt_score(const S& s, int v, int32_t offset) {
  auto turned = [](uint32_t x, int by) { return ((x << by) & P) | (x >> (31 - by)); };
  if constexpr (SHORT) {
    const uint32_t a = signed32_mod_p(s[0][v] + 2 * s[4][v] + 512 * s[5][v]);      // below 2^30 + 2^24
    const uint32_t b = signed32_mod_p(256 * s[1][v] + offset);                     // below 2^31: the offset is centered
    const uint32_t c = signed32_mod_p(s[2][v] + 2 * s[6][v] + 256 * s[3][v]);      // below 3 2^29 + 2^23
    return m31_add(m31_add(a, b), turned(c, 16));
  } else {
    uint32_t x = m31_add(signed32_mod_p(s[0][v]), signed32_mod_p(offset));
#pragma unroll
    for (int g = 1; g < 7; g++) x = m31_add(x, turned(signed32_mod_p(s[g][v]), g < 4 ? 8 * g : 8 * g - 31));
    return x;
  }
}

constexpr uint32_t kPromptCounters = 2;  // a launch's words of PromptArgs::counter
constexpr uint32_t kPromptSome = 1, kPromptAll = 2;
struct PromptArgs {
  const int8_t *k, *v;
  const uint32_t *q, *mask;
  uint32_t* clear;  // the mask once more, for the call's last launch, else none
  AttOut o;
  uint32_t blocks;  // of a kv head, all sequences'
  uint32_t n, kv_heads, group, dim, chunks;
  uint32_t offset, table_mask;
  const uint32_t* upper;  // the packing's, a word a block
  // todo: a word an item, whether the int8 kernel left it; counter: how many items the
  // other has taken, and whether it has some of them (kPromptSome, by todo) or all
  uint32_t items, general_items, *todo, *counter;
  struct {
    uint32_t item0, tiles;  // its first item of this launch, its tiles of rows (int8 kernel)
    uint32_t general0;      // its first item of the other kernel, whose tiles are `per` of these
    uint32_t len, at, row;  // tokens; its first block; its first row of q
  } e[kPromptSeqs];
};


// Weights of four scores, a byte each, from their table places g (bytes of
// bits 16 .. 19 of the scores; 10 .. 15 are 10): byte tables that v_perm_b32 looks
// up, eight entries at a time.  The weights are negated, so that eight powers of
// two fit a signed byte.
__device__ __forceinline__ uint32_t prompt_upper(uint32_t g) {  // 0xff for bytes of 8 and more
  // selector 5 is a byte of zero, 13 gives 0xff
  return __builtin_amdgcn_perm(0u, 0u, (g & 0x08080808u) | 0x05050505u);
}
// 2^(g - 3) for g = 3 .. 10, else 0; what is left: 2^g for g = 0 .. 2.
__device__ __forceinline__ uint32_t prompt_wide(uint32_t g, uint32_t upper) {
  const uint32_t below = __builtin_amdgcn_perm(0xf0f8fcfeu, 0xff000000u, g), above = __builtin_amdgcn_perm(0x80808080u, 0x8080c0e0u, g ^ 0x08080808u);
  return (above & upper) | (below & ~upper);
}
__device__ __forceinline__ uint32_t prompt_small(uint32_t g, uint32_t upper) {
  return __builtin_amdgcn_perm(0u, 0x00fcfeffu, g) & ~upper;
}
// 2^g for g = 0 .. 7, 2^(g - 8) for g = 8 .. 10.
__device__ __forceinline__ uint32_t prompt_low(uint32_t g, uint32_t upper) {
  return __builtin_amdgcn_perm(0x80c0e0f0u, 0xf8fcfeffu, g) & ~upper;
}
__device__ __forceinline__ uint32_t prompt_high(uint32_t g, uint32_t upper) {
  return __builtin_amdgcn_perm(0xfcfcfcfcu, 0xfcfcfeffu, g ^ 0x08080808u) & upper;
}
// Bits 16 .. 23 of four words, a byte each.
__device__ __forceinline__ uint32_t prompt_places(const uint32_t (&x)[4]) {
  return __builtin_amdgcn_perm(x[1], x[0], 0x0c0c0602u) | __builtin_amdgcn_perm(x[3], x[2], 0x06020c0cu);
}
// Tables of more than 2^20 entries have places past 15: 15 for them.
__device__ __forceinline__ uint32_t prompt_cap(uint32_t g) {
  uint32_t high = g & 0xf0f0f0f0u;
  high |= high >> 1;
  high |= high >> 2;
  high = (high >> 4) & 0x01010101u;  // whether any of a byte's bits 4 .. 7 is set
  return (g & 0x0f0f0f0fu) | ((high << 4) - high);
}
// Bytes of the tokens first .. first + 3 that are among the first `seen`.
__device__ __forceinline__ uint32_t prompt_seen(int left) { return left >= 4 ? ~0u : left <= 0 ? 0u : (1u << (8 * left)) - 1; }

// The end of a row's element: as att_finish, with the reciprocal of 2 z at hand.
__device__ __forceinline__ uint32_t prompt_mean(int64_t total, uint32_t z, double inv) {
  const uint64_t num = 2 * (uint64_t)(total < 0 ? -total : total) + z, den = 2 * (uint64_t)z;
  uint32_t r = (uint32_t)((double)num * inv);  // off by one at most: the quotient is at most 2^30
  const int64_t rest = (int64_t)(num - (uint64_t)r * den);
  r += rest < 0 ? -1 : rest >= (int64_t)den ? 1 : 0;
  return total < 0 ? m31_neg(r) : r;
}

// The same of int8-range values, from the negated total and -1 / z, to a word: the
// quotient is at most 128, |total| / z + 1/2 a multiple of 1 / 2 z, 2^-28 and more,
// and its error below 2^-37 (1 / z to 2^-45 by k_prompt_int8's step of Newton's, so
// 2^-38 of the quotient; prompt_end divides, to 2^-53), so 2^-30 more decides it; the
// conversion cuts towards zero.
__device__ __forceinline__ uint32_t prompt_mean(double negated, double inv) {
  const int32_t r = (int32_t)__builtin_fma(negated, inv, __builtin_copysign(0.5 + 0x1p-30, -negated));
  return umin32((uint32_t)r, (uint32_t)r + P);
}

// Four scores of a row, its tokens first .. first + 3: kept as words, 0 where they
// are not seen.
__device__ __forceinline__ void prompt_keep(const AttOut& o, uint64_t at, uint32_t first, uint32_t seen, const v4i& y,
                                            int32_t add) {
  if (seen == 0) return;  // no such row
  v4i_word x;
#pragma unroll
  for (int v = 0; v < 4; v++) x[v] = first + v < seen ? (int)signed32_mod_p(y[v] + add) : 0;
  if (first + 4 <= o.score_cols) {
    *(v4i_word*)(o.scores + at + first) = x;
  } else {
#pragma unroll
    for (int v = 0; v < 4; v++)
      if (first + v < o.score_cols) o.scores[at + first + v] = (uint32_t)x[v];
  }
}
// Scores behind a wave's last block (`mine` of them) are cleared.
template <int R>
__device__ __forceinline__ void prompt_clear(const PromptArgs& a, uint32_t i, uint32_t kvh, uint32_t row0, uint32_t mine) {
  const uint32_t rows = a.e[i].len * a.group, end = row0 + 16 * R < rows ? row0 + 16 * R : rows;
  for (uint32_t row = row0; row < end; row++) {
    const uint32_t token = row / a.group;
    const uint64_t at = (((uint64_t)a.e[i].row + token) * a.kv_heads + kvh) * a.group + (row - token * a.group);
    for (uint64_t t = (uint64_t)mine * kAttBlock + (threadIdx.x & 63); t < a.o.score_cols; t += 64) a.o.scores[at * a.o.score_cols + t] = 0;
  }
}
// The end of a wave's rows: acc and z as the tiles leave them.
template <int NP, int DT, int R, bool TRACE>
__device__ __forceinline__ void prompt_end(const PromptArgs& a, uint32_t i, uint32_t kvh, uint32_t row0, uint32_t mine,
                                           const v4i (&acc)[R][4 * DT][NP + 1], const int32_t (&z)[R][2]) {
  constexpr int CH = 4 * DT, NV = NP + 1;
  const uint32_t lane = threadIdx.x & 63, col = lane & 15, quarter = lane >> 4;
  const uint32_t rows = a.e[i].len * a.group;
  auto whole_total = [&](int r, int d, int v) {
    if constexpr (NP == 1) return -((int64_t)acc[r][d][0][v] + ((int64_t)acc[r][d][1][v] << 3));
    int64_t total = 0;
#pragma unroll
    for (int g = 0; g < NV; g++) total -= (int64_t)acc[r][d][g][v] << (8 * g);
    return total;
  };
#pragma unroll
  for (int r = 0; r < R; r++) {
    uint32_t zc = (uint32_t)-(NP == 1 ? z[r][0] + 8 * z[r][1] : z[r][0] + 256 * z[r][1]);
    zc += __shfl_xor(zc, 16);
    zc += __shfl_xor(zc, 32);
#pragma unroll
    for (int v = 0; v < 4; v++) {
      const uint32_t row = row0 + 16 * r + 4 * quarter + v, zr = __shfl(zc, 4 * quarter + v);
      if (row >= rows) continue;
      const uint32_t token = row / a.group;
      const uint64_t at = (((uint64_t)a.e[i].row + token) * a.kv_heads + kvh) * a.group + (row - token * a.group);
      if (a.o.sums && col == 0) a.o.sums[at] = shift16(m31_from_u32(zr));
      const double inv = (NP == 1 ? -1.0 : 0.5) / zr;
#pragma unroll
      for (int d = 0; d < (int)CH; d++) {
        const bool there = 16 * d + col < a.dim;
        if constexpr (NP == 1) {
          const double total = __builtin_fma(8.0, (double)acc[r][d][1][v], (double)acc[r][d][0][v]);  // negated
          const uint32_t mean = prompt_mean(total, inv);
          if (there) a.o.out[at * a.dim + 16 * d + col] = mean;
        } else {
          const uint32_t mean = prompt_mean(whole_total(r, d, v), zr, inv);
          if (there) a.o.out[at * a.dim + 16 * d + col] = mean;
        }
      }
      if (TRACE && a.o.weighted) {
#pragma unroll
        for (int d = 0; d < (int)CH; d++)
          if (16 * d + col < a.dim) a.o.weighted[at * a.dim + 16 * d + col] = shift16(signed_mod_p(whole_total(r, d, v)));
      }
    }
  }
  if (TRACE && a.o.scores && row0 < rows) prompt_clear<R>(a, i, kvh, row0, mine);
}
// A workgroup's W waves have R tiles of 16 rows each and take the blocks in step:
// keys and values of a block go through LDS, each on its way from memory while
// the other is used.
template <int NP, int NQ, int DT, int R, int W, bool TRACE>
__device__ __forceinline__ void prompt_tile(const PromptArgs& a, v4i* __restrict__ lk, v4i* __restrict__ lv, uint32_t i,
                                            uint32_t kvh, uint32_t tile0, uint32_t row0, const v4i (&qd)[R][DT][NQ]) {
  constexpr int NG = NP + NQ - 1, NV = NP + 1;  // NP = 1: sums of the small and of the wide weights
  constexpr uint32_t CH = 4 * DT;               // chunks of 16 dims in LDS
  constexpr int ND = (int)((CH * NP + W - 1) / W);  // 1 KB pieces of keys, and of values, a wave copies
  const uint32_t lane = threadIdx.x & 63, col = lane & 15, quarter = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t len = a.e[i].len, rows = len * a.group, plane = 1024 * a.chunks;
  const uint32_t tile_end = tile0 + 16 * R * W < rows ? tile0 + 16 * R * W : rows;
  const uint32_t wave_end = row0 + 16 * R < rows ? row0 + 16 * R : rows;
  const uint32_t blocks = ((tile_end - 1) / a.group + kAttBlock) / kAttBlock;
  // this wave's: none past its last row's end, whole ones up to its first row's
  const uint32_t mine = row0 < rows ? ((wave_end - 1) / a.group + kAttBlock) / kAttBlock : 0;
  const uint32_t whole = row0 < rows ? (row0 / a.group + 1) / kAttBlock : 0;
  uint32_t seen[R];  // tokens that row row0 + 16 r + col sees
#pragma unroll
  for (int r = 0; r < R; r++) {
    const uint32_t row = row0 + 16 * r + col;
    seen[r] = row < rows ? row / a.group + 1 : 0;
  }
  const uint64_t block0 = (uint64_t)kvh * a.blocks + a.e[i].at, base = block0 * (4 * plane) + 16 * lane;
  uint32_t from[ND];  // of this wave's pieces; chunks past the last are the last one again (the query is zero there)
#pragma unroll
  for (int j = 0; j < ND; j++) {
    const uint32_t piece = wave * ND + j, chunk = piece % CH < a.chunks ? piece % CH : a.chunks - 1;
    from[j] = piece < CH * NP ? piece / CH * plane + 1024 * chunk : 0;
  }
  // the upper planes of keys or values that have none are zero and not in memory; the
  // word that tells goes a block ahead
  uint32_t upper = NP > 1 ? a.upper[block0] : 0;
  auto load = [&](v4i (&in)[ND], const int8_t* m, uint32_t b, uint32_t bit) {  // past the last block: again, unused
    const int8_t* const block = m + base + (uint64_t)(b < blocks ? b : blocks - 1) * (4 * plane);
    const bool have = __builtin_amdgcn_readfirstlane((int)upper) >> bit & 1;
#pragma unroll
    for (int j = 0; j < ND; j++) {
      if (NP == 1 || wave * ND + j < CH || have) in[j] = *(const v4i*)(block + from[j]);  // uniform
      else in[j] = v4i{0, 0, 0, 0};
    }
  };
  auto put = [&](const v4i (&in)[ND], v4i* to) {
#pragma unroll
    for (int j = 0; j < ND; j++)
      if (ND * W == CH * NP || wave * ND + j < CH * NP) to[(wave * ND + j) * 64 + lane] = in[j];
  };
  v4i acc[R][CH][NV];
#pragma unroll
  for (int r = 0; r < R; r++)
#pragma unroll
    for (int d = 0; d < (int)CH; d++)
#pragma unroll
      for (int g = 0; g < NV; g++) acc[r][d][g] = v4i{0, 0, 0, 0};
  int32_t z[R][2] = {};
  const int32_t off = a.offset > P / 2 ? (int32_t)(a.offset - P) : (int32_t)a.offset;
  const uint32_t place_mask = (a.table_mask >> 16) * 0x01010101u;
  const bool many = a.table_mask >> 20 != 0;
  v4i in[ND];
  load(in, a.k, 0, 0);
  put(in, lk);
#pragma unroll 1
  for (uint32_t b = 0; b < blocks; b++) {
    __syncthreads();  // the keys are there, the values' place is free
    load(in, a.v, b, 1);
    if (NP > 1) upper = a.upper[block0 + (b + 1 < blocks ? b + 1 : b)];
    uint32_t w0[R][4], w1[R][4];  // NP = 1: small and wide weights; else the digits base 256
    bool some_small = false;
    const bool busy = b < mine;
    if (busy) {
#pragma unroll
      for (int t = 0; t < 4; t++) {
        v4i sc[R][NG];
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
          for (int g = 0; g < NG; g++) {
            const int init = g == 0 && NG < 7 ? off : 0;
            sc[r][g] = v4i{init, init, init, init};
          }
#pragma unroll
        for (int s = 0; s < DT; s++)
#pragma unroll
          for (int p = 0; p < NP; p++) {
            const v4i kd = lk[(p * CH + 4 * s + quarter) * 64 + 16 * t + col];
#pragma unroll
            for (int r = 0; r < R; r++)
#pragma unroll
              for (int g = 0; g < NQ; g++)
                sc[r][p + g] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kd, qd[r][s][g], sc[r][p + g], 0, 0, 0);
          }
#pragma unroll
        for (int r = 0; r < R; r++) {
          uint32_t x[4];
#pragma unroll
          for (int v = 0; v < 4; v++) {
            if constexpr (NG == 4) {
              // |sc[g]| <= 2^22 and the offset: pairs in 32 bits, the upper one turned by 16 of 31 bits
              const uint32_t low = signed32_mod_p(sc[r][0][v]), mid = signed32_mod_p(sc[r][1][v] << 8);
              const uint32_t high = signed32_mod_p(sc[r][2][v] + (sc[r][3][v] << 8));
              x[v] = m31_add(m31_add(low, mid), ((high << 16) & P) | (high >> 15));
            } else {
              x[v] = prompt_score<(DT <= 2)>(sc[r], v, off);
            }
          }
          if (TRACE && a.o.scores) {
            const uint32_t row = row0 + 16 * r + col, token = row / a.group;
            const uint64_t at = ((((uint64_t)a.e[i].row + token) * a.kv_heads + kvh) * a.group + (row - token * a.group)) * a.o.score_cols;
            prompt_keep(a.o, at, b * kAttBlock + 16 * t + 4 * quarter, seen[r], v4i{(int)x[0], (int)x[1], (int)x[2], (int)x[3]}, 0);
          }
          w0[r][t] = prompt_places(x) & place_mask;
        }
      }
      {
        if (many) {  // uniform
#pragma unroll
          for (int r = 0; r < R; r++)
#pragma unroll
            for (int t = 0; t < 4; t++) w0[r][t] = prompt_cap(w0[r][t]);
        }
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
          for (int t = 0; t < 4; t++) {
            const uint32_t g = w0[r][t], upper = prompt_upper(g);
            w0[r][t] = NP == 1 ? prompt_small(g, upper) : prompt_low(g, upper);
            w1[r][t] = NP == 1 ? prompt_wide(g, upper) : prompt_high(g, upper);
          }
        if (b >= whole) {  // uniform: tokens that a row does not see have no weight
#pragma unroll
          for (int r = 0; r < R; r++)
#pragma unroll
            for (int t = 0; t < 4; t++) w0[r][t] &= prompt_seen((int)(seen[r] - (b * kAttBlock + 16 * t + 4 * quarter)));
        }
        uint32_t any_small = 0;
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
          for (int t = 0; t < 4; t++) {
            any_small |= w0[r][t];
            z[r][0] = __builtin_amdgcn_sdot4((int)w0[r][t], 0x01010101, z[r][0], false);
          }
        some_small = __any(any_small != 0);
      }
      if (b >= whole) {
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
          for (int t = 0; t < 4; t++) w1[r][t] &= prompt_seen((int)(seen[r] - (b * kAttBlock + 16 * t + 4 * quarter)));
      }
#pragma unroll
      for (int r = 0; r < R; r++)
#pragma unroll
        for (int t = 0; t < 4; t++) z[r][1] = __builtin_amdgcn_sdot4((int)w1[r][t], 0x01010101, z[r][1], false);
    }
    put(in, lv);
    __syncthreads();  // the values are there, the keys' place is free
    load(in, a.k, b + 1, 0);
    if (busy) {
      auto product = [&](int r, int d, int g, const uint32_t (&w)[4], const v4i& vd) {
        const v4i wd = {(int)w[0], (int)w[1], (int)w[2], (int)w[3]};
        acc[r][d][g] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wd, vd, acc[r][d][g], 0, 0, 0);
      };
      if constexpr (NP == 1) {
#pragma unroll
        for (int d = 0; d < (int)CH; d++) {
          const v4i vd = lv[d * 64 + lane];
#pragma unroll
          for (int r = 0; r < R; r++) product(r, d, 1, w1[r], vd);
        }
        if (some_small) {
#pragma unroll
          for (int d = 0; d < (int)CH; d++) {
            const v4i vd = lv[d * 64 + lane];
#pragma unroll
            for (int r = 0; r < R; r++) product(r, d, 0, w0[r], vd);
          }
        }
      } else {
#pragma unroll
        for (int d = 0; d < (int)CH; d++)
#pragma unroll
          for (int p = 0; p < NP; p++) {
            const v4i vd = lv[(p * CH + d) * 64 + lane];
#pragma unroll
            for (int r = 0; r < R; r++) {
              product(r, d, p, w0[r], vd);
              product(r, d, p + 1, w1[r], vd);
            }
          }
      }
    }
    put(in, lk);
  }
  prompt_end<NP, DT, R, TRACE>(a, i, kvh, row0, mine, acc, z);
}
// The four digit planes of a wave's R tiles of queries.
template <int DT, int R>
__device__ __forceinline__ void prompt_query(const PromptArgs& a, uint32_t i, uint32_t kvh, uint32_t row0, v4i (&qd)[R][DT][4]) {
  const uint32_t lane = threadIdx.x & 63, col = lane & 15, quarter = lane >> 4, rows = a.e[i].len * a.group;
#pragma unroll
  for (int r = 0; r < R; r++) {
    const uint32_t here = row0 + 16 * r + col, row = here < rows ? here : rows - 1, token = row / a.group;
    const uint32_t* const from =
        a.q + ((((uint64_t)a.e[i].row + token) * a.kv_heads + kvh) * a.group + (row - token * a.group)) * a.dim;
    v4i w[DT][4];
    if (a.dim % 4 == 0) {  // uniform
#pragma unroll
      for (int s = 0; s < DT; s++)
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) {
          const uint32_t d = 64 * s + 16 * quarter + 4 * j;
          w[s][j] = *(const v4i_word*)(from + (d < a.dim ? d : 0));
        }
    } else {
#pragma unroll
      for (int s = 0; s < DT; s++)
#pragma unroll
        for (uint32_t j = 0; j < 4; j++)
#pragma unroll
          for (uint32_t t = 0; t < 4; t++) {
            const uint32_t d = 64 * s + 16 * quarter + 4 * j + t;
            w[s][j][t] = (int)from[d < a.dim ? d : 0];
          }
    }
#pragma unroll
    for (int s = 0; s < DT; s++)
#pragma unroll
      for (uint32_t j = 0; j < 4; j++) {
        uint32_t x[4], out[4];
#pragma unroll
        for (uint32_t t = 0; t < 4; t++) x[t] = 64 * s + 16 * quarter + 4 * j + t < a.dim ? digit_bytes((uint32_t)w[s][j][t]) : 0u;
        transpose_bytes(x, out);
#pragma unroll
        for (int p = 0; p < 4; p++) qd[r][s][p][j] = (int)out[p];
      }
  }
}
// Rows of a wave: token and head of row x counted from the first (x below 2^17), by
// a product with 1 / group: x / group is 0.5 / group away from the next whole
// number, more than the product's error.
struct PromptRows {
  uint32_t token0, head0, group;  // of the first row
  float inv;
  __device__ __forceinline__ PromptRows(uint32_t row0, uint32_t group_) : group(group_), inv(1.0f / (float)group_) {
    token0 = row0 / group_;
    head0 = row0 - token0 * group_;
  }
  __device__ __forceinline__ void at(uint32_t x, uint32_t& token, uint32_t& head) const {  // token from token0 on
    x += head0;
    token = (uint32_t)(((float)x + 0.5f) * inv);
    head = x - token * group;
  }
};

// One pass over the blocks of a wave's R tiles of 16 rows, int8-range words on all
// sides: sums of the values by the wide weights (SMALL: by the small ones).  A
// block's keys and values come straight into LDS while the block before it is
// used, a wave's share of them a piece of 1 KB at a time: two halves of LDS, which
// are arrays of their own, so that a read of one does not wait for the other; one
// barrier a block.  The blocks where a small weight was met are marked in `marks`, a
// bit each, and the small weights' pass visits those only.
template <int DT, int R, int W, bool SMALL, bool TRACE>
struct PromptPass {
  static constexpr uint32_t CH = 4 * DT;
  const PromptArgs& a;
  const int8_t *k, *v;  // block 0's piece of this wave
  uint32_t i, kvh, row0, wave, lane, blocks, mine, whole;
  const uint32_t (&seen)[R];  // tokens that row 16 r + lane % 16 of the wave sees
  const v4i (&qd)[R][DT];
  v4i (&acc)[R][CH];
  int32_t (&z)[R];
  uint32_t* marks;

  __device__ __forceinline__ void load(uint32_t b, v4i* keys, v4i* values) const {
    const uint64_t at = (uint64_t)b * (4 * 1024 * a.chunks);
#pragma unroll
    for (uint32_t j = 0; j < CH / W; j++) {
      const uint32_t piece = wave * (CH / W) + j;
      if (piece >= a.chunks) continue;  // uniform; not multiplied by anything, or not stored
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(k + at + 1024 * j),
                                       (__attribute__((address_space(3))) void*)(keys + piece * 64), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(v + at + 1024 * j),
                                       (__attribute__((address_space(3))) void*)(values + piece * 64), 16, 0, 0);
    }
  }
  // The loads into LDS have arrived (they are not among what a barrier waits for)
  // and all waves are here.
  __device__ __forceinline__ void arrive() const {
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
    __syncthreads();
  }
  __device__ __forceinline__ uint32_t sight(uint32_t b, int r, int t) const {
    return prompt_seen((int)(seen[r] - (b * kAttBlock + 16 * t + 4 * (lane >> 4))));
  }
  // the first marked block from b on, or `blocks`
  __device__ __forceinline__ uint32_t marked(uint32_t b) const {
    while (b < blocks) {
      const uint32_t word = (uint32_t)__builtin_amdgcn_readfirstlane((int)marks[b / 32]) >> (b % 32);
      if (word) return min(b + (uint32_t)__builtin_ctz(word), blocks);
      b = (b / 32 + 1) * 32;
    }
    return blocks;
  }
  __device__ __forceinline__ void block(uint32_t b, uint32_t next, const v4i* __restrict__ keys, const v4i* __restrict__ values,
                                        v4i* __restrict__ next_keys, v4i* __restrict__ next_values) {
    arrive();
    if (next < blocks) load(next, next_keys, next_values);
    if (b >= mine) return;  // uniform in the wave
    const uint32_t col = lane & 15, quarter = lane >> 4;
    // scores less `low` 2^16, not reduced: below 0 where the place is below `low` or the score negative
    const uint32_t places = a.table_mask >> 16, low = places < 8 ? 0 : 3;
    const int32_t start = (a.offset > P / 2 ? (int32_t)(a.offset - P) : (int32_t)a.offset) - (int32_t)(low << 16);
    v4i y[R][4];
#pragma unroll
    for (int t = 0; t < 4; t++) {
#pragma unroll
      for (int r = 0; r < R; r++) y[r][t] = v4i{start, start, start, start};
#pragma unroll
      for (int s = 0; s < DT; s++) {
        const v4i kd = keys[(4 * s + quarter) * 64 + 16 * t + col];
#pragma unroll
        for (int r = 0; r < R; r++) y[r][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kd, qd[r][s], y[r][t], 0, 0, 0);
      }
    }
    if (TRACE && !SMALL && a.o.scores) {
      const uint32_t rows = a.e[i].len * a.group;
#pragma unroll
      for (int r = 0; r < R; r++) {
        const uint32_t row = row0 + 16 * r + col < rows ? row0 + 16 * r + col : rows - 1, token = row / a.group;
        const uint64_t at = ((((uint64_t)a.e[i].row + token) * a.kv_heads + kvh) * a.group + (row - token * a.group)) * a.o.score_cols;
#pragma unroll
        for (int t = 0; t < 4; t++) prompt_keep(a.o, at, b * kAttBlock + 16 * t + 4 * quarter, seen[r], y[r][t], low << 16);
      }
    }
    uint32_t w[R][4], most[R] = {}, left = 0;
    if (!SMALL) {
#pragma unroll
      for (int r = 0; r < R; r++)
#pragma unroll
        for (int t = 0; t < 4; t++) most[r] = max(max(most[r], max((uint32_t)y[r][t][0], (uint32_t)y[r][t][1])), max((uint32_t)y[r][t][2], (uint32_t)y[r][t][3]));
#pragma unroll
      for (int r = 1; r < R; r++) most[0] = max(most[0], most[r]);
    }
    if (!SMALL && !__any(most[0] > a.table_mask - (low << 16))) {  // all places at `low` and above: cut off at 10
      const uint32_t top = low ? 0x7ffffu : 0xffffffu;
#pragma unroll
      for (int r = 0; r < R; r++)
#pragma unroll
        for (int t = 0; t < 4; t++) {
          uint32_t x[4];
#pragma unroll
          for (int j = 0; j < 4; j++) x[j] = min((uint32_t)y[r][t][j], top);
          w[r][t] = __builtin_amdgcn_perm(0x80c0e0f0u, 0xf8fcfeffu, prompt_places(x));
        }
    } else {
      const uint32_t place_mask = places * 0x01010101u;
#pragma unroll
      for (int r = 0; r < R; r++)
#pragma unroll
        for (int t = 0; t < 4; t++) {
          uint32_t x[4];
#pragma unroll
          for (int j = 0; j < 4; j++) x[j] = signed32_mod_p(y[r][t][j] + (int32_t)(low << 16));
          uint32_t g = prompt_places(x) & place_mask;
          if (places > 15) g = prompt_cap(g);  // uniform
          const uint32_t upper = prompt_upper(g);
          if (low == 0) {  // uniform: places 0 .. 7, no other weights
            w[r][t] = prompt_low(g, upper);
          } else if (SMALL) {
            w[r][t] = prompt_small(g, upper);
          } else {
            w[r][t] = prompt_wide(g, upper);
            left |= prompt_small(g, upper) & sight(b, r, t);
          }
        }
    }
    if (!SMALL && __any(left != 0) && lane == 0) atomicOr(&marks[b / 32], 1u << (b % 32));
    if (b >= whole) {  // uniform: tokens that a row does not see have no weight
#pragma unroll
      for (int r = 0; r < R; r++)
#pragma unroll
        for (int t = 0; t < 4; t++) w[r][t] &= sight(b, r, t);
    }
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
      for (int t = 0; t < 4; t++) z[r] = __builtin_amdgcn_sdot4((int)w[r][t], 0x01010101, z[r], false);
#pragma unroll
    for (int d = 0; d < (int)CH; d++) {
      const v4i vd = values[d * 64 + lane];
#pragma unroll
      for (int r = 0; r < R; r++) {
        const v4i wd = {(int)w[r][0], (int)w[r][1], (int)w[r][2], (int)w[r][3]};
        acc[r][d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wd, vd, acc[r][d], 0, 0, 0);
      }
    }
  }
  // k0 and v0 hold the first block (on its way)
  __device__ __forceinline__ void run(v4i* k0, v4i* v0, v4i* k1, v4i* v1) {
#pragma unroll
    for (int r = 0; r < R; r++) {
#pragma unroll
      for (int d = 0; d < (int)CH; d++) acc[r][d] = v4i{0, 0, 0, 0};
      z[r] = 0;
    }
    uint32_t b = SMALL ? marked(0) : 0;
#pragma unroll 1
    while (b < blocks) {
      const uint32_t second = SMALL ? marked(b + 1) : b + 1;
      block(b, second, k0, v0, k1, v1);
      if (second >= blocks) break;
      b = SMALL ? marked(second + 1) : second + 1;
      block(second, b, k1, v1, k0, v0);
    }
  }
};

// The int8 kernel.  A workgroup's W waves have R tiles of 16 rows each.
template <int DT, int R, int W, int OCC, bool TRACE>
static __global__ void __launch_bounds__(64 * W, OCC) k_prompt_int8(PromptArgs a) {
  constexpr uint32_t CH = 4 * DT, KB = CH * 64;
  __shared__ v4i k0[KB], v0[KB], k1[KB], v1[KB];
  __shared__ uint32_t general[W], marks[(kMaxPrompt + kAttBlock) / kAttBlock / 32 + 1];
  const uint32_t flagged = prompt_mask(a.mask);
  const uint32_t lane = threadIdx.x & 63, col = lane & 15, quarter = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (uint32_t w = threadIdx.x; w < sizeof(marks) / 4; w += 64 * W) marks[w] = 0;
  const uint32_t item = blockIdx.x;
  uint32_t i = 0;
  for (uint32_t up = a.n; up - i > 1;) {  // the last sequence that begins at or before this item
    const uint32_t mid = (i + up) / 2;
    if (a.e[mid].item0 <= item) i = mid;
    else up = mid;
  }
  const uint32_t in = item - a.e[i].item0, turn = in / a.kv_heads, tile = a.e[i].tiles - 1 - turn, kvh = in - turn * a.kv_heads;
  const uint32_t tile0 = tile * (16 * R * W), row0 = tile0 + wave * (16 * R), rows = a.e[i].len * a.group;
  const uint32_t first = row0 < rows ? row0 : rows - 1;  // a wave without rows has the last one again, unused
  const PromptRows place(first, a.group);
  // word offsets of rows from `origin`: 2^32 bytes are enough for a tile's (4096 kv heads of 256, 256 rows)
  const uint64_t origin = (((uint64_t)a.e[i].row + place.token0) * a.kv_heads + kvh) * (uint64_t)a.group * a.dim;
  const uint32_t token_words = a.kv_heads * a.group * a.dim;

  // the queries' words, whole rows at a time, to bytes in the operand order through
  // LDS (the second half of the blocks' place), a wave 16 R rows in its share of it.
  // c(x) mod 2^31 is x, or x + 1 for a negative number: its low byte, where the rest
  // is the byte's sign
  static_assert(2 * KB * 16 >= W * R * CH * 256, "the queries' place");
  int8_t* const mine_q = (int8_t*)(wave < W / 2 ? k1 : v1) + (wave % (W / 2)) * (R * CH * 256);
  uint32_t high = 0;
  constexpr uint32_t VR = 16 * DT, N = 16 * VR / 64;  // vectors of four words of a row; a lane's of 16 rows
  const uint32_t d = lane % VR * 4;
  v4i w[R][N];
#pragma unroll
  for (int r = 0; r < R; r++)
#pragma unroll
    for (uint32_t j = 0; j < N; j++) {
      const uint32_t x = 16 * r + j * (64 / VR) + lane / VR;
      uint32_t token, head;
      place.at(first + x < rows ? x : rows - 1 - first, token, head);
      const uint32_t* const from = a.q + origin + (uint64_t)token * token_words + head * a.dim;
      if (a.dim % 4 == 0) {  // uniform
        w[r][j] = *(const v4i_word*)(from + (d < a.dim ? d : 0));
      } else {
#pragma unroll
        for (uint32_t t = 0; t < 4; t++) w[r][j][t] = (int)from[d + t < a.dim ? d + t : 0];
      }
    }
  if (__any(flagged != 0)) {  // uniform: the other kernel's
    if (item == 0 && threadIdx.x == 0) a.counter[1] = kPromptAll;
    return;
  }
#pragma unroll
  for (int r = 0; r < R; r++)
#pragma unroll
    for (uint32_t j = 0; j < N; j++) {
      const uint32_t x = j * (64 / VR) + lane / VR;
      uint32_t b[4];
#pragma unroll
      for (uint32_t t = 0; t < 4; t++) {
        b[t] = (uint32_t)w[r][j][t];
        b[t] += b[t] >> 30;
        if (d + t >= a.dim) b[t] = 0;
        high |= b[t] + 128;
      }
      // chunk by chunk 16 rows of 16 bytes, in another order in each chunk: neither side meets its own banks
      *(uint32_t*)(mine_q + ((r * CH + d / 16) * 16 + (x ^ (d / 16 & 15))) * 16 + d % 16) = pick_bytes<0>(b);
    }
  high &= 0x7fffff00u;
  const uint64_t block0 = ((uint64_t)kvh * a.blocks + a.e[i].at) * (4 * 1024 * a.chunks) + 1024 * wave * (CH / W) + 16 * lane;
  const uint32_t tile_end = tile0 + 16 * R * W < rows ? tile0 + 16 * R * W : rows;
  const uint32_t blocks = ((tile_end - 1) / a.group + kAttBlock) / kAttBlock;
  uint32_t seen[R], last_seen;
  {
    uint32_t token, head;
#pragma unroll
    for (int r = 0; r < R; r++) {
      place.at(16 * r + col, token, head);
      seen[r] = row0 + 16 * r + col < rows ? place.token0 + token + 1 : 0;
    }
    place.at(first + 16 * R < rows ? 16 * R - 1 : rows - 1 - first, token, head);
    last_seen = place.token0 + token + 1;
  }
  // blocks up to this wave's last row's end, and whole ones up to its first row's
  const uint32_t my_blocks = (uint32_t)__builtin_amdgcn_readfirstlane((int)((last_seen + kAttBlock - 1) / kAttBlock));
  const uint32_t whole = (uint32_t)__builtin_amdgcn_readfirstlane((int)((place.token0 + 1) / kAttBlock));
  v4i qd[R][DT], acc[R][CH];
  int32_t z[R];
  auto pass = [&](auto small) {
    constexpr bool SMALL = decltype(small)::value;
    return PromptPass<DT, R, W, SMALL, TRACE>{a, a.k + block0, a.v + block0, i, kvh, row0, wave, lane, blocks,
                                              row0 < rows ? my_blocks : 0u, whole, seen, qd, acc, z, marks};
  };
  auto wide = pass(std::false_type{});
  wide.load(0, k0, v0);
  {
    const bool any_high = __any(high != 0);
    if (lane == 0) general[wave] = any_high;
  }
  wave_exchange();
#pragma unroll
  for (int r = 0; r < R; r++)
#pragma unroll
    for (int s = 0; s < DT; s++) {
      const uint32_t chunk = 4 * s + quarter;
      qd[r][s] = *(const v4i*)(mine_q + ((r * CH + chunk) * 16 + (col ^ (chunk & 15))) * 16);
    }
  wide.arrive();
  uint32_t some = 0;
#pragma unroll
  for (int w = 0; w < W; w++) some |= general[w];
  if (threadIdx.x == 0) {
    a.todo[item] = some;
    if (some) a.counter[1] = kPromptSome;
  }
  if (some) return;  // uniform: queries of four planes are the other kernel's
  wide.run(k0, v0, k1, v1);
  __syncthreads();
  const uint32_t first_marked = wide.marked(0);
  const bool again = first_marked < blocks;

  // the ends: a lane has rows 16 r + 4 quarter + v, dims 16 d + col
  const WitBuffer out = wit_buffer(a.o.out, origin, ~0ull);
  uint32_t at[R][4];  // byte offsets from origin; none for rows that are not there
#pragma unroll
  for (int r = 0; r < R; r++)
#pragma unroll
    for (int v = 0; v < 4; v++) {
      const uint32_t x = 16 * r + 4 * quarter + v;
      uint32_t token, head;
      place.at(x, token, head);
      at[r][v] = row0 + x < rows ? 4 * (token * token_words + head * a.dim + col) : kOutside;
    }
  uint32_t zs[R];
  auto negate = [&](uint32_t by) {
#pragma unroll
    for (int r = 0; r < R; r++) {
      uint32_t s = (uint32_t)-z[r] * by;
      s += __shfl_xor(s, 16);
      s += __shfl_xor(s, 32);
      zs[r] = by == 1 && again ? zs[r] + s : s;
    }
  };
  const uint32_t unit = a.table_mask >> 19 ? 8 : 1;  // of the wide weights
  negate(unit);
  if (again) {  // small weights too: the wide ones' sums wait in the output
#pragma unroll
    for (int d = 0; d < (int)CH; d++)
#pragma unroll
      for (int r = 0; r < R; r++)
#pragma unroll
        for (int v = 0; v < 4; v++)
          if (16 * d + col < a.dim) wit_write(out, at[r][v] == kOutside ? kOutside : at[r][v] + 64 * d, (uint32_t)acc[r][d][v]);
    auto rest = pass(std::true_type{});
    rest.load(first_marked, k0, v0);  // all waves are past the loop
    rest.run(k0, v0, k1, v1);
    negate(1);
  }
  uint32_t zv[R][4];
  double inv[R][4];
#pragma unroll
  for (int r = 0; r < R; r++)
#pragma unroll
    for (int v = 0; v < 4; v++) {
      zv[r][v] = __shfl(zs[r], 4 * quarter + v);
      // 1 / z to 2^-45 by a step of Newton's from the reciprocal's 2^-23 or better
      const double zd = zv[r][v], guess = __builtin_amdgcn_rcp(zd);
      inv[r][v] = -__builtin_fma(guess, __builtin_fma(-zd, guess, 1.0), guess);
      if (a.o.sums && col == 0 && at[r][v] != kOutside) {
        uint32_t token, head;
        place.at(16 * r + 4 * quarter + v, token, head);
        a.o.sums[(((uint64_t)a.e[i].row + place.token0 + token) * a.kv_heads + kvh) * a.group + head] = shift16(m31_from_u32(zv[r][v]));
      }
    }
#pragma unroll
  for (int d = 0; d < (int)CH; d++) {
    const bool there = 16 * d + col < a.dim;
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
      for (int v = 0; v < 4; v++) {
        const uint32_t to = there && at[r][v] != kOutside ? at[r][v] + 64 * d : kOutside;
        double total;
        if (again) total = __builtin_fma((double)unit, (double)(int32_t)wit_read(out, to), (double)acc[r][d][v]);
        else total = (double)unit * (double)acc[r][d][v];
        if (TRACE && a.o.weighted && to != kOutside)
          a.o.weighted[origin + to / 4] = shift16(signed_mod_p(-(int64_t)total));
        wit_write(out, to, prompt_mean(total, inv[r][v]));
      }
  }
  if (TRACE && a.o.scores && row0 < rows)  // behind the last block they are cleared
    prompt_clear<R>(a, i, kvh, row0, wide.mine);
}
// Words that are not int8-range: keys or values (by the packing's mask), or the
// queries of an item (a.todo, by the int8 kernel; PER of its items are one here).  No more
// workgroups than fit at once: the items are taken in turn, the longest first, and
// with nothing to do the launch is short (4.7 us; 7.5 with a workgroup for each of 2432
// items).  Items of one kv head for the workgroups of an XCD gain nothing (1501 general
// tokens, 40 heads on 8 x 128: the same either way).  Those tokens take 180 us here
// where it runs again and again (203 in the first few dozen calls under a tracer, when
// the clock is lower), 7.7 in the packing and 6 in the int8 kernel; the call 191 without
// a tracer.  The matrix cores are busy a third of the cycles: a wave holds the five digit
// sums of all dims, and registers spill (116 at up to 128 dims, 810 above; with traces 247
// and 899).  The mask is the int8 kernel's to
// read; the last launch of a call zeroes it, so that a graph of one prompt, whose
// replays all have the same mask, does not find it set by general words of an earlier
// one (1500 int8 tokens, 16 heads of 128: 46 us, and 176 for every replay behind such).
template <int DT, int R, int W, int OCC, uint32_t PER, bool TRACE>
static __global__ void __launch_bounds__(64 * W, OCC) k_prompt(PromptArgs a) {
  __shared__ v4i lk[4 * 4 * DT * 64], lv[4 * 4 * DT * 64];
  __shared__ uint32_t taken;
  const uint32_t left = (uint32_t)__builtin_amdgcn_readfirstlane((int)a.counter[1]);
  if (!left) return;  // uniform
  const bool flagged = left == kPromptAll;
  if (flagged && a.clear && blockIdx.x == 0 && threadIdx.x < kPromptWords) a.clear[kMaskStride * threadIdx.x] = 0;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t item = blockIdx.x;
#pragma unroll 1
  for (;; item += gridDim.x) {
    if (flagged) {
      if (threadIdx.x == 0) taken = atomicAdd(a.counter, 1u);
      __syncthreads();
      item = taken;
    }
    if (item >= a.general_items) return;  // uniform
    uint32_t i = 0;
    for (uint32_t up = a.n; up - i > 1;) {  // the last sequence that begins at or before this item
      const uint32_t mid = (i + up) / 2;
      if (a.e[mid].general0 <= item) i = mid;
      else up = mid;
    }
    const uint32_t in = item - a.e[i].general0, tiles = a.e[i].tiles, tile = (tiles + PER - 1) / PER - 1 - in / a.kv_heads;
    const uint32_t kvh = in % a.kv_heads, tile0 = tile * (16 * R * W), row0 = tile0 + wave * (16 * R);
    if (!flagged) {
      uint32_t some = 0;
      for (uint32_t t = PER * tile; t < PER * tile + PER && t < tiles; t++)
        some |= a.todo[a.e[i].item0 + (tiles - 1 - t) * a.kv_heads + kvh];
      if (!some) continue;  // uniform
    }
    v4i qd[R][DT][4];
    prompt_query<DT, R>(a, i, kvh, row0, qd);
    if (flagged) prompt_tile<4, 4, DT, R, W, TRACE>(a, lk, lv, i, kvh, tile0, row0, qd);
    else prompt_tile<1, 4, DT, R, W, TRACE>(a, lk, lv, i, kvh, tile0, row0, qd);
    __syncthreads();  // LDS is written again
  }
}

}  // namespace gkr
