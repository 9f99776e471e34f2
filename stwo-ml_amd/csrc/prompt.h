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

struct PromptPack {
  uint32_t n, kv_heads, dim, chunks;
  uint64_t head_bytes;  // of a kv head's blocks, all sequences'
  struct {
    uint32_t block0, len, at;  // its first block in this launch; tokens; its first block of all
    uint32_t pad;
    uint64_t row;              // its first row of k and v
  } e[kPromptSeqs];
};
// Bytes of plane p of a block begin at p * chunks * 1024.
__device__ __forceinline__ uint32_t prompt_key(uint32_t token, uint32_t chunk) { return chunk * 1024 + 16 * token; }
__device__ __forceinline__ uint32_t prompt_value(uint32_t quarter, uint32_t dim) {
  return dim / 16 * 1024 + 256 * quarter + 16 * (dim % 16);
}
// A workgroup packs a block of 64 tokens of one kv head, a wave 16 dims at a time.
// Words of the mask are set where a digit above plane 0 is not zero, and `clear`,
// the mask of the next operator on the stream, is zeroed, as in k_wit_pack.
// Places behind a sequence's last token get its words again: they have no weight.
static __global__ void __launch_bounds__(256) k_prompt_pack(PromptPack a, const uint32_t* __restrict__ k,
                                                            const uint32_t* __restrict__ v, int8_t* __restrict__ ko,
                                                            int8_t* __restrict__ vo, uint32_t* __restrict__ mask,
                                                            uint32_t* __restrict__ clear) {
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x < kMaskWords) clear[kMaskStride * threadIdx.x] = 0;
  uint32_t i = 0;
  for (uint32_t up = a.n; up - i > 1;) {  // the last sequence that begins at or before this block
    const uint32_t mid = (i + up) / 2;
    if (a.e[mid].block0 <= blockIdx.x) i = mid;
    else up = mid;
  }
  const uint32_t in = blockIdx.x - a.e[i].block0, first = in * kAttBlock, last = a.e[i].len - 1, head = blockIdx.y;
  const uint64_t width = (uint64_t)a.kv_heads * a.dim;
  const uint64_t to = head * a.head_bytes + (uint64_t)(a.e[i].at + in) * (4 * 1024 * a.chunks);
  const uint32_t lane = threadIdx.x & 63, q = lane & 3, plane = 1024 * a.chunks;
  uint32_t high = 0;
  auto words = [&](const uint32_t* m, uint32_t token, uint32_t d, uint32_t (&x)[4]) {
    const uint32_t t = first + token < last ? first + token : last;
    const uint32_t* const from = m + (a.e[i].row + t) * width + (uint64_t)head * a.dim + d;
    if (d + 4 <= a.dim) {
      const v4i_word w = *(const v4i_word*)from;
#pragma unroll
      for (int j = 0; j < 4; j++) x[j] = digit_bytes((uint32_t)w[j]);
    } else {
#pragma unroll
      for (uint32_t j = 0; j < 4; j++) x[j] = d + j < a.dim ? digit_bytes(from[j]) : 0u;
    }
  };
  for (uint32_t chunk = threadIdx.x >> 6; chunk < a.chunks; chunk += 4) {
    // keys: lane 4 t + q has token t's dims 4 q .. + 3, and stores plane q of its 16
#pragma unroll
    for (uint32_t t0 = 0; t0 < 64; t0 += 16) {
      uint32_t x[4], out[4];
      words(k, t0 + lane / 4, 16 * chunk + 4 * q, x);
      transpose_bytes(x, out);
      high |= out[1] | out[2] | out[3];
      quad_transpose(out);
      *(uint4*)(ko + to + q * plane + prompt_key(t0 + lane / 4, chunk)) = make_uint4(out[0], out[1], out[2], out[3]);
    }
    // values: lane 16 c + 4 g + t has tokens 16 t + 4 c .. + 3 of dims 4 g .. + 3
    const uint32_t c = lane / 16, g = lane / 4 % 4;
    uint32_t x[4][4], y[4][4];  // [token][dim], [dim][plane]
#pragma unroll
    for (uint32_t j = 0; j < 4; j++) words(v, 16 * q + 4 * c + j, 16 * chunk + 4 * g, x[j]);
#pragma unroll
    for (uint32_t d = 0; d < 4; d++) {
      const uint32_t of[4] = {x[0][d], x[1][d], x[2][d], x[3][d]};
      transpose_bytes(of, y[d]);
      high |= y[d][1] | y[d][2] | y[d][3];
    }
#pragma unroll
    for (uint32_t p = 0; p < 4; p++) {
      uint32_t w[4] = {y[0][p], y[1][p], y[2][p], y[3][p]};
      quad_transpose(w);  // lane q of a quad: dim 4 g + q, all of t
      *(uint4*)(vo + to + p * plane + prompt_value(c, 16 * chunk + 4 * g + q)) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  if (__any(high != 0) && lane == 0) {
    volatile uint32_t* const word = mask + kMaskStride * ((blockIdx.x * 4 + (threadIdx.x >> 6)) % kMaskWords);
    if (!*word) *word = 1;
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

struct PromptArgs {
  const int8_t *k, *v;
  const uint32_t *q, *mask;
  AttOut o;
  uint64_t head_bytes;
  uint32_t n, kv_heads, group, dim, chunks;
  uint32_t offset, table_mask;
  struct {
    uint32_t item0, tiles;  // its first item of this launch, its tiles of rows
    uint32_t len, at;       // tokens; its first block
    uint64_t row;           // its first row of q
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

// A workgroup's W waves have R tiles of 16 rows each and take the blocks in step:
// keys and values of a block go through LDS, each on its way from memory while
// the other is used.
template <int NP, int NQ, int DT, int R, int W, bool TRACE>
__device__ __forceinline__ void prompt_tile(const PromptArgs& a, v4i* lds, uint32_t i, uint32_t kvh, uint32_t tile0,
                                            uint32_t row0, const v4i (&qd)[R][DT][NQ]) {
  constexpr int NG = NP + NQ - 1, NV = NP + 1;  // NP = 1: sums of the small and of the wide weights
  constexpr uint32_t CH = 4 * DT;               // chunks of 16 dims in LDS
  constexpr int ND = (int)(CH * NP / W);        // 1 KB pieces of keys, and of values, a wave copies
  v4i *const lk = lds, *const lv = lds + NP * CH * 64;
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
  const uint64_t base = kvh * a.head_bytes + (uint64_t)a.e[i].at * (4 * plane) + 16 * lane;
  v4i in[ND];
  auto load = [&](const int8_t* from, uint32_t b) {
#pragma unroll
    for (int j = 0; j < ND; j++) {
      const uint32_t piece = wave * ND + j, p = piece / CH, chunk = piece % CH;
      if (CH == 4 && a.chunks < CH && chunk >= a.chunks) continue;
      in[j] = *(const v4i*)(from + base + (uint64_t)b * (4 * plane) + p * plane + 1024 * (chunk < a.chunks ? chunk : a.chunks - 1));
    }
  };
  auto put = [&](v4i* to) {
#pragma unroll
    for (int j = 0; j < ND; j++) to[(wave * ND + j) * 64 + lane] = in[j];
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
  load(a.k, 0);
  put(lk);
#pragma unroll 1
  for (uint32_t b = 0; b < blocks; b++) {
    __syncthreads();  // the keys are there, the values' place is free
    load(a.v, b);
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
            if constexpr (NG == 1) {
              x[v] = signed32_mod_p(sc[r][0][v]);
            } else if constexpr (NG == 4) {
              // |sc[g]| <= 2^22 and the offset: pairs in 32 bits, the upper one turned by 16 of 31 bits
              const uint32_t low = signed32_mod_p(sc[r][0][v]), mid = signed32_mod_p(sc[r][1][v] << 8);
              const uint32_t high = signed32_mod_p(sc[r][2][v] + (sc[r][3][v] << 8));
              x[v] = m31_add(m31_add(low, mid), ((high << 16) & P) | (high >> 15));
            } else {
              x[v] = prompt_score<(DT <= 2)>(sc[r], v, off);
            }
          }
          if (TRACE) {
            const uint32_t first = b * kAttBlock + 16 * t + 4 * quarter;
            const uint32_t row = row0 + 16 * r + col, token = row / a.group;
            const uint64_t at = (((a.e[i].row + token) * a.kv_heads + kvh) * a.group + (row - token * a.group)) * a.o.score_cols + first;
            if (seen[r]) {
              if (first + 4 <= a.o.score_cols) {
                v4i_word kept;
#pragma unroll
                for (int v = 0; v < 4; v++) kept[v] = first + v < seen[r] ? (int)x[v] : 0;
                *(v4i_word*)(a.o.scores + at) = kept;
              } else {
#pragma unroll
                for (int v = 0; v < 4; v++)
                  if (first + v < a.o.score_cols) a.o.scores[at + v] = first + v < seen[r] ? x[v] : 0u;
              }
            }
          }
          w0[r][t] = pick_bytes<2>(x) & place_mask;
        }
      }
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
          for (int t = 0; t < 4; t++) {
            const uint32_t in_sight = prompt_seen((int)(seen[r] - (b * kAttBlock + 16 * t + 4 * quarter)));
            w0[r][t] &= in_sight;
            w1[r][t] &= in_sight;
          }
      }
      uint32_t any_small = 0;
#pragma unroll
      for (int r = 0; r < R; r++)
#pragma unroll
        for (int t = 0; t < 4; t++) {
          any_small |= w0[r][t];
          z[r][0] = __builtin_amdgcn_sdot4((int)w0[r][t], 0x01010101, z[r][0], false);
          z[r][1] = __builtin_amdgcn_sdot4((int)w1[r][t], 0x01010101, z[r][1], false);
        }
      some_small = __any(any_small != 0);
    }
    put(lv);
    __syncthreads();  // the values are there, the keys' place is free
    if (b + 1 < blocks) load(a.k, b + 1);
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
    if (b + 1 < blocks) put(lk);
  }
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
      const uint64_t at = ((a.e[i].row + token) * a.kv_heads + kvh) * a.group + (row - token * a.group);
      if (a.o.sums && col == 0) a.o.sums[at] = shift16(m31_from_u32(zr));
      const double inv = 0.5 / zr;
#pragma unroll
      for (int d = 0; d < (int)CH; d++) {
        int64_t total = 0;
        if constexpr (NP == 1) {
          total = -((int64_t)acc[r][d][0][v] + ((int64_t)acc[r][d][1][v] << 3));
        } else {
#pragma unroll
          for (int g = 0; g < NV; g++) total -= (int64_t)acc[r][d][g][v] << (8 * g);
        }
        if (16 * d + col < a.dim) {
          a.o.out[at * a.dim + 16 * d + col] = prompt_mean(total, zr, inv);
          if (a.o.weighted) a.o.weighted[at * a.dim + 16 * d + col] = shift16(signed_mod_p(total));
        }
      }
    }
  }
  if (TRACE && row0 < rows)  // behind the last block they are cleared
    for (uint32_t row = row0; row < wave_end; row++) {
      const uint32_t token = row / a.group;
      const uint64_t at = ((a.e[i].row + token) * a.kv_heads + kvh) * a.group + (row - token * a.group);
      for (uint64_t t = (uint64_t)mine * kAttBlock + lane; t < a.o.score_cols; t += 64) a.o.scores[at * a.o.score_cols + t] = 0;
    }
}
// NP planes of the keys and values; NP = 1 takes four of the queries where a row
// of its workgroup has them, a tile at a time.
template <int NP, int DT, int R, int W, bool TRACE>
__global__ void __launch_bounds__(64 * W, DT == 4 ? 1 : 2) k_prompt(PromptArgs a) {
  __shared__ v4i lds[2 * NP * 4 * DT * 64];
  __shared__ uint32_t general;
  if (wit_four(a.mask) != (NP > 1)) return;  // uniform
  const uint32_t item = blockIdx.x;
  uint32_t i = 0;
  for (uint32_t up = a.n; up - i > 1;) {  // the last sequence that begins at or before this item
    const uint32_t mid = (i + up) / 2;
    if (a.e[mid].item0 <= item) i = mid;
    else up = mid;
  }
  const uint32_t in = item - a.e[i].item0, tile = a.e[i].tiles - 1 - in / a.kv_heads, kvh = in % a.kv_heads;
  const uint32_t lane = threadIdx.x & 63, col = lane & 15, quarter = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t tile0 = tile * (16 * R * W), row0 = tile0 + wave * (16 * R), rows = a.e[i].len * a.group;
  uint32_t high = 0;
  auto query = [&](uint32_t at, auto& qd, auto planes) {  // of 16 rows
    const uint32_t row = at + col < rows ? at + col : rows - 1, token = row / a.group;
    const uint32_t* const from =
        a.q + (((a.e[i].row + token) * a.kv_heads + kvh) * a.group + (row - token * a.group)) * a.dim;
#pragma unroll
    for (int s = 0; s < DT; s++)
#pragma unroll
      for (uint32_t j = 0; j < 4; j++) {
        const uint32_t d = 64 * s + 16 * quarter + 4 * j;
        uint32_t x[4], out[4];
        if (d + 4 <= a.dim) {
          const v4i_word w = *(const v4i_word*)(from + d);
#pragma unroll
          for (int t = 0; t < 4; t++) x[t] = digit_bytes((uint32_t)w[t]);
        } else {
#pragma unroll
          for (uint32_t t = 0; t < 4; t++) x[t] = d + t < a.dim ? digit_bytes(from[d + t]) : 0u;
        }
        transpose_bytes(x, out);
        high |= out[1] | out[2] | out[3];
#pragma unroll
        for (int p = 0; p < decltype(planes)::value; p++) qd[s][p][j] = (int)out[p];
      }
  };
  if constexpr (NP == 1) {
    v4i qd[R][DT][1];
    if (threadIdx.x == 0) general = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; r++) query(row0 + 16 * r, qd[r], std::integral_constant<int, 1>{});
    if (__any(high != 0) && lane == 0) general = 1;
    __syncthreads();
    if (!general) {  // uniform
      prompt_tile<1, 1, DT, R, W, TRACE>(a, lds, i, kvh, tile0, row0, qd);
      return;
    }
#pragma unroll 1
    for (int r = 0; r < R; r++) {
      const uint32_t start = tile0 + r * (16 * W);
      if (start >= rows) return;  // uniform
      v4i qg[1][DT][4];
      query(start + 16 * wave, qg[0], std::integral_constant<int, 4>{});
      prompt_tile<1, 4, DT, 1, W, TRACE>(a, lds, i, kvh, start, start + 16 * wave, qg);
      __syncthreads();  // LDS is written again
    }
  } else {
    v4i qd[R][DT][4];
#pragma unroll
    for (int r = 0; r < R; r++) query(row0 + 16 * r, qd[r], std::integral_constant<int, 4>{});
    prompt_tile<NP, 4, DT, R, W, TRACE>(a, lds, i, kvh, tile0, row0, qd);
  }
}

}  // namespace gkr
