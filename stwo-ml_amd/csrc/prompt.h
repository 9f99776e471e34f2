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

// A wave has R tiles of 16 rows.
template <int NP, int NQ, int DT, int R>
__device__ __forceinline__ void prompt_tile(const PromptArgs& a, uint32_t i, uint32_t kvh, uint32_t row0, const v4i (&qd)[R][DT][4]) {
  constexpr int NG = NP + NQ - 1, NV = NP + 1;
  const uint32_t lane = threadIdx.x & 63, col = lane & 15, quarter = lane >> 4;
  const uint32_t len = a.e[i].len, rows = len * a.group, plane = 1024 * a.chunks;
  uint32_t seen[R];  // of row row0 + 16 r + col
  uint32_t last = row0 + 16 * R < rows ? row0 + 16 * R : rows;
  const uint32_t blocks = ((last - 1) / a.group + kAttBlock) / kAttBlock;
#pragma unroll
  for (int r = 0; r < R; r++) {
    const uint32_t row = row0 + 16 * r + col;
    seen[r] = row < rows ? row / a.group + 1 : 0;
  }
  v4i acc[R][DT * 4][NV];
#pragma unroll
  for (int r = 0; r < R; r++)
#pragma unroll
    for (int d = 0; d < DT * 4; d++)
#pragma unroll
      for (int g = 0; g < NV; g++) acc[r][d][g] = v4i{0, 0, 0, 0};
  uint32_t z[R] = {};
  const uint64_t base = kvh * a.head_bytes + (uint64_t)a.e[i].at * (4 * plane);
#pragma unroll 1
  for (uint32_t b = 0; b < blocks; b++) {
    const int8_t *const kb = a.k + base + (uint64_t)b * (4 * plane), *const vb = a.v + base + (uint64_t)b * (4 * plane);
    v4i w0[R], w1[R];
#pragma unroll
    for (int t = 0; t < 4; t++) {
      v4i sc[R][NG];
#pragma unroll
      for (int r = 0; r < R; r++)
#pragma unroll
        for (int g = 0; g < NG; g++) sc[r][g] = v4i{0, 0, 0, 0};
#pragma unroll
      for (int s = 0; s < DT; s++) {
        const uint32_t chunk = 4 * s + quarter < a.chunks ? 4 * s + quarter : a.chunks - 1;  // the query is zero there
#pragma unroll
        for (int p = 0; p < NP; p++) {
          const v4i kd = *(const v4i*)(kb + p * plane + prompt_key(16 * t + col, chunk));
#pragma unroll
          for (int r = 0; r < R; r++)
#pragma unroll
            for (int g = 0; g < NQ; g++)
              sc[r][p + g] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kd, qd[r][s][g], sc[r][p + g], 0, 0, 0);
        }
      }
#pragma unroll
      for (int r = 0; r < R; r++) {
        const uint32_t first = b * kAttBlock + 16 * t + 4 * quarter;
        uint32_t e[4], e8[4], x[4];
#pragma unroll
        for (int v = 0; v < 4; v++) {
          // sum_g 256^g sc[g], below 2^52, with 2^32 = 2 (mod P)
          int64_t sum = (int64_t)sc[r][0][v];
#pragma unroll
          for (int g = 1; g < NG; g++) sum += (int64_t)sc[r][g][v] << (g < 4 ? 8 * g : 8 * g - 31);
          x[v] = m31_add(m31_reduce64((uint64_t)(sum + ((int64_t)P << 24))), a.offset);
          uint32_t g = (x[v] & a.table_mask) >> 16;
          g = g < 10 ? g : 10;
          const bool in = first + v < seen[r];
          x[v] = in ? x[v] : 0;
          e[v] = in ? 1u << g : 0u;
          e8[v] = e[v] + 0x80u;  // digits base 256, balanced: 128 is 256 - 128
          z[r] += e[v];
        }
        w0[r][t] = (int)pick_bytes<0>(e);
        w1[r][t] = (int)pick_bytes<1>(e8);
        if (a.o.scores && seen[r]) {
          const uint32_t row = row0 + 16 * r + col, token = row / a.group;
          const uint64_t at = ((a.e[i].row + token) * a.kv_heads + kvh) * a.group + (row - token * a.group);
#pragma unroll
          for (int v = 0; v < 4; v++)
            if (first + v < a.o.score_cols) a.o.scores[at * a.o.score_cols + first + v] = x[v];
        }
      }
    }
#pragma unroll
    for (int d = 0; d < DT * 4; d++) {
      const uint32_t chunk = d < (int)a.chunks ? d : a.chunks - 1;  // not stored
#pragma unroll
      for (int p = 0; p < NP; p++) {
        const v4i vd = *(const v4i*)(vb + p * plane + 1024 * chunk + 16 * lane);
#pragma unroll
        for (int r = 0; r < R; r++) {
          acc[r][d][p] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w0[r], vd, acc[r][d][p], 0, 0, 0);
          acc[r][d][p + 1] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w1[r], vd, acc[r][d][p + 1], 0, 0, 0);
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; r++) {
    z[r] += __shfl_xor(z[r], 16);
    z[r] += __shfl_xor(z[r], 32);
#pragma unroll
    for (int v = 0; v < 4; v++) {
      const uint32_t row = row0 + 16 * r + 4 * quarter + v, zr = __shfl(z[r], 4 * quarter + v);
      const uint32_t token = row / a.group;
      const uint64_t at = ((a.e[i].row + token) * a.kv_heads + kvh) * a.group + (row - token * a.group);
      if (row >= rows) continue;
      if (a.o.sums && col == 0) a.o.sums[at] = shift16(m31_from_u32(zr));
#pragma unroll
      for (int d = 0; d < DT * 4; d++) {
        int64_t total = 0;
#pragma unroll
        for (int g = 0; g < NV; g++) total += (int64_t)acc[r][d][g][v] << (8 * g);
        if (16 * d + col < a.dim) att_finish(a.o, at * a.dim + 16 * d + col, total, zr);
      }
    }
  }
  if (a.o.scores)  // behind the last block they are cleared
    for (uint32_t row = row0; row < last; row++) {
      const uint32_t token = row / a.group;
      const uint64_t at = ((a.e[i].row + token) * a.kv_heads + kvh) * a.group + (row - token * a.group);
      for (uint64_t t = (uint64_t)blocks * kAttBlock + lane; t < a.o.score_cols; t += 64) a.o.scores[at * a.o.score_cols + t] = 0;
    }
}
template <int NP, int DT, int R>
static __global__ void __launch_bounds__(256) k_prompt(PromptArgs a) {
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
  const uint32_t row0 = tile * (64 * R) + (threadIdx.x >> 6) * (16 * R), rows = a.e[i].len * a.group;
  if (row0 >= rows) return;
  v4i qd[R][DT][4];
  uint32_t high = 0;
#pragma unroll
  for (int r = 0; r < R; r++) {
    const uint32_t row = row0 + 16 * r + col < rows ? row0 + 16 * r + col : rows - 1, token = row / a.group;
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
        for (int p = 0; p < 4; p++) qd[r][s][p][j] = (int)out[p];
      }
  }
  if (NP == 1 && !__any(high != 0)) prompt_tile<NP, 1, DT, R>(a, i, kvh, row0, qd);
  else prompt_tile<NP, 4, DT, R>(a, i, kvh, row0, qd);
}

}  // namespace gkr
