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
// digits (gemm.h; one plane in an int8 cache), 1 KB per plane and 16 dims, in
// the operand order of v_mfma_i32_16x16x64_i8:
//   keys    [plane][dim / 16][token][dim % 16]: lane l of the score product
//           reads token 16 t + l % 16, dims 16 (4 s + l / 16) .. + 15;
//   values  [plane][dim / 16][c][dim % 16][4 t + v] holds token 16 t + 4 c + v:
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
constexpr uint32_t kAttMaxBlocks = 1024;  // blocks per workgroup: 65536 tokens keep the digit sums below 2^31

struct KvPool {
  int8_t *k, *v;
  const uint32_t* pages;  // [seq][width]: the pages of a sequence's tokens
  uint32_t width, page_blocks, kv_heads, dim, chunks, planes;
};
__device__ __forceinline__ uint64_t kv_block(const KvPool& p, uint32_t seq, uint32_t block, uint32_t head) {
  const uint32_t page = p.pages[(uint64_t)seq * p.width + block / p.page_blocks];
  return (((uint64_t)page * p.kv_heads + head) * p.page_blocks + block % p.page_blocks) * p.planes * p.chunks * 1024;
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
// A workgroup takes four token positions 4 i .. 4 i + 3 of a sequence; a
// thread, one value of them at a time (neighbours read neighbouring words).
// Bytes are stored one by one, so tokens that were there stay.  A word outside
// an int8 cache's range sets *bad (host memory).
static __global__ void __launch_bounds__(256) k_kv_append(KvPool p, KvAppend a, const uint32_t* __restrict__ k,
                                                          const uint32_t* __restrict__ v, uint32_t* bad) {
  uint32_t i = 0;
  while (i + 1 < a.n && a.e[i + 1].quad0 <= blockIdx.x) i++;
  const uint32_t pos = a.e[i].pos, end = pos + a.e[i].count;
  const uint32_t t0 = (pos / 4 + (blockIdx.x - a.e[i].quad0)) * 4;  // never crosses a block
  const uint32_t width = p.kv_heads * p.dim, block = t0 / kAttBlock;
  const uint64_t plane = (uint64_t)p.chunks * 1024;
  for (uint32_t w = threadIdx.x; w < width; w += blockDim.x) {
    const uint32_t head = w / p.dim, d = w % p.dim;
    const uint64_t base = kv_block(p, a.e[i].seq, block, head);
    for (uint32_t t = t0 < pos ? pos : t0; t < t0 + 4 && t < end; t++) {
      const uint64_t at = (a.e[i].row + (t - pos)) * width + w;
      const uint32_t in = t % kAttBlock;
      const uint64_t ko = base + kv_key_byte(in, d), vo = base + kv_value_byte(in, d);
      int32_t dk[4], dv[4];
      balanced_digits(center_m31(k[at]), dk);
      balanced_digits(center_m31(v[at]), dv);
      if (p.planes == 1 && (dk[1] | dk[2] | dk[3] | dv[1] | dv[2] | dv[3])) *(volatile uint32_t*)bad = 1;
      for (uint32_t q = 0; q < p.planes; q++) {
        p.k[q * plane + ko] = (int8_t)dk[q];
        p.v[q * plane + vo] = (int8_t)dv[q];
      }
    }
  }
}

struct AttRowArgs {
  uint32_t n;
  struct {
    uint32_t seq, len, part0;  // part0: workgroups of the rows before it
  } e[kAttRows];
};
struct AttOut {
  uint32_t *out, *weighted, *sums, *scores;
  uint64_t score_cols;
};

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
    const uint64_t u = (uint64_t)(total < 0 ? -total : total);
    const uint32_t r = (uint32_t)((2 * u + z) / (2 * (uint64_t)z));  // |c(v)| <= 2^30: r too
    mean = total < 0 ? m31_neg(r) : r;
  }
  o.out[at] = mean;
  if (o.weighted) o.weighted[at] = shift16(signed_mod_p(total));
}

// A store of four scores, on a 4-byte boundary at least.
struct __attribute__((packed, aligned(4))) Scores4 {
  uint32_t v[4];
};

// One workgroup: up to 16 query heads of one kv head, `bpw` blocks of one row.
// Four blocks a step: wave w forms the scores and weights of block w, all
// waves read the four blocks' weights from LDS (two buffers, one barrier a
// step), and wave w takes the dims 16 (w + 4 i) .. + 15 of the values.  The
// loads run ahead: a wave holds NS of its four token tiles of keys and NS of
// the step's four blocks of values, and refills each as it has used it, across
// steps (values are loaded before their weights are known).
// NP planes of the cache; DT = dims / 64 rounded up.
template <int NP, int DT>
static __global__ void __launch_bounds__(256) k_attend(KvPool p, AttRowArgs rows, uint32_t bpw,
                                                       const uint32_t* __restrict__ q, uint32_t heads,
                                                       uint32_t row0, uint32_t offset, uint32_t mask,
                                                       int64_t* __restrict__ part, uint32_t* __restrict__ part_z,
                                                       AttOut o) {
  constexpr int NG = NP + 3, NV = NP + 1;  // digit groups of the scores and of the weighted sums
  constexpr int NS = NP * DT <= 4 ? 4 : NP * DT <= 8 ? 2 : 1;
  __shared__ v4i weights[2][4][2][64];
  __shared__ uint32_t zsum[4][16];
  const uint32_t lane = threadIdx.x & 63, col = lane & 15, quarter = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t r = 0;
  while (r + 1 < rows.n && rows.e[r + 1].part0 <= blockIdx.x) r++;
  const uint32_t group = heads / p.kv_heads, tiles = (group + kAttHeads - 1) / kAttHeads;
  const uint32_t kvh = blockIdx.y / tiles, h0 = blockIdx.y % tiles * kAttHeads;
  const uint32_t mine = group - h0 < kAttHeads ? group - h0 : kAttHeads;  // heads of this workgroup
  const uint32_t seq = rows.e[r].seq, len = rows.e[r].len, nblocks = (len + kAttBlock - 1) / kAttBlock;
  const uint64_t row = row0 + r;
  const uint32_t b0 = (blockIdx.x - rows.e[r].part0) * bpw;
  const uint32_t head0 = kvh * group + h0;
  const uint32_t plane = p.chunks * 1024;
  const uint32_t b_end = b0 + bpw, seen_end = b_end < nblocks ? b_end : nblocks;

  v4i kd[NS][DT][NP], vd[NS][DT][NP];
  const int8_t *kbase = nullptr, *vbase[4] = {};
  auto key_block = [&](uint32_t b) {  // this wave's block of the step from b: past the end, the last one again
    const uint32_t block = b + wave < seen_end ? b + wave : seen_end - 1;
    kbase = p.k + kv_block(p, seq, block, kvh);
  };
  auto load_keys = [&](int slot, int t) {
#pragma unroll
    for (int s = 0; s < DT; s++) {
      const uint32_t chunk = 4 * s + quarter;  // past the dims the query's digits are zero
      const uint32_t at = (chunk < p.chunks ? chunk : p.chunks - 1) * 1024 + 256 * t + 16 * col;
#pragma unroll
      for (int pk = 0; pk < NP; pk++) kd[slot][s][pk] = __builtin_nontemporal_load((const v4i*)(kbase + (at + pk * plane)));
    }
  };
  auto value_blocks = [&](uint32_t b) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const uint32_t block = b + j < seen_end ? b + j : seen_end - 1;
      vbase[j] = p.v + kv_block(p, seq, block, kvh);
    }
  };
  auto load_values = [&](int slot, int j) {
#pragma unroll
    for (int i = 0; i < DT; i++) {
      const uint32_t tile = wave + 4 * i < p.chunks ? wave + 4 * i : p.chunks - 1;  // past the dims: not stored
#pragma unroll
      for (int pv = 0; pv < NP; pv++)
        vd[slot][i][pv] = __builtin_nontemporal_load((const v4i*)(vbase[j] + (tile * 1024 + pv * plane + 16 * lane)));
    }
  };
  if (b0 < seen_end) {
    key_block(b0);
    value_blocks(b0);
#pragma unroll
    for (int t = 0; t < NS; t++) load_keys(t, t);
#pragma unroll
    for (int j = 0; j < NS; j++) load_values(j, j);
  }

  v4i qd[DT][4];  // the query's digits: head col, dims 16 (4 s + quarter) .. + 15
#pragma unroll
  for (int s = 0; s < DT; s++) {
    uint32_t w[4][4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      uint32_t d[4], out[4];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const uint32_t dim = 16 * (4 * s + quarter) + 4 * i + j;
        d[j] = digit_bytes(col < mine && dim < p.dim ? q[(row * heads + head0 + col) * p.dim + dim] : 0u);
      }
      transpose_bytes(d, out);
#pragma unroll
      for (int g = 0; g < 4; g++) w[g][i] = out[g];
    }
#pragma unroll
    for (int g = 0; g < 4; g++) qd[s][g] = v4i{(int)w[g][0], (int)w[g][1], (int)w[g][2], (int)w[g][3]};
  }
  v4i acc[DT][NV];
#pragma unroll
  for (int i = 0; i < DT; i++)
#pragma unroll
    for (int g = 0; g < NV; g++) acc[i][g] = v4i{0, 0, 0, 0};
  uint32_t z = 0;
  uint32_t* const my_scores =
      o.scores && col < mine ? o.scores + (row * heads + head0 + col) * o.score_cols : nullptr;
  auto store_scores = [&](uint32_t block, int t, const uint32_t (&x)[4]) {
    const uint64_t tok = (uint64_t)block * kAttBlock + 16 * t + 4 * quarter;
    if (!my_scores || block >= b_end || tok >= o.score_cols) return;
    if (tok + 4 <= o.score_cols)
      *(Scores4*)(my_scores + tok) = Scores4{{x[0], x[1], x[2], x[3]}};
    else
      for (int v = 0; v < 4; v++)
        if (tok + v < o.score_cols) my_scores[tok + v] = x[v];
  };
  uint32_t b = b0;
  for (uint32_t turn = 0; b < seen_end; b += 4, turn ^= 1) {
    const uint32_t block = b + wave, first = block * kAttBlock + 4 * quarter;
    v4i w0, w1;
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
      if (t + NS == 4 && b + 4 < seen_end) key_block(b + 4);
      if (t + NS < 4 || b + 4 < seen_end) load_keys(t % NS, (t + NS) % 4);
      uint32_t x[4], lo = 0, hi = 0;
#pragma unroll
      for (int v = 0; v < 4; v++) {
        // sum_g 256^g sc[g], below 2^52, with 2^32 = 2 (mod P)
        int64_t sum = (int64_t)sc[0][v] + ((int64_t)sc[1][v] << 8) + ((int64_t)sc[2][v] << 16) + ((int64_t)sc[3][v] << 24);
        if constexpr (NP > 1)
          sum += ((int64_t)sc[4][v] << 1) + ((int64_t)sc[5][v] << 9) + ((int64_t)sc[6][v] << 17);
        const uint32_t xv = m31_add(m31_reduce64((uint64_t)(sum + ((int64_t)P << 24))), offset);
        const bool seen = block < seen_end && first + 16 * t + v < len;
        uint32_t g = (xv & mask) >> 16;
        g = g < 10 ? g : 10;
        const uint32_t e = seen ? 1u << g : 0u;  // digits base 256, balanced: 128 is 256 - 128
        x[v] = seen ? xv : 0u;
        z += e;
        lo |= (e & 0xffu) << (8 * v);
        hi |= ((e + 0x80u) >> 8) << (8 * v);
      }
      w0[t] = (int)lo;
      w1[t] = (int)hi;
      store_scores(block, t, x);
    }
    weights[turn][wave][0][lane] = w0;
    weights[turn][wave][1][lane] = w1;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; j++) {  // blocks past the end have no weight
      const v4i e0 = weights[turn][j][0][lane], e1 = weights[turn][j][1][lane];
#pragma unroll
      for (int i = 0; i < DT; i++)
#pragma unroll
        for (int pv = 0; pv < NP; pv++) {
          acc[i][pv] = __builtin_amdgcn_mfma_i32_16x16x64_i8(e0, vd[j % NS][i][pv], acc[i][pv], 0, 0, 0);
          acc[i][pv + 1] = __builtin_amdgcn_mfma_i32_16x16x64_i8(e1, vd[j % NS][i][pv], acc[i][pv + 1], 0, 0, 0);
        }
      if (j + NS == 4 && b + 4 < seen_end) value_blocks(b + 4);
      if (j + NS < 4 || b + 4 < seen_end) load_values(j % NS, (j + NS) % 4);
    }
  }
  if (o.scores) {  // scores behind the last token are cleared
    const uint32_t none[4] = {0, 0, 0, 0};
    for (; b < b_end; b += 4)
      for (int t = 0; t < 4; t++) store_scores(b + wave, t, none);
  }
  z += __shfl_xor(z, 16);
  z += __shfl_xor(z, 32);
  if (lane < 16) zsum[wave][lane] = z;
  __syncthreads();
  const uint32_t parts = (r + 1 < rows.n ? rows.e[r + 1].part0 : gridDim.x) - rows.e[r].part0;
#pragma unroll
  for (int v = 0; v < 4; v++) {
    const uint32_t h = 4 * quarter + v;
    if (h >= mine) continue;
    const uint32_t zh = zsum[0][h] + zsum[1][h] + zsum[2][h] + zsum[3][h];
#pragma unroll
    for (int i = 0; i < DT; i++) {
      const uint32_t d = 16 * (wave + 4 * i) + col;
      if (d >= p.dim) continue;
      int64_t total = 0;
#pragma unroll
      for (int g = 0; g < NV; g++) total += (int64_t)acc[i][g][v] << (8 * g);
      if (parts == 1)
        att_finish(o, (row * heads + head0 + h) * p.dim + d, total, zh);
      else
        part[((uint64_t)blockIdx.x * heads + head0 + h) * p.dim + d] = total;
    }
    if (wave == 0 && col == 0) {
      if (parts > 1) part_z[(uint64_t)blockIdx.x * heads + head0 + h] = zh;
      else if (o.sums) o.sums[row * heads + head0 + h] = shift16(m31_from_u32(zh));
    }
  }
}

// Joins the parts of rows that have several: workgroup (row, head), whose
// eight waves take the parts in turn and a lane up to four dims.
static __global__ void __launch_bounds__(512) k_attend_join(AttRowArgs rows, uint32_t n_parts, uint32_t heads,
                                                            uint32_t dim, uint32_t row0,
                                                            const int64_t* __restrict__ part,
                                                            const uint32_t* __restrict__ part_z, AttOut o) {
  __shared__ unsigned long long total[256];
  __shared__ uint32_t z;
  const uint32_t r = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
  const uint32_t first = rows.e[r].part0, last = r + 1 < rows.n ? rows.e[r + 1].part0 : n_parts;
  if (last - first == 1) return;
  if (tid < 256) total[tid] = 0;
  if (tid == 0) z = 0;
  __syncthreads();
  for (uint32_t d = tid & 63; d < dim; d += 64) {
    int64_t t = 0;
#pragma unroll 8
    for (uint32_t i = first + (tid >> 6); i < last; i += 8) t += part[((uint64_t)i * heads + h) * dim + d];
    atomicAdd(&total[d], (unsigned long long)t);
  }
  uint32_t mine = 0;
  for (uint32_t i = first + tid; i < last; i += 512) mine += part_z[(uint64_t)i * heads + h];
  if (mine) atomicAdd(&z, mine);
  __syncthreads();
  if (tid < dim) att_finish(o, ((uint64_t)(row0 + r) * heads + h) * dim + tid, (int64_t)total[tid], z);
  if (tid == 0 && o.sums) o.sums[(uint64_t)(row0 + r) * heads + h] = shift16(m31_from_u32(z));
}

}  // namespace gkr
