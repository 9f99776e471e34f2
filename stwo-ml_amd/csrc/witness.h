// The witness operators' kernels: products of canonical M31 words by digit
// planes on the matrix cores (gemm.h), with the element-wise work behind them
// (bias, activation, residual, the gate's product) in the same launch.
#pragma once
#include <stdint.h>

#include "field.h"
#include "gemm.h"
#include "witness_sizes.h"

namespace gkr {

// act(z): table == nullptr and relu == 0 is z itself; the table's entry at
// z mod 2^log is what the LogUp layer proves (mask = 2^log - 1).
struct ActArg {
  const uint32_t* table;
  uint32_t mask, relu;
};
// E elements of a thread at once: their loads go out together.
template <int E>
__device__ __forceinline__ void activate(const ActArg& a, uint32_t (&z)[E]) {
  if (a.table) {
#pragma unroll
    for (int e = 0; e < E; e++) z[e] = a.table[z[e] & a.mask];
  } else if (a.relu) {
#pragma unroll
    for (int e = 0; e < E; e++) z[e] = z[e] > (P >> 1) ? 0u : z[e];
  }
}

// Words of a row-major m x n matrix from word `first` on, as a buffer: a lane
// adds a 32-bit byte offset, and a place behind the matrix's last word (a tile's
// rows past m; kOutside for columns past n) reads zero and is not written, with
// no comparison for it.  A matrix that is not given has no bytes.
typedef __amdgpu_buffer_rsrc_t WitBuffer;
__device__ __forceinline__ WitBuffer wit_buffer(const uint32_t* p, uint64_t first, uint64_t count) {
  const uint64_t bytes = p && first < count ? 4 * (count - first) : 0;
  return __builtin_amdgcn_make_buffer_rsrc((void*)(p + (bytes ? first : 0)), 0,
                                           (int)(uint32_t)(bytes < kOutside ? bytes : kOutside), 0x00027000);
}
__device__ __forceinline__ uint32_t wit_read(WitBuffer b, uint32_t at) {
  return (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(b, (int)at, 0, 0);
}
__device__ __forceinline__ void wit_write(WitBuffer b, uint32_t at, uint32_t x) {
  __builtin_amdgcn_raw_buffer_store_b32((int)x, b, (int)at, 0, 0);
}

// What happens to a sum of the product (fused, scaled) or a pair of sums (gated),
// for E elements (byte offsets `at` into the Tile, matrix rows `row`: those of a
// tile's elements past m may be more) of a thread.  fetch() sends out the
// loads that need no sums, begin() takes the sums and sends out those that do,
// finish() stores, so that the next elements' loads can go out before these
// ones' stores.  `c`: what is the columns'.
struct FusedEnd {
  ActArg act;
  const uint32_t* bias;      // n
  const uint32_t* residual;  // m x n; may be out (read by the thread that writes the element)
  uint32_t* pre;
  uint32_t* out;
  struct Tile {
    WitBuffer residual, pre, out;
  };
  struct Column {
    uint32_t bias;
  };
  template <int E>
  struct Slot {
    uint32_t z[E], y[E], residual[E];
  };
  __device__ __forceinline__ Tile tile(uint64_t first, uint64_t count) const {
    return Tile{wit_buffer(residual, first, count), wit_buffer(pre, first, count), wit_buffer(out, first, count)};
  }
  __device__ __forceinline__ Column column(uint64_t col, bool ok) const { return Column{bias && ok ? bias[col] : 0u}; }
  template <int E>
  __device__ __forceinline__ void fetch(Slot<E>& s, const Tile& t, const uint32_t (&at)[E], const uint32_t (&)[E]) const {
    if (residual) {
#pragma unroll
      for (int e = 0; e < E; e++) s.residual[e] = wit_read(t.residual, at[e]);
    }
  }
  template <int E>
  __device__ __forceinline__ void begin(Slot<E>& s, const Column (&c)[E], const uint32_t (&z)[1][E]) const {
#pragma unroll
    for (int e = 0; e < E; e++) s.y[e] = s.z[e] = m31_add(z[0][e], c[e].bias);
    activate(act, s.y);
  }
  template <int E>
  __device__ __forceinline__ void finish(Slot<E>& s, const Tile& t, const uint32_t (&at)[E]) const {
    if (pre) {
#pragma unroll
      for (int e = 0; e < E; e++) wit_write(t.pre, at[e], s.z[e]);
    }
    if (residual) {
#pragma unroll
      for (int e = 0; e < E; e++) s.y[e] = m31_add(s.y[e], s.residual[e]);
    }
#pragma unroll
    for (int e = 0; e < E; e++) wit_write(t.out, at[e], s.y[e]);
  }
};
struct GatedEnd {
  ActArg act;
  uint32_t *gate, *act_out, *up, *out;
  struct Tile {
    WitBuffer gate, act, up, out;
  };
  struct Column {};
  template <int E>
  struct Slot {
    uint32_t z[E], y[E], u[E];
  };
  __device__ __forceinline__ Tile tile(uint64_t first, uint64_t count) const {
    return Tile{wit_buffer(gate, first, count), wit_buffer(act_out, first, count), wit_buffer(up, first, count),
                wit_buffer(out, first, count)};
  }
  __device__ __forceinline__ Column column(uint64_t, bool) const { return {}; }
  template <int E>
  __device__ __forceinline__ void fetch(Slot<E>&, const Tile&, const uint32_t (&)[E], const uint32_t (&)[E]) const {}
  template <int E>
  __device__ __forceinline__ void begin(Slot<E>& s, const Column (&)[E], const uint32_t (&z)[2][E]) const {
#pragma unroll
    for (int e = 0; e < E; e++) {
      s.y[e] = s.z[e] = z[0][e];
      s.u[e] = z[1][e];
    }
    activate(act, s.y);
  }
  template <int E>
  __device__ __forceinline__ void finish(Slot<E>& s, const Tile& t, const uint32_t (&at)[E]) const {
    if (gate) {
#pragma unroll
      for (int e = 0; e < E; e++) wit_write(t.gate, at[e], s.z[e]);
    }
    if (act_out) {
#pragma unroll
      for (int e = 0; e < E; e++) wit_write(t.act, at[e], s.y[e]);
    }
    if (up) {
#pragma unroll
      for (int e = 0; e < E; e++) wit_write(t.up, at[e], s.u[e]);
    }
#pragma unroll
    for (int e = 0; e < E; e++) wit_write(t.out, at[e], m31_mul(s.y[e], s.u[e]));
  }
};
__device__ __forceinline__ uint32_t word_of(int32_t v) { return (uint32_t)v + ((uint32_t)(v >> 31) & P); }
// Rescaled sums: t = round(c(z) r s / 2^shift) + c(bias), halves away from zero,
// cut off at +-limit, with the row's and the column's scale as whole numbers.
// |c(z)| r is below 2^61 and its product with s below 2^92, held in three words;
// what is left of it after the shift is needed to 32 bits only, as limit and
// bias are below 2^30.
struct ScaledEnd {
  const uint32_t* row_scales;  // m, or none (1)
  const uint32_t* col_scales;  // n, or none
  const uint32_t* bias;        // n
  const uint32_t* residual;    // m x n; may be out
  uint32_t *pre, *out;
  uint32_t shift, last_row;  // at most 63; m - 1
  int32_t limit;
  struct Tile {
    WitBuffer residual, pre, out;
  };
  struct Column {
    uint32_t scale, bias;
  };
  template <int E>
  struct Slot {
    uint32_t z[E], y[E], residual[E], row[E];
  };
  __device__ __forceinline__ Tile tile(uint64_t first, uint64_t count) const {
    return Tile{wit_buffer(residual, first, count), wit_buffer(pre, first, count), wit_buffer(out, first, count)};
  }
  __device__ __forceinline__ Column column(uint64_t col, bool ok) const {
    return Column{col_scales && ok ? col_scales[col] : 1u, bias && ok ? bias[col] : 0u};
  }
  template <int E>
  __device__ __forceinline__ void fetch(Slot<E>& s, const Tile& t, const uint32_t (&at)[E], const uint32_t (&row)[E]) const {
#pragma unroll
    for (int e = 0; e < E; e++) s.row[e] = row_scales ? row_scales[umin32(row[e], last_row)] : 1u;
    if (residual) {
#pragma unroll
      for (int e = 0; e < E; e++) s.residual[e] = wit_read(t.residual, at[e]);
    }
  }
  // In three words: |c(z)| r s + half below 2^93, its bits from `shift` on in a word, or
  // all ones where there are more.  The bias moves the bounds: what is cut off at them
  // plus the bias is what the sum would be cut off to.
  __device__ __forceinline__ uint32_t scale(uint32_t z, uint32_t r, const Column& c) const {
    const int32_t v = center_m31(z), sign = v >> 31, bias_of = center_m31(c.bias);
    const uint64_t a = (uint64_t)(uint32_t)((v ^ sign) - sign) * r, half = shift ? 1ull << (shift - 1) : 0;
    const uint64_t low = (uint64_t)(uint32_t)a * c.scale + (uint32_t)half;
    const uint64_t top = (a >> 32) * c.scale + ((low >> 32) + (half >> 32));  // < 2^61
    const bool far = shift >= 32;  // uniform
    const uint32_t w0 = far ? (uint32_t)top : (uint32_t)low, w1 = far ? (uint32_t)(top >> 32) : (uint32_t)top;
    const uint32_t over = ((far ? 0u : (uint32_t)(top >> 32)) | w1 >> (shift & 31));
    const uint32_t t = over ? ~0u : __builtin_amdgcn_alignbit(w1, w0, shift & 31);
    const int32_t y = (int32_t)umin32(t, 0x7fffffffu);
    const int32_t cut = max(min((y ^ sign) - sign, limit - bias_of), -limit - bias_of) + bias_of;
    return word_of(cut);
  }
  template <int E>
  __device__ __forceinline__ void begin(Slot<E>& s, const Column (&c)[E], const uint32_t (&z)[1][E]) const {
#pragma unroll
    for (int e = 0; e < E; e++) {
      s.z[e] = z[0][e];
      s.y[e] = scale(z[0][e], s.row[e], c[e]);
    }
  }
  template <int E>
  __device__ __forceinline__ void finish(Slot<E>& s, const Tile& t, const uint32_t (&at)[E]) const {
    if (pre) {
#pragma unroll
      for (int e = 0; e < E; e++) wit_write(t.pre, at[e], s.z[e]);
    }
    if (residual) {
#pragma unroll
      for (int e = 0; e < E; e++) s.y[e] = m31_add(s.y[e], s.residual[e]);
    }
#pragma unroll
    for (int e = 0; e < E; e++) wit_write(t.out, at[e], s.y[e]);
  }
};
// Columns of elements that share one.
template <int E, class Column>
__device__ __forceinline__ void same_column(Column (&c)[E], const Column& of) {
#pragma unroll
  for (int e = 0; e < E; e++) c[e] = of;
}
// A split's sums, into its part of each matrix.
template <int NW, int E>
__device__ __forceinline__ void wit_parts(uint32_t* part, uint32_t split, uint64_t first, uint64_t count,
                                          const uint32_t (&at)[E], const uint32_t (&z)[NW][E]) {
#pragma unroll
  for (int x = 0; x < NW; x++) {
    const WitBuffer b = wit_buffer(part + (uint64_t)(split * NW + x) * count, first, count);
#pragma unroll
    for (int e = 0; e < E; e++) wit_write(b, at[e], z[x][e]);
  }
}

// A digit plane stack of a weight: planes of kGemmBlockBytes blocks (gemm.h).
struct WitWeight {
  const int8_t* planes;
  uint32_t count;  // planes that are not zero everywhere
};

// sum_p 256^p s[p] mod P for digit sums of fewer than 2^31 in magnitude.
__device__ __forceinline__ uint32_t digit_sum_mod_p(const int32_t (&s)[4]) {
  const int64_t t = (int64_t)s[0] + ((int64_t)s[1] << 8) + ((int64_t)s[2] << 16) + ((int64_t)s[3] << 24);  // < 2^56
  return m31_reduce64((uint64_t)(t + ((int64_t)P << 26)));
}

// round(c(x) levels / a), halves away from zero, for |c(x)| <= a < 2^30 and levels <
// 128.  The product with a rounded ratio is off by less than 127 2^-21, its nearest
// whole number q by one at most; the rest |c| levels - q a, below 1.5 a and so whole
// in 32 bits, says which way.
struct Quantizer {
  float ratio;
  uint32_t a, levels;
  __device__ __forceinline__ Quantizer(uint32_t most, uint32_t to)
      : ratio(most ? (float)to / (float)most : 0.0f), a(most), levels(to) {}
  __device__ __forceinline__ int32_t operator()(uint32_t x) const {
    const int32_t v = center_m31(x), sign = v >> 31;
    const uint32_t c = (uint32_t)((v ^ sign) - sign), q = (uint32_t)__builtin_fmaf((float)c, ratio, 0.5f);
    const int32_t rest = (int32_t)(c * levels - q * a), half = (int32_t)(a >> 1);
    const int32_t r = (int32_t)q + (rest < -half ? -1 : rest > (int32_t)(a - 1) - half && a ? 1 : 0);
    return (r ^ sign) - sign;
  }
};
__device__ __forceinline__ uint32_t size_of_word(uint32_t x) {  // |c(x)|
  const int32_t v = center_m31(x);
  return (uint32_t)(v < 0 ? -v : v);
}
// Rows that are brought to 8 bits before they are multiplied: levels, and where
// their words (m x k) and scales (m) go, if anywhere.
struct WitQuant {
  uint32_t levels;
  uint32_t *words, *scales;
};

// Few rows.  The rows' digit planes are rows of one product: row' 4 i + p is
// plane p of row i, 16 of them to a v_mfma_i32_16x16x64_i8, so general words cost
// no more than int8-range ones, and lane 16 j + c of the accumulator of tile t
// holds the four digit sums of row 4 t + j, column c.
//
// A workgroup has 32 columns of the weights and all of K: it lays the rows'
// digits out in LDS (one to four rows kRowLds bytes at a time, more rows at
// once) and its waves take K pairs of 32 in turn, a pair's 2 KB per plane in two
// loads, U pairs in flight; then the waves' sums meet in LDS (integers: any
// order gives the same).  No packing launch, no partial sums in memory: bound by
// the weights' bytes (packing, the product, its splits' sum and the epilogue as
// launches of their own, then this: 1 x 576 x 192 11.4 -> 4.5 us; 1 x 13824 x
// 5120 39.1 -> 14.0, 5.1 TB/s; gated 1 x 5120 x 13824 47.0 -> 23.2, 6.1 TB/s,
// where a read of 4 GiB reaches 6.4).  The rows' words are asked for before the
// weights: behind them they came last, and the layout with them (17.2 and 29.3
// us, also with sixteen waves for the gated pair's 432 column tiles).
// W waves: sixteen, or eight, of which two workgroups fit a CU, where there are
// more column tiles than CUs.
// QUANT: every workgroup brings the rows, up to kQuantFew words that its threads
// hold, to 8 bits itself, from their largest magnitudes (1 x 13824 x 5120 33.2 us
// with a launch of a workgroup a row that does it, 16.5 so); the words that are asked
// for are stored by all of them, each a part.
constexpr uint32_t kQuantFew = 16384;
template <int MR, int PB, bool GATED, int W, bool QUANT, class End>
static __global__ void __launch_bounds__(64 * W, PB == 1 || !GATED ? 4 : 2)
    k_rows(const uint32_t* __restrict__ X, WitWeight w0, WitWeight w1, uint32_t m, uint32_t k, uint32_t n, End end,
           WitQuant quant) {
  constexpr int NW = GATED ? 2 : 1, RT = MR <= 4 ? 1 : MR / 4, U = PB > 1 ? 1 : MR > 4 ? 2 : 4;
  constexpr uint32_t kChunk = kRowLds / (4 * MR);  // K per LDS fill
  static_assert(MR > 4 || kChunk / 64 % (W * U) == 0, "a fill ends where the loads in flight start over");
  extern __shared__ __align__(16) int8_t digits[];  // [K / 16][4 MR][16]
  __shared__ int32_t sums[NW][PB][MR][4][32];
  __shared__ uint32_t most[MR];  // QUANT: largest magnitudes
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, ct = blockIdx.x;
  const uint32_t nsteps = (k + kGemmK - 1) / kGemmK, npairs = (nsteps + 1) / 2;
  const uint64_t plane = (uint64_t)((n + kGemmTile - 1) / kGemmTile) * nsteps * kGemmBlockBytes;
  const uint32_t quarter = lane >> 4, col = lane & 15;
  const WitWeight w[2] = {w0, w1};
  v4i b[U][NW][PB][2];
  auto load = [&](int u, uint32_t pair) {
    uint32_t step = 2 * (pair < npairs ? pair : npairs - 1) + quarter / 2;
    step = step < nsteps ? step : nsteps - 1;  // past K: the rows' digits are zero there
    const uint64_t at = ((uint64_t)ct * nsteps + step) * kGemmBlockBytes + (quarter & 1) * 512 + col * 16;
#pragma unroll
    for (int i = 0; i < NW; i++)
#pragma unroll
      for (int q = 0; q < PB; q++)
        if (q == 0 || q < (int)w[i].count) {
#pragma unroll
          for (int h = 0; h < 2; h++)
            b[u][i][q][h] = __builtin_nontemporal_load((const v4i*)(w[i].planes + q * plane + at + 256 * h));
        }
  };
  // four words of a row a thread: quad t of a fill from k0
  auto words = [&](uint32_t t, uint32_t k0, uint32_t left, uint32_t quads, uint32_t (&x)[4]) {
    const uint32_t i = t / quads, kk = t % quads * 4;
    const uint32_t* const from = X + (uint64_t)i * k + k0 + kk;
    if (i < m && kk + 4 <= left) {
      const v4i_word q = *(const v4i_word*)from;
#pragma unroll
      for (int j = 0; j < 4; j++) x[j] = (uint32_t)q[j];
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++) x[j] = i < m && kk + j < left ? from[j] : 0u;
    }
  };
  auto lay_out = [&](uint32_t t, uint32_t quads, const uint32_t (&x)[4]) {
    const uint32_t i = t / quads, kk = t % quads * 4;
    uint32_t d[4], out[4];
#pragma unroll
    for (int j = 0; j < 4; j++) d[j] = digit_bytes(x[j]);
    transpose_bytes(d, out);
#pragma unroll
    for (int p = 0; p < 4; p++)
      *(uint32_t*)(digits + (kk / 16 * (4 * MR) + 4 * i + p) * 16 + kk % 16) = out[p];
  };
  // the first rows' words go out before the weights' loads, which are then in
  // flight while the words are laid out
  constexpr int XQ = QUANT ? (int)(kQuantFew / (256 * W)) : 4;
  uint32_t x[XQ][4];
  {
    const uint32_t left = k < kChunk ? k : kChunk, quads = (left + 63) / 64 * 16;
#pragma unroll
    for (int q = 0; q < XQ; q++)
      if (threadIdx.x + q * 64 * W < MR * quads) words(threadIdx.x + q * 64 * W, 0, left, quads, x[q]);
  }
#pragma unroll
  for (int u = 0; u < U; u++) load(u, wave + u * W);
  for (uint32_t i = threadIdx.x; i < NW * PB * MR * 128; i += blockDim.x) (&sums[0][0][0][0][0])[i] = 0;
  if constexpr (QUANT) {
    if (threadIdx.x < MR) most[threadIdx.x] = 0;
    __syncthreads();
    // The words wait where their digits go to; a loop takes them from there, since a
    // short launch takes as long as its instructions' way from memory (with them in
    // registers and the loop unrolled 20.9 us).
    const uint32_t quads = (k + 63) / 64 * 16;
    auto place = [&](uint32_t t) {
      const uint32_t i = t / quads, kk = t % quads * 4;
      return (uint32_t*)(digits + (kk / 16 * (4 * MR) + 4 * i) * 16 + kk % 16);
    };
#pragma unroll
    for (int q = 0; q < XQ; q++) {
      const uint32_t t = threadIdx.x + q * 64 * W;
      if (t >= MR * quads) break;  // sixteen lanes together, which have the same row
      uint32_t* const to = place(t);
      uint32_t a = 0;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        a = max(a, size_of_word(x[q][j]));
        to[4 * j] = x[q][j];
      }
      a = max(a, (uint32_t)__builtin_amdgcn_mov_dpp((int)a, 0xb1, 0xf, 0xf, true));   // lane ^ 1
      a = max(a, (uint32_t)__builtin_amdgcn_mov_dpp((int)a, 0x4e, 0xf, 0xf, true));   // lane ^ 2
      a = max(a, (uint32_t)__builtin_amdgcn_mov_dpp((int)a, 0x141, 0xf, 0xf, true));  // lane ^ 7
      a = max(a, (uint32_t)__builtin_amdgcn_mov_dpp((int)a, 0x140, 0xf, 0xf, true));  // lane ^ 15
      if ((threadIdx.x & 15) == 0) atomicMax(&most[t / quads], a);
    }
    __syncthreads();
#pragma unroll 1
    for (uint32_t t = threadIdx.x; t < MR * quads; t += 64 * W) {
      const uint32_t i = t / quads, kk = t % quads * 4;
      const Quantizer quantizer(most[i], quant.levels);
      uint32_t* const to = place(t);
      uint32_t b[4];
#pragma unroll
      for (int j = 0; j < 4; j++) b[j] = (uint32_t)quantizer(to[4 * j]);
      to[0] = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u) | __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu);
#pragma unroll
      for (int p = 1; p < 4; p++) to[4 * p] = 0;
      if (quant.words && i < m && t / 64 % gridDim.x == ct) {
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (kk + j < k) quant.words[i * k + kk + j] = word_of((int32_t)b[j]);
      }
    }
    if (quant.scales && ct == 0 && threadIdx.x < m) quant.scales[threadIdx.x] = most[threadIdx.x];
  }
  v4i acc[NW][PB][2][RT];
#pragma unroll
  for (int i = 0; i < NW; i++)
#pragma unroll
    for (int q = 0; q < PB; q++)
#pragma unroll
      for (int h = 0; h < 2; h++)
#pragma unroll
        for (int t = 0; t < RT; t++) acc[i][q][h][t] = v4i{0, 0, 0, 0};
  uint32_t pair = wave;
  for (uint32_t k0 = 0; k0 < k; k0 += kChunk) {
    const uint32_t left = k - k0 < kChunk ? k - k0 : kChunk, fill = (left + 63) / 64 * 64;
    if (k0) __syncthreads();
    uint32_t t = threadIdx.x;
    if (!QUANT && k0 == 0) {
#pragma unroll
      for (int q = 0; q < XQ; q++, t += 64 * W)
        if (t < MR * (fill / 4)) lay_out(t, fill / 4, x[q]);
    }
    for (; !QUANT && t < MR * (fill / 4); t += 64 * W) {
      uint32_t later[4];
      words(t, k0, left, fill / 4, later);
      lay_out(t, fill / 4, later);
    }
    __syncthreads();
    const uint32_t pair0 = k0 / 64, pair1 = pair0 + fill / 64;
    auto multiply = [&](int u) {
      v4i a[RT];
#pragma unroll
      for (int t = 0; t < RT; t++)
        a[t] = *(const v4i*)(digits + ((4 * (pair - pair0) + quarter) * (4 * MR) + (16 * t + col) % (4 * MR)) * 16);
#pragma unroll
      for (int i = 0; i < NW; i++)
#pragma unroll
        for (int q = 0; q < PB; q++)
          if (q == 0 || q < (int)w[i].count) {
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
              for (int t = 0; t < RT; t++)
                acc[i][q][h][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[t], b[u][i][q][h], acc[i][q][h][t], 0, 0, 0);
          }
    };
    // U pairs at a time without a branch between: with one, a wait for any load would be for all
    while (pair + (U - 1) * W < pair1) {
#pragma unroll
      for (int u = 0; u < U; u++) {
        multiply(u);
        load(u, pair + U * W);
        pair += W;
      }
    }
#pragma unroll
    for (int u = 0; u < U - 1; u++)
      if (pair < pair1) {  // the last pairs of all: their loads are out
        multiply(u);
        pair += W;
      }
  }
#pragma unroll
  for (int t = 0; t < RT; t++) {
    const uint32_t row = 4 * t + quarter;
    if (row < MR) {
#pragma unroll
      for (int i = 0; i < NW; i++)
#pragma unroll
        for (int q = 0; q < PB; q++)
#pragma unroll
          for (int h = 0; h < 2; h++)
#pragma unroll
            for (int v = 0; v < 4; v++) atomicAdd(&sums[i][q][row][v][16 * h + col], acc[i][q][h][t][v]);
    }
  }
  const uint32_t r = threadIdx.x / 32, c = threadIdx.x % 32, column = ct * kGemmTile + c;
  const bool ok = r < m && column < n;
  const uint32_t at[1] = {4 * (r * n + column)};  // inside the buffer: few_rows_fit
  const uint32_t row[1] = {r};
  const typename End::Column of_column[1] = {end.column(column, ok)};
  typename End::template Slot<1> slot;
  const typename End::Tile tile = end.tile(0, (uint64_t)m * n);
  if (ok) end.fetch(slot, tile, at, row);
  if constexpr (QUANT) slot.row[0] = most[r < MR ? r : 0];
  __syncthreads();
  if (!ok) return;
  uint32_t z[NW][1];
#pragma unroll
  for (int i = 0; i < NW; i++) {
    uint64_t t = 0;
#pragma unroll
    for (int q = 0; q < PB; q++) {
      const int32_t s[4] = {sums[i][q][r][0][c], sums[i][q][r][1][c], sums[i][q][r][2][c], sums[i][q][r][3][c]};
      t += (uint64_t)digit_sum_mod_p(s) << (8 * q);
    }
    z[i][0] = m31_reduce64(t);
  }
  end.begin(slot, of_column, z);
  end.finish(slot, tile, at);
}

// More rows: the rows' digits are packed first, as operand blocks (gemm.h) in
// two forms, one of which the product reads: plane 0 alone, row r as row r, and
// all four planes interleaved, plane p of row r as row 4 r + p, so that a lane
// of an accumulator holds the four digit sums of its elements.  Words of
// the mask are set where a digit above plane 0 is not zero, and `clear`, the mask
// of the next product on the stream, is zeroed.  A wave takes a block of eight
// rows, four words a lane, and a quad's lanes exchange them so that each stores
// one plane's 16 bytes: loads and stores of whole lines (512 x 13824 words 15 us,
// 3.7 TB/s; 16 words a lane, every load and store a quarter of its lines, 19 us).
// Two or four blocks a wave gain 1 to 3 us there and cost 37 x 1537 0.5 to 1.7.
// Rows past m are left as they are (their sums are not stored).
constexpr uint32_t kMaskWords = 64, kMaskStride = 32;
__device__ __forceinline__ bool wit_four(const uint32_t* mask) {  // the same in every wave
  return __any(mask[kMaskStride * (threadIdx.x & 63)] != 0);
}
// Word p of a quad's lane q and word q of its lane p change places.
__device__ __forceinline__ void quad_transpose(uint32_t (&x)[4]) {
#pragma unroll
  for (int bit = 1; bit <= 2; bit *= 2)
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if (i & bit) continue;
      const bool upper = threadIdx.x & bit;
      const int give = (int)(upper ? x[i] : x[i + bit]);
      const uint32_t take = (uint32_t)(bit == 1 ? __builtin_amdgcn_mov_dpp(give, 0xb1, 0xf, 0xf, true)    // lanes 1 0 3 2
                                                : __builtin_amdgcn_mov_dpp(give, 0x4e, 0xf, 0xf, true));  // 2 3 0 1
      (upper ? x[i] : x[i + bit]) = take;
    }
}
static __global__ void __launch_bounds__(256) k_wit_pack(const uint32_t* __restrict__ X, uint64_t m, uint64_t k,
                                                         uint32_t nsteps, int8_t* __restrict__ one,
                                                         int8_t* __restrict__ four, uint32_t* __restrict__ mask,
                                                         uint32_t* __restrict__ clear) {
  if (blockIdx.x == 0 && threadIdx.x < kMaskWords) clear[kMaskStride * threadIdx.x] = 0;
  const uint32_t q = threadIdx.x & 3, row8 = threadIdx.x >> 2 & 7, half = threadIdx.x >> 5 & 1;
  const uint32_t blk = (uint32_t)__builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));
  const uint32_t rt8 = blk / nsteps, step = blk - rt8 * nsteps;
  const uint64_t row = 8 * (uint64_t)rt8 + row8, k0 = (uint64_t)step * kGemmK + 16 * half + 4 * q;
  const uint32_t* const from = X + row * k + k0;
  uint32_t d[4], w[4];
  if (row < m && k0 + 4 <= k) {
    const v4i_word x = *(const v4i_word*)from;
#pragma unroll
    for (int j = 0; j < 4; j++) d[j] = digit_bytes((uint32_t)x[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++) d[j] = digit_bytes(row < m && k0 + j < k ? from[j] : 0u);
  }
  transpose_bytes(d, w);
  const bool high = __any((w[1] | w[2] | w[3]) != 0);
  quad_transpose(w);  // plane q of the row's 16 words
  if (row < m) {
    const uint4 words = make_uint4(w[0], w[1], w[2], w[3]);
    *(uint4*)(four + (uint64_t)blk * kGemmBlockBytes + 512 * half + 64 * row8 + 16 * q) = words;
    if (!high && q == 0)  // with a higher digit anywhere plane 0 alone is not read
      *(uint4*)(one + ((row >> 5) * nsteps + step) * kGemmBlockBytes + 512 * half + 16 * (row & 31)) = words;
  }
  if (high && (threadIdx.x & 63) == 0) {
    // stores to one address take about 20 ns each, one after another: 64 words
    // on lines of their own, and only while a word is not set
    volatile uint32_t* const word = mask + kMaskStride * (blockIdx.x % kMaskWords);
    if (!*word) *word = 1;
  }
}

// The packing of rows that are brought to 8 bits: a workgroup has two rows, 256
// threads each, and goes over their words twice, the second time back from the end:
// the last of them are in registers and the others in this XCD's cache, where 32
// workgroups of 110 KB fit (four rows a workgroup, the words of 16 turns in registers
// and both loops unrolled: 512 x 13824 24.5 us, 37 x 1537 8.1, most of it the
// instructions' way from memory; so 19.0 and 6.2).  Plane 0 alone is stored, 16 bytes a lane:
// a quad's lanes exchange the words of four turns.  Both masks are zeroed, the product's own
// too: there are no rows of four planes.
constexpr uint32_t kQuantRows = 2;
static __global__ void __launch_bounds__(256 * kQuantRows) k_wit_quantize(const uint32_t* __restrict__ X, uint64_t m, uint64_t k,
                                                                          uint32_t nsteps, int8_t* __restrict__ one,
                                                                          WitQuant quant, uint32_t* __restrict__ mask,
                                                                          uint32_t* __restrict__ clear) {
  __shared__ uint32_t most[kQuantRows][4];
  if (blockIdx.x == 0 && threadIdx.x < kMaskWords) mask[kMaskStride * threadIdx.x] = clear[kMaskStride * threadIdx.x] = 0;
  const uint32_t r = threadIdx.x / 256, t = threadIdx.x % 256, q = threadIdx.x & 3;
  const uint64_t row = (uint64_t)blockIdx.x * kQuantRows + r;
  const uint32_t groups = (nsteps * (kGemmK / 4) + 1023) / 1024;  // of four turns
  const uint32_t* const from = X + (row < m ? row : m - 1) * k;
  const bool whole = k % 4 == 0;  // uniform
  uint32_t x[4][4];
  auto words = [&](uint32_t group) {
    uint32_t at[4];  // k is below 2^31
#pragma unroll
    for (int i = 0; i < 4; i++) at[i] = 4 * ((4 * group + i) * 256 + t);
    if (whole) {
      v4i_word w[4];
#pragma unroll
      for (int i = 0; i < 4; i++) w[i] = *(const v4i_word*)(from + (at[i] < k ? at[i] : 0));
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) x[i][j] = at[i] < k ? (uint32_t)w[i][j] : 0u;
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) x[i][j] = from[at[i] + j < k ? at[i] + j : 0];
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) x[i][j] = at[i] + j < k ? x[i][j] : 0u;
    }
  };
  uint32_t a = 0;
#pragma unroll 1
  for (uint32_t g = 0; g < groups; g++) {
    words(g);
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int j = 0; j < 4; j++) a = max(a, size_of_word(x[i][j]));
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) a = max(a, (uint32_t)__shfl_xor(a, off));
  if ((threadIdx.x & 63) == 0) most[r][t / 64] = a;
  __syncthreads();
  a = max(max(most[r][0], most[r][1]), max(most[r][2], most[r][3]));
  const Quantizer quantizer(a, quant.levels);
  if (row >= m) return;
  if (t == 0) quant.scales[row] = a;
#pragma unroll 1
  for (uint32_t g = groups; g-- > 0;) {
    if (g + 1 < groups) words(g);
    uint32_t bytes[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      uint32_t b[4];
#pragma unroll
      for (int j = 0; j < 4; j++) b[j] = (uint32_t)quantizer(x[i][j]);
      bytes[i] = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u) | __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu);
    }
    if (quant.words) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const uint32_t at = 4 * ((4 * g + i) * 256 + t);
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = word_of((int8_t)(bytes[i] >> (8 * j)));
        uint32_t* const to = quant.words + row * k + at;
        if (whole && at < k) *(v4i_word*)to = v4i_word{(int)w[0], (int)w[1], (int)w[2], (int)w[3]};
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (!whole && at + j < k) to[j] = w[j];
      }
    }
    quad_transpose(bytes);  // lane q of a quad: 16 bytes of turn q
    const uint32_t k16 = ((4 * g + q) * 256 + t) / 4;  // from 16 K on
    if (k16 < 2 * nsteps)
      *(uint4*)(one + ((row >> 5) * nsteps + k16 / 2) * kGemmBlockBytes + 512 * (k16 & 1) + 16 * (row & 31)) =
          make_uint4(bytes[0], bytes[1], bytes[2], bytes[3]);
  }
}

// How a product of several rows is cut, for rows of one plane and of four: row
// groups, K splits and K steps per split.
struct WitPlan {
  uint32_t rtiles, rgroups, splits, steps;
};
struct WitProduct {
  const int8_t *one, *four;  // the packed rows
  const uint32_t* mask;
  WitWeight w[2];
  uint64_t m, n;
  uint32_t nsteps, ctiles, cgroups;
  WitPlan plan[2];
  uint32_t* part;  // [split][matrix][m][n] where there are splits
};

// Up to 64 rows: a stream of the weights.  A workgroup has one column tile of
// each matrix and WR * RT row tiles of 32 (packed) rows; its W waves are WR
// down the rows, RT tiles each, by W / WR that take the K steps in turn,
// operands straight from memory into registers with U steps in flight; the
// waves' sums meet in LDS.  WR goes with the rows' planes (WR1, WR4), so that
// both take the same registers.  Bound by the weights' bytes where there are
// many column tiles (gated 64 x 5120 x 13824 with 14 MB of outputs 36 us, 4.3
// TB/s), by a workgroup's chain of first loads, steps, sums and stores where
// there are few (64 x 5120 x 5120 13 us for 28 MB; 37 x 1537 x 1111 of general
// words 11 us).
template <int RT, int PB, bool GATED, int W, int WR, bool FOUR, class End>
__device__ __forceinline__ void wit_tiles(const WitProduct& g, int32_t* sums, uint32_t rg, uint32_t cg, uint32_t split,
                                          const End& end) {
  constexpr int NW = GATED ? 2 : 1, NB = NW * PB, WK = W / WR, TILES = WR * RT;
  constexpr int U = W == 16 ? (RT + NB <= 2 ? 8 : RT + NB <= 3 ? 6 : 2) : (RT + NB <= 3 ? 6 : RT + NB <= 4 ? 3 : 2);
  const WitPlan& plan = g.plan[FOUR ? 1 : 0];
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t wr = wave % WR, wk = wave / WR;
  const uint32_t s0 = split * plan.steps, s1 = s0 + plan.steps < g.nsteps ? s0 + plan.steps : g.nsteps;
  const uint64_t plane = (uint64_t)g.ctiles * g.nsteps * kGemmBlockBytes;
  const int8_t* ab[RT];
  const int8_t* bb[NW][PB];
#pragma unroll
  for (int i = 0; i < RT; i++) {  // tiles past the edge are the last one again, and not stored
    const uint32_t rt = rg * TILES + wr * RT + i < plan.rtiles ? rg * TILES + wr * RT + i : plan.rtiles - 1;
    ab[i] = (FOUR ? g.four : g.one) + (uint64_t)rt * g.nsteps * kGemmBlockBytes;
  }
#pragma unroll
  for (int x = 0; x < NW; x++)
#pragma unroll
    for (int q = 0; q < PB; q++)
      bb[x][q] = g.w[x].planes + (q < (int)g.w[x].count ? q : 0) * plane + (uint64_t)cg * g.nsteps * kGemmBlockBytes;
  v4i a[U][RT], b[U][NW][PB];
  auto load = [&](int u, uint32_t s) {
    const uint32_t at = (s < s1 ? s : s1 - 1) * kGemmBlockBytes + 16 * lane;  // past the end: again, unused
#pragma unroll
    for (int x = 0; x < NW; x++)
#pragma unroll
      for (int q = 0; q < PB; q++)
        if (q == 0 || q < (int)g.w[x].count)
          b[u][x][q] = WR == 1 ? __builtin_nontemporal_load((const v4i*)(bb[x][q] + at)) : *(const v4i*)(bb[x][q] + at);
#pragma unroll
    for (int i = 0; i < RT; i++) a[u][i] = *(const v4i*)(ab[i] + at);
  };
#pragma unroll
  for (int u = 0; u < U; u++) load(u, s0 + wk + u * WK);
  for (uint32_t i = threadIdx.x; i < TILES * NB * 1024; i += 64 * W) sums[i] = 0;
  v16i acc[RT][NW][PB];
#pragma unroll
  for (int i = 0; i < RT; i++)
#pragma unroll
    for (int x = 0; x < NW; x++)
#pragma unroll
      for (int q = 0; q < PB; q++)
#pragma unroll
        for (int v = 0; v < 16; v++) acc[i][x][q][v] = 0;
  auto multiply = [&](int u) {
#pragma unroll
    for (int x = 0; x < NW; x++)
#pragma unroll
      for (int q = 0; q < PB; q++)
        if (q == 0 || q < (int)g.w[x].count) {
#pragma unroll
          for (int i = 0; i < RT; i++)
            acc[i][x][q] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[u][i], b[u][x][q], acc[i][x][q], 0, 0, 0);
        }
  };
  uint32_t s = s0 + wk;
  // U steps at a time without a branch between: with one, a wait for any load would be for all
#pragma unroll 1
  for (; s + (U - 1) * WK < s1; s += U * WK) {
#pragma unroll
    for (int u = 0; u < U; u++) {
      multiply(u);
      load(u, s + (u + U) * WK);
    }
  }
#pragma unroll
  for (int u = 0; u < U - 1; u++)
    if (s + u * WK < s1) multiply(u);
  // this thread's elements
  constexpr uint32_t ROWS = FOUR ? 8 : 32;  // of a tile
  constexpr int ALL = TILES * ROWS * 32, E = ALL <= 64 * W ? 1 : ALL / (64 * W);
  static_assert(E * 64 * W == ALL || E == 1, "whole elements");
  const uint32_t c = threadIdx.x % 32;
  const uint64_t col = (uint64_t)cg * 32 + c, first = (uint64_t)rg * (TILES * ROWS) * g.n + (uint64_t)cg * 32;
  uint32_t at[E], rows[E], row[E];
#pragma unroll
  for (int e = 0; e < E; e++) {
    rows[e] = threadIdx.x / 32 + e * 2 * W;
    row[e] = rg * (TILES * ROWS) + rows[e];
    at[e] = rows[e] < TILES * ROWS && col < g.n ? 4 * (rows[e] * (uint32_t)g.n + c) : kOutside;
  }
  typename End::Column of_column[E];
  same_column(of_column, end.column(col, col < g.n));
  typename End::template Slot<E> slot;
  const typename End::Tile tile = end.tile(first, plan.splits == 1 ? g.m * g.n : 0);
  end.fetch(slot, tile, at, row);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < RT; i++)
#pragma unroll
    for (int x = 0; x < NW; x++)
#pragma unroll
      for (int q = 0; q < PB; q++)
#pragma unroll
        for (int v = 0; v < 16; v++)
          atomicAdd(&sums[(((wr * RT + i) * NB + x * PB + q) * 32 + 8 * (v / 4) + 4 * (lane >> 5) + v % 4) * 32 + (lane & 31)],
                    acc[i][x][q][v]);
  __syncthreads();
  uint32_t z[NW][E];
#pragma unroll
  for (int e = 0; e < E; e++) {
    const uint32_t r = rows[e] < TILES * ROWS ? rows[e] : 0;
#pragma unroll
    for (int x = 0; x < NW; x++) {
      uint64_t t = 0;
#pragma unroll
      for (int q = 0; q < PB; q++) {
        const int32_t* const from = sums + (r / ROWS * NB + x * PB + q) * 1024 + c;
        uint32_t one;
        if constexpr (FOUR) {
          const uint32_t r4 = 4 * (r % 8);
          const int32_t d[4] = {from[r4 * 32], from[r4 * 32 + 32], from[r4 * 32 + 64], from[r4 * 32 + 96]};
          one = digit_sum_mod_p(d);
        } else {
          one = gemm_mod_p(from[r % 32 * 32]);
        }
        t += (uint64_t)one << (8 * q);
      }
      z[x][e] = m31_reduce64(t);
    }
  }
  if (plan.splits == 1) {
    end.begin(slot, of_column, z);
    end.finish(slot, tile, at);
  } else {
    wit_parts(g.part, split, first, g.m * g.n, at, z);
  }
}
template <int RT, int PB, bool GATED, int W, int WR1, int WR4, class End>
static __global__ void __launch_bounds__(64 * W) k_wit_tiles(WitProduct g, uint32_t rgroups, End end) {
  __shared__ int32_t sums[(WR1 > WR4 ? WR1 : WR4) * RT * PB * (GATED ? 2 : 1) * 1024];
  const bool four = wit_four(g.mask);
  const WitPlan& plan = g.plan[four ? 1 : 0];
  uint32_t rg, cg;
  if (!gemm_group(rgroups, g.cgroups, rg, cg) || rg >= plan.rgroups || blockIdx.y >= plan.splits) return;  // uniform
  if (four)
    wit_tiles<RT, PB, GATED, W, WR4, true>(g, sums, rg, cg, blockIdx.y, end);
  else
    wit_tiles<RT, PB, GATED, W, WR1, false>(g, sums, rg, cg, blockIdx.y, end);
}

// Some hundred rows of one plane by weights of one plane: a workgroup has RT row tiles
// by CT column tiles and all of K, and its eight waves take the K steps in turn, each
// all of the tiles, straight from memory into registers.  No operand is read twice by
// a workgroup, nothing waits for another wave until the waves' sums meet in LDS, and
// no parts go through memory: where k_wit_blocks' 256 x 256 leave most CUs without a
// workgroup or split K (scales, no residual, operands in the caches: 512 x 5120 x 5120
// 38 us with the join, 25 so; 512 x 13824 x 5120 58 and 47; 700 x 576 x 1536 27 and 8; with
// the packing and operands from memory 512 x 5120 x 5120 40 and 29, 512 x 13824 x 5120,
// quantized, 82.6 and 78.8).  Between start and end bound by a CU's way to its
// second-level cache, 7 KB a K step at 78 GB/s (two, three or four steps in flight, 2 x 4
// and 2 x 5 tiles: the same); over the whole kernel the matrix cores are busy two fifths
// of the cycles, as all the waves' sums meet at the end and nothing is there at the start.
template <int RT, int CT, class End>
__device__ __forceinline__ void wit_wide(const WitProduct& g, int32_t* sums, uint32_t rg, uint32_t cg, const End& end) {
  constexpr int W = 8, U = 2;
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int8_t *ab[RT], *bb[CT];  // tiles past an edge are the last one again, and not stored
#pragma unroll
  for (int i = 0; i < RT; i++)
    ab[i] = g.one + (uint64_t)umin32(rg * RT + i, g.plan[0].rtiles - 1) * g.nsteps * kGemmBlockBytes;
#pragma unroll
  for (int j = 0; j < CT; j++)
    bb[j] = g.w[0].planes + (uint64_t)umin32(cg * CT + j, g.ctiles - 1) * g.nsteps * kGemmBlockBytes;
  v4i a[U][RT], b[U][CT];
  auto load = [&](int u, uint32_t s) {
    const uint32_t at = umin32(s, g.nsteps - 1) * kGemmBlockBytes + 16 * lane;  // past the end: again, unused
#pragma unroll
    for (int j = 0; j < CT; j++) b[u][j] = *(const v4i*)(bb[j] + at);
#pragma unroll
    for (int i = 0; i < RT; i++) a[u][i] = *(const v4i*)(ab[i] + at);
  };
#pragma unroll
  for (int u = 0; u < U; u++) load(u, wave + u * W);
#pragma unroll 1
  for (uint32_t i = threadIdx.x; i < RT * CT * 256; i += 64 * W) ((v4i*)sums)[i] = v4i{0, 0, 0, 0};
  v16i acc[RT][CT];
#pragma unroll
  for (int i = 0; i < RT; i++)
#pragma unroll
    for (int j = 0; j < CT; j++)
#pragma unroll
      for (int v = 0; v < 16; v++) acc[i][j][v] = 0;
  auto multiply = [&](int u) {
#pragma unroll
    for (int j = 0; j < CT; j++)
#pragma unroll
      for (int i = 0; i < RT; i++) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[u][i], b[u][j], acc[i][j], 0, 0, 0);
  };
  uint32_t s = wave;
  // U steps at a time without a branch between: with one, a wait for any load would be for all
#pragma unroll 1
  for (; s + (U - 1) * W < g.nsteps; s += U * W) {
#pragma unroll
    for (int u = 0; u < U; u++) {
      multiply(u);
      load(u, s + (u + U) * W);
    }
  }
#pragma unroll
  for (int u = 0; u < U - 1; u++)
    if (s + u * W < g.nsteps) multiply(u);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < RT; i++)
#pragma unroll
    for (int j = 0; j < CT; j++)
#pragma unroll
      for (int v = 0; v < 16; v++)
        atomicAdd(&sums[((j * RT + i) * 32 + 8 * (v / 4) + 4 * (lane >> 5) + v % 4) * 32 + (lane & 31)], acc[i][j][v]);
  __syncthreads();
  // the end, a column tile at a time
  constexpr int E = RT * 1024 / (64 * W);
  const uint32_t c = threadIdx.x % 32, r0 = threadIdx.x / 32;
#pragma unroll 1
  for (int j = 0; j < CT; j++) {
    const uint64_t col0 = ((uint64_t)cg * CT + j) * 32, col = col0 + c;
    if (col0 >= g.n) return;  // uniform
    const typename End::Tile tile = end.tile((uint64_t)rg * (RT * 32) * g.n + col0, g.m * g.n);
    uint32_t at[E], row[E], z[1][E];
#pragma unroll
    for (int e = 0; e < E; e++) {
      const uint32_t r = r0 + e * 2 * W;
      row[e] = rg * (RT * 32) + r;
      at[e] = col < g.n ? 4 * (r * (uint32_t)g.n + c) : kOutside;
      z[0][e] = gemm_mod_p(sums[(j * RT * 32 + r) * 32 + c]);
    }
    typename End::Column of_column[E];
    same_column(of_column, end.column(col, col < g.n));
    typename End::template Slot<E> slot;
    end.fetch(slot, tile, at, row);
    end.begin(slot, of_column, z);
    end.finish(slot, tile, at);
  }
}

// Between a wave's stores to LDS and its lanes' reads of each other's words, and
// between those reads and the next stores: the wave's LDS instructions run in
// order, but the compiler sees one lane's addresses, which it may prove apart
// and put in another order.
__device__ __forceinline__ void wave_exchange() {
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

// More rows: 8 row tiles of (packed) rows by 8 column tiles of the weights (4 of
// each of two matrices) a workgroup, through LDS.  Both operands lie in memory
// as the matrix cores take them, so a tile's K step is 1 KB that one wave
// copies and any wave reads back without bank conflicts.  A stage is four K
// steps, 64 KB; while a stage is multiplied the next goes from registers to the
// other half of LDS and the one after it is on its way from memory.  Eight
// waves, two down the rows (four tiles each) by four across (two tiles, or one
// of each matrix): 6 KB from LDS feed 8 matrix instructions of 32 cycles.
// Bound by the matrix cores: 512 x 13824 x 5120 of general rows (2.9e11
// operations) 133 to 144 us with its parts' stores, 2.0 to 2.2 POP/s, where a
// library product of 8192^3 reaches 2.17; gated 512 x 5120 x 13824 of one plane
// 93 to 96 us, about 15 of them the 7 M table look-ups at the end (a line each).
constexpr int kBlockStage = 4;  // K steps
// Weights of several planes: a column tile's four planes are four of the eight,
// two to a wave, whose sums two waves bring together.
template <int PB, bool GATED, bool FOUR, class End>
__device__ __forceinline__ void wit_block(const WitProduct& g, v4i* lds, uint32_t rg, uint32_t cg, uint32_t split,
                                          const End& end) {
  constexpr int NW = GATED ? 2 : 1, CT = 8 / (NW * PB);  // column tiles of a workgroup
  static_assert(!GATED || PB == 1, "two matrices of one plane");
  const WitPlan& plan = g.plan[FOUR ? 1 : 0];
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t s0 = split * plan.steps, s1 = s0 + plan.steps < g.nsteps ? s0 + plan.steps : g.nsteps;
  // this wave copies the 8 row tiles (even waves) or column tiles (odd) of step wave / 2 of each stage
  const int8_t* from[8];
#pragma unroll
  for (int i = 0; i < 8; i++) {  // tiles past the edges are the last one again, and not stored
    if (wave & 1) {
      const uint32_t ct = cg * CT + i / (NW * PB), t = ct < g.ctiles ? ct : g.ctiles - 1;
      const uint32_t q = i % PB;  // a plane that the weight does not have is zero: no pointer
      from[i] = q && q >= g.w[0].count ? nullptr
                                       : g.w[i % NW].planes + ((uint64_t)q * g.ctiles + t) * g.nsteps * kGemmBlockBytes;
    } else {
      const uint32_t rt = rg * 8 + i, t = rt < plan.rtiles ? rt : plan.rtiles - 1;
      from[i] = (FOUR ? g.four : g.one) + (uint64_t)t * g.nsteps * kGemmBlockBytes;
    }
  }
  v4i in[8];
  auto load = [&](int i, uint32_t s) {  // tile i of the stage from step s
    const uint32_t step = s + wave / 2, at = (step < s1 ? step : s1 - 1) * kGemmBlockBytes + 16 * lane;
    if (PB > 1 && !from[i]) in[i] = v4i{0, 0, 0, 0};  // uniform
    else in[i] = *(const v4i*)(from[i] + at);
  };
  auto put = [&](int i, uint32_t half) { lds[(half * 8 * kBlockStage * 2 + wave * 8 + i) * 64 + lane] = in[i]; };
  const uint32_t wr = wave & 1, wc = wave >> 1;
  v16i acc[4][2];
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int j = 0; j < 2; j++)
#pragma unroll
      for (int v = 0; v < 16; v++) acc[i][j][v] = 0;
  v4i a[2][4], b[2][2];  // a K step's operands, and the next one's
  auto read = [&](int to, uint32_t half, int k, int o) {  // operand o of six
    const v4i* const at = lds + (half * 8 * kBlockStage * 2 + k * 16) * 64 + lane;
    if (o < 2) b[to][o] = at[(8 + wc * 2 + o) * 64];
    else a[to][o - 2] = at[(wr * 4 + o - 2) * 64];
  };
  auto multiply = [&](int of, int t) {  // product t of eight
    acc[t / 2][t % 2] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[of][t / 2], b[of][t % 2], acc[t / 2][t % 2], 0, 0, 0);
  };
#pragma unroll
  for (int i = 0; i < 8; i++) load(i, s0);
#pragma unroll
  for (int i = 0; i < 8; i++) put(i, 0);
#pragma unroll
  for (int i = 0; i < 8; i++) load(i, s0 + kBlockStage);
  __syncthreads();
  uint32_t half = 0, s = s0;
#pragma unroll
  for (int o = 0; o < 6; o++) read(0, 0, 0, o);
  // Between a K step's products go the next step's operands, one after each,
  // and a third of the next stage's way to LDS: issued together they hold the
  // matrix cores up, as all eight waves do it at the same time.  The barrier
  // comes before a stage's last step, whose operands are there, so that the
  // next stage's first are read under that step's products.
#pragma unroll 1
  for (; s + kBlockStage <= s1; s += kBlockStage, half ^= 1) {
#pragma unroll
    for (int k = 0; k < kBlockStage; k++) {
      const bool turn = k + 1 == kBlockStage;
      if (turn) __syncthreads();
#pragma unroll
      for (int t = 0; t < 8; t++) {
        multiply(k & 1, t);
        if (t < 6) read((k + 1) & 1, turn ? half ^ 1 : half, turn ? 0 : k + 1, t);
        const int i = 3 * k + t / 2 - 1;
        if (!turn && t >= 2 && t % 2 == 1 && i < 8) {
          put(i, half ^ 1);
          load(i, s + 2 * kBlockStage);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
#pragma unroll 1
  for (int k = 0; s + k < s1; k++) {  // a last, shorter stage
#pragma unroll
    for (int o = 0; o < 6; o++) read(0, half, k, o);
#pragma unroll
    for (int t = 0; t < 8; t++) multiply(0, t);
  }
  // The end, half of a wave's tiles at a time: through its 16 KB of LDS into
  // rows, eight elements a lane and turn.
  __syncthreads();
  constexpr uint32_t ROWS = FOUR ? 8 : 32, TI = 4 / NW;  // of a tile; tiles down the rows at a time
  int32_t* const mine = (int32_t*)lds + wave * 4096;
  if constexpr (PB > 1) {
    // two row tiles at a time; of a pair of waves with the same rows and column
    // tile, one has planes 0 and 1 of both, one 2 and 3, and each ends one
    constexpr int E = 4;
    const uint32_t c = lane & 31, hi = lane >> 5, odd = wc & 1;
    const int32_t* const low = (const int32_t*)lds + (wave & ~2u) * 4096;
    const uint64_t col0 = ((uint64_t)cg * CT + wc / 2) * 32;
    typename End::Column of_column[E];
    same_column(of_column, end.column(col0 + c, col0 + c < g.n));
#pragma unroll
    for (uint32_t part = 0; part < 2; part++) {
      if (part) __syncthreads();
#pragma unroll
      for (uint32_t t = 0; t < 4; t++)
#pragma unroll
        for (int v = 0; v < 16; v++)
          mine[t * 1024 + (8 * (v / 4) + 4 * hi + v % 4) * 32 + c] = acc[part * 2 + t / 2][t % 2][v];
      __syncthreads();
      const uint32_t row0 = (rg * 8 + wr * 4 + part * 2 + odd) * ROWS;
      const uint64_t first = (uint64_t)row0 * g.n + col0;
      const typename End::Tile tile = end.tile(plan.splits == 1 ? first : 0, plan.splits == 1 ? g.m * g.n : 0);
#pragma unroll 1
      for (uint32_t r0 = 0; r0 < ROWS; r0 += 2 * E) {
        uint32_t at[E], row[E], z[1][E];
#pragma unroll
        for (int e = 0; e < E; e++) {
          const uint32_t r = r0 + 2 * e + hi;
          row[e] = row0 + r;
          at[e] = col0 + c < g.n ? 4 * (r * (uint32_t)g.n + c) : kOutside;
          uint64_t sum = 0;
#pragma unroll
          for (int q = 0; q < PB; q++) {
            const int32_t* const t = low + (q / 2) * (2 * 4096) + (odd * 2 + q % 2) * 1024 + c;
            uint32_t one;
            if constexpr (FOUR) {
              const int32_t d[4] = {t[r * 128], t[r * 128 + 32], t[r * 128 + 64], t[r * 128 + 96]};
              one = digit_sum_mod_p(d);
            } else {
              one = gemm_mod_p(t[r * 32]);
            }
            sum += (uint64_t)one << (8 * q);
          }
          z[0][e] = m31_reduce64(sum);
        }
        if (plan.splits == 1) {
          typename End::template Slot<E> slot;
          end.fetch(slot, tile, at, row);
          end.begin(slot, of_column, z);
          end.finish(slot, tile, at);
        } else {
          wit_parts(g.part, split, first, g.m * g.n, at, z);
        }
      }
    }
    return;
  }
  constexpr int E = 8;
#pragma unroll
  for (uint32_t part = 0; part < 2; part++) {
    if (part) wave_exchange();
#pragma unroll
    for (uint32_t t = 0; t < 4; t++) {
      const v16i& from = GATED ? acc[part * TI + t / 2][t % 2] : acc[t][part];
#pragma unroll
      for (int v = 0; v < 16; v++) mine[t * 1024 + (8 * (v / 4) + 4 * (lane >> 5) + v % 4) * 32 + (lane & 31)] = from[v];
    }
    wave_exchange();
    const uint32_t tile0 = rg * 8 + wr * 4 + (GATED ? part * TI : 0), c = lane & 31, hi = lane >> 5;
    const uint64_t col0 = ((uint64_t)cg * CT + (GATED ? wc : wc * 2 + part)) * 32;
    const uint64_t first = (uint64_t)tile0 * ROWS * g.n + col0;
    typename End::Column of_column[E];
    same_column(of_column, end.column(col0 + c, col0 + c < g.n));
    const uint32_t pitch = 8 * (uint32_t)g.n;  // bytes of two rows
    const uint32_t at0 = col0 + c < g.n ? 4 * (hi * (uint32_t)g.n + c) : kOutside;
    const int32_t* const from = mine + hi * (FOUR ? 128 : 32) + c;
    // rows r0 + 2 e + hi, r0 a multiple of 16
    auto places = [&](uint32_t r0, uint32_t (&at)[E]) {
#pragma unroll
      for (int e = 0; e < E; e++) at[e] = at0 == kOutside ? kOutside : at0 + (r0 / 2 + e) * pitch;
    };
    auto values = [&](uint32_t r0, uint32_t (&z)[NW][E]) {
#pragma unroll
      for (int e = 0; e < E; e++)
#pragma unroll
        for (int x = 0; x < NW; x++) {
          if constexpr (FOUR) {  // a tile has eight rows, of four planes each
            const int32_t* const t = from + (r0 / 8 * NW + e / 4 * NW + x) * 1024 + e % 4 * 256;
            const int32_t d[4] = {t[0], t[32], t[64], t[96]};
            z[x][e] = digit_sum_mod_p(d);
          } else {
            z[x][e] = gemm_mod_p(from[(r0 / 32 * NW + x) * 1024 + r0 % 32 * 32 + e * 64]);
          }
        }
    };
    constexpr uint32_t ALL = TI * ROWS;
    if (plan.splits == 1) {  // two turns at a time, the second's loads before the first's stores
      const typename End::Tile tile = end.tile(first, g.m * g.n);
      typename End::template Slot<E> slot[2];
      auto begin = [&](int i, uint32_t r0) {
        uint32_t at[E], row[E], z[NW][E];
        places(r0, at);
#pragma unroll
        for (int e = 0; e < E; e++) row[e] = tile0 * ROWS + r0 + 2 * e + hi;
        end.fetch(slot[i], tile, at, row);
        values(r0, z);
        end.begin(slot[i], of_column, z);
      };
      auto finish = [&](int i, uint32_t r0) {
        uint32_t at[E];
        places(r0, at);
        end.finish(slot[i], tile, at);
      };
      static_assert(ALL % (4 * E) == 0 || ALL == 2 * E, "two turns");
      begin(0, 0);
#pragma unroll 1
      for (uint32_t r0 = 0; r0 < ALL; r0 += 4 * E) {
        if (ALL > 2 * E) begin(1, r0 + 2 * E);
        finish(0, r0);
        if (r0 + 4 * E < ALL) begin(0, r0 + 4 * E);
        if (ALL > 2 * E) finish(1, r0 + 2 * E);
      }
    } else {
#pragma unroll 1
      for (uint32_t r0 = 0; r0 < ALL; r0 += 2 * E) {
        uint32_t at[E], z[NW][E];
        places(r0, at);
        values(r0, z);
        wit_parts(g.part, split, first, g.m * g.n, at, z);
      }
    }
  }
}
// As gemm_group, over the groups and K splits that a product has, in one grid
// dimension: those that it does not have come last, where they wait for no one.
__device__ __forceinline__ bool wit_group(const WitPlan& plan, uint32_t cgroups, uint32_t& rg, uint32_t& cg,
                                          uint32_t& split) {
  const uint32_t groups = plan.rgroups * cgroups, per_xcd = (groups + 7) / 8;
  split = blockIdx.x / (8 * per_xcd);
  const uint32_t x = blockIdx.x % (8 * per_xcd), at = (x & 7) * per_xcd + (x >> 3);
  rg = at % plan.rgroups;
  cg = at / plan.rgroups;
  return split < plan.splits && at < groups;
}
template <int PB, bool GATED, class End>
static __global__ void __launch_bounds__(512) k_wit_blocks(WitProduct g, End end) {
  __shared__ v4i lds[2 * 16 * kBlockStage * 64];
  const bool four = wit_four(g.mask);
  const WitPlan& plan = g.plan[four ? 1 : 0];
  uint32_t rg, cg, split;
  if (!wit_group(plan, g.cgroups, rg, cg, split)) return;  // uniform
  if (four)
    wit_block<PB, GATED, true>(g, lds, rg, cg, split, end);
  else
    wit_block<PB, GATED, false>(g, lds, rg, cg, split, end);
}
template <int RT, int CT, class End>
static __global__ void __launch_bounds__(512) k_wit_wide(WitProduct g, End end) {
  __shared__ v4i lds[2 * 16 * kBlockStage * 64];
  static_assert(RT * CT * 4096 <= sizeof(lds), "the waves' sums");
  const bool four = wit_four(g.mask);
  uint32_t rg, cg, split;
  if (!wit_group(g.plan[four ? 1 : 0], four ? g.cgroups : (g.ctiles + CT - 1) / CT, rg, cg, split)) return;  // uniform
  if (four)
    wit_block<1, false, true>(g, lds, rg, cg, split, end);
  else
    wit_wide<RT, CT>(g, (int32_t*)lds, rg, cg, end);
}
// 65 to 256 rows: rows of one plane are still a stream of the weights
// (wit_tiles, all of the rows in a workgroup), rows of four are blocks.
template <int RT, int WR, bool GATED, class End>
static __global__ void __launch_bounds__(512) k_wit_mixed(WitProduct g, End end) {
  __shared__ v4i lds[2 * 16 * kBlockStage * 64];
  static_assert(WR * RT * (GATED ? 2 : 1) * 4096 <= sizeof(lds), "the waves' sums");
  const bool four = wit_four(g.mask);
  const WitPlan& plan = g.plan[four ? 1 : 0];
  uint32_t rg, cg, split;
  if (!wit_group(plan, four ? g.cgroups : g.ctiles, rg, cg, split)) return;  // uniform
  if (four)
    wit_block<1, GATED, true>(g, lds, rg, cg, split, end);
  else
    wit_tiles<RT, 1, GATED, 8, WR, false>(g, (int32_t*)lds, rg, cg, 0, end);
}

// The end of a product whose K was split: four elements a thread, four parts'
// loads together.  Bound by the parts' way through memory: 512 x 5120 of three
// parts 10.6 us, 3.9 TB/s (two at a time and the residual behind them 15.4).
constexpr uint32_t kJoinParts = 4;
template <bool GATED, class End>
static __global__ void __launch_bounds__(256) k_wit_join(WitProduct g, End end) {
  const uint32_t splits = g.plan[wit_four(g.mask) ? 1 : 0].splits;
  if (splits == 1) return;  // done where it was computed
  constexpr int NW = GATED ? 2 : 1;
  const uint64_t count = g.m * g.n;
  constexpr int E = 4;
  for (uint64_t first = (uint64_t)blockIdx.x * (256 * E); first < count; first += (uint64_t)gridDim.x * (256 * E)) {
    const uint32_t row0 = (uint32_t)(first / g.n), column0 = (uint32_t)(first - (uint64_t)row0 * g.n);
    uint64_t t[NW][E] = {};
    uint32_t at[E], row[E], z[NW][E];
    typename End::Column of_column[E];
#pragma unroll
    for (int e = 0; e < E; e++) {
      const uint32_t in = column0 + threadIdx.x + 256 * e;
      row[e] = row0 + in / (uint32_t)g.n;
      of_column[e] = end.column(in % (uint32_t)g.n, true);
      at[e] = 4 * (threadIdx.x + 256 * e);
    }
    typename End::template Slot<E> slot;
    const typename End::Tile tile = end.tile(first, count);
    end.fetch(slot, tile, at, row);
    for (uint32_t s0 = 0; s0 < splits; s0 += kJoinParts) {  // those past the last have no bytes and read zero
      uint32_t part[kJoinParts][NW][E];
#pragma unroll
      for (uint32_t s = 0; s < kJoinParts; s++)
#pragma unroll
        for (int x = 0; x < NW; x++) {
          const WitBuffer from =
              wit_buffer(g.part + (uint64_t)((s0 + s) * NW + x) * count, first, s0 + s < splits ? count : 0);
#pragma unroll
          for (int e = 0; e < E; e++) part[s][x][e] = wit_read(from, at[e]);
        }
#pragma unroll
      for (uint32_t s = 0; s < kJoinParts; s++)
#pragma unroll
        for (int x = 0; x < NW; x++)
#pragma unroll
          for (int e = 0; e < E; e++) t[x][e] += part[s][x][e];
    }
#pragma unroll
    for (int x = 0; x < NW; x++)
#pragma unroll
      for (int e = 0; e < E; e++) z[x][e] = m31_reduce64(t[x][e]);
    end.begin(slot, of_column, z);
    end.finish(slot, tile, at);
  }
}

// One thread per element, behind products of their own.
template <bool GATED, class End>
static __global__ void __launch_bounds__(256) k_wit_end(const uint32_t* __restrict__ z0, const uint32_t* __restrict__ z1,
                                                        uint64_t count, uint64_t n, End end) {
  for (uint64_t first = (uint64_t)blockIdx.x * 256; first < count; first += (uint64_t)gridDim.x * 256) {
    const uint64_t i = first + threadIdx.x < count ? first + threadIdx.x : count - 1;
    const uint64_t r = i / n;
    const uint32_t at[1] = {4 * threadIdx.x}, row[1] = {(uint32_t)r};
    const typename End::Column of_column[1] = {end.column(i - r * n, true)};
    uint32_t z[GATED ? 2 : 1][1];
    z[0][0] = z0[i];
    if constexpr (GATED) z[1][0] = z1[i];
    typename End::template Slot<1> slot;
    const typename End::Tile tile = end.tile(first, count);
    end.fetch(slot, tile, at, row);
    end.begin(slot, of_column, z);
    end.finish(slot, tile, at);
  }
}

}  // namespace gkr
