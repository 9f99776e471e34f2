// The witness operators' kernels: products of canonical M31 words by digit
// planes on the matrix cores (gemm.h), with the element-wise work behind them
// (bias, activation, residual, the gate's product) in the same launch.
#pragma once
#include <stdint.h>

#include "field.h"
#include "gemm.h"

namespace gkr {

// act(z): table == nullptr and relu == 0 is z itself; the table's entry at
// z mod 2^log is what the LogUp layer proves (mask = 2^log - 1).
struct ActArg {
  const uint32_t* table;
  uint32_t mask, relu;
};
__device__ __forceinline__ uint32_t activate(const ActArg& a, uint32_t z) {
  if (a.table) return a.table[z & a.mask];
  return a.relu && z > (P >> 1) ? 0u : z;
}

// What happens to a sum of the product (fused) or a pair of sums (gated).
struct FusedEnd {
  ActArg act;
  const uint32_t* bias;      // n
  const uint32_t* residual;  // m x n; may be out (read by the thread that writes the element)
  uint32_t* pre;
  uint32_t* out;
};
__device__ __forceinline__ void fused_end(const FusedEnd& e, uint64_t at, uint64_t col, uint32_t z) {
  if (e.bias) z = m31_add(z, e.bias[col]);
  if (e.pre) e.pre[at] = z;
  uint32_t y = activate(e.act, z);
  if (e.residual) y = m31_add(y, e.residual[at]);
  e.out[at] = y;
}
struct GatedEnd {
  ActArg act;
  uint32_t *gate, *act_out, *up, *out;
};
__device__ __forceinline__ void gated_end(const GatedEnd& e, uint64_t at, uint32_t g, uint32_t u) {
  const uint32_t a = activate(e.act, g);
  if (e.gate) e.gate[at] = g;
  if (e.act_out) e.act_out[at] = a;
  if (e.up) e.up[at] = u;
  e.out[at] = m31_mul(a, u);
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

// One to four rows.  The rows' digit planes are rows of one product: row' 4 i
// + p of the 16 that v_mfma_i32_16x16x64_i8 takes is plane p of row i, so
// general words cost no more than int8-range ones, and lane 16 i + c of the
// accumulator holds the four digit sums of row i, column c.
//
// A workgroup has 32 columns of the weights and all of K: it lays the rows'
// digits out in LDS (kRowLds bytes at a time) and its waves take K pairs of 32
// in turn, a pair's 2 KB per plane in two loads, U pairs in flight; then the
// waves' sums meet in LDS (integers: any order gives the same).  No packing
// launch, no partial sums in memory: bound by the weights' bytes (packing, the
// product, its splits' sum and the epilogue as launches of their own, then
// this: 1 x 576 x 192 11.4 -> 4.7 us, 1 x 13824 x 5120 39.1 -> 16.2, 4.4 TB/s;
// gated 1 x 5120 x 13824 47.0 -> 28.7, 4.9 TB/s, where a copy reaches 4.8).
constexpr uint32_t kRowWaves = 16;
constexpr uint32_t kRowLds = 65536;
template <int MR, int PB, bool GATED, class End>
static __global__ void __launch_bounds__(64 * kRowWaves) k_rows(const uint32_t* __restrict__ X, WitWeight w0, WitWeight w1,
                                                                uint32_t m, uint32_t k, uint32_t n, End end) {
  constexpr int NW = GATED ? 2 : 1, U = PB == 1 ? 4 : 1;
  constexpr uint32_t kChunk = kRowLds / (4 * MR);  // K per LDS fill
  static_assert(kChunk / 64 % (kRowWaves * U) == 0, "a fill ends where the loads in flight start over");
  extern __shared__ __align__(16) int8_t digits[];  // [K / 16][4 MR][16]
  __shared__ int32_t sums[NW][PB][MR][4][32];
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
#pragma unroll
  for (int u = 0; u < U; u++) load(u, wave + u * kRowWaves);
  for (uint32_t i = threadIdx.x; i < NW * PB * MR * 128; i += blockDim.x) (&sums[0][0][0][0][0])[i] = 0;
  v4i acc[NW][PB][2];
#pragma unroll
  for (int i = 0; i < NW; i++)
#pragma unroll
    for (int q = 0; q < PB; q++)
#pragma unroll
      for (int h = 0; h < 2; h++) acc[i][q][h] = v4i{0, 0, 0, 0};
  uint32_t pair = wave;
  for (uint32_t k0 = 0; k0 < k; k0 += kChunk) {
    const uint32_t left = k - k0 < kChunk ? k - k0 : kChunk, fill = (left + 63) / 64 * 64;
    if (k0) __syncthreads();
    for (uint32_t t = threadIdx.x; t < MR * (fill / 4); t += blockDim.x) {
      const uint32_t i = t / (fill / 4), kk = t % (fill / 4) * 4;
      uint32_t d[4], out[4];
#pragma unroll
      for (int j = 0; j < 4; j++)
        d[j] = i < m && kk + j < left ? digit_bytes(X[(uint64_t)i * k + k0 + kk + j]) : 0u;
      transpose_bytes(d, out);
#pragma unroll
      for (int p = 0; p < 4; p++)
        *(uint32_t*)(digits + (kk / 16 * (4 * MR) + 4 * i + p) * 16 + kk % 16) = out[p];
    }
    __syncthreads();
    const uint32_t pair0 = k0 / 64, pair1 = pair0 + fill / 64;
    while (pair < pair1) {
#pragma unroll
      for (int u = 0; u < U; u++) {
        if (pair < pair1) {  // uniform in the wave
          const v4i a = *(const v4i*)(digits + ((4 * (pair - pair0) + quarter) * (4 * MR) + col % (4 * MR)) * 16);
#pragma unroll
          for (int i = 0; i < NW; i++)
#pragma unroll
            for (int q = 0; q < PB; q++)
              if (q == 0 || q < (int)w[i].count) {
#pragma unroll
                for (int h = 0; h < 2; h++)
                  acc[i][q][h] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b[u][i][q][h], acc[i][q][h], 0, 0, 0);
              }
          load(u, pair + U * kRowWaves);
          pair += kRowWaves;
        }
      }
    }
  }
  if (quarter < MR) {
#pragma unroll
    for (int i = 0; i < NW; i++)
#pragma unroll
      for (int q = 0; q < PB; q++)
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
          for (int v = 0; v < 4; v++) atomicAdd(&sums[i][q][quarter][v][16 * h + col], acc[i][q][h][v]);
  }
  __syncthreads();
  const uint32_t r = threadIdx.x / 32, c = threadIdx.x % 32, column = ct * kGemmTile + c;
  if (r >= m || column >= n) return;
  uint32_t z[NW];
#pragma unroll
  for (int i = 0; i < NW; i++) {
    uint64_t t = 0;
#pragma unroll
    for (int q = 0; q < PB; q++) {
      const int32_t s[4] = {sums[i][q][r][0][c], sums[i][q][r][1][c], sums[i][q][r][2][c], sums[i][q][r][3][c]};
      t += (uint64_t)digit_sum_mod_p(s) << (8 * q);
    }
    z[i] = m31_reduce64(t);
  }
  if constexpr (GATED)
    gated_end(end, (uint64_t)r * n + column, z[0], z[1]);
  else
    fused_end(end, (uint64_t)r * n + column, column, z[0]);
}

// One thread per element, behind the products.
static __global__ void k_fused_end(const uint32_t* __restrict__ z, uint64_t count, uint64_t n, FusedEnd e) {
  for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < count; i += (uint64_t)gridDim.x * blockDim.x)
    fused_end(e, i, i % n, z[i]);
}
static __global__ void k_gated_end(const uint32_t* __restrict__ g, const uint32_t* __restrict__ u, uint64_t count,
                                   GatedEnd e) {
  for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < count; i += (uint64_t)gridDim.x * blockDim.x)
    gated_end(e, i, g[i], u[i]);
}

}  // namespace gkr
