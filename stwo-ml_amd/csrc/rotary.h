// Rotary positions: pairs of a head's values turned by position times frequency.
//
//   y0 = round((c(x0) C - c(x1) S) / 2^shift),  y1 = round((c(x1) C + c(x0) S) / 2^shift)
//
// with C = round(A cos t), S = round(A sin t), t = 2 pi (position f mod 2^64) / 2^64:
// frequencies are whole numbers of 2^-64 turns a position, so the angle of a far
// position is exact (as a float64 product it would have lost 17 bits at position
// 131071).  C and S lie in a table, eight bytes a pair and position, made once.
#pragma once
#include <stdint.h>

#include "field.h"
#include "gemm.h"

namespace gkr {

constexpr uint32_t kTurnSeqs = 256;      // sequences per launch
constexpr uint32_t kTurnRows = 1u << 22;  // rows per launch

// The table.  The quarter turn goes off in whole numbers, so that the rest, at
// most an eighth of a turn, keeps all of a float64's bits: C and S are the
// nearest whole numbers but for values within 2^-50 A of a half.
static __global__ void __launch_bounds__(256) k_turns(const uint64_t* __restrict__ freqs, uint32_t pairs, uint64_t count,
                                                      double amplitude, int2* __restrict__ table) {
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (uint64_t)gridDim.x * 256) {
    const uint64_t position = i / pairs, phase = position * freqs[i - position * pairs];
    const uint32_t quarter = (uint32_t)((phase >> 61) + 1) >> 1;
    const double rest = (double)(int64_t)(phase - ((uint64_t)quarter << 62)) * (6.283185307179586476925 / 18446744073709551616.0);
    double s, c;
    sincos(rest, &s, &c);
    if (quarter & 1) {
      const double t = c;
      c = -s;
      s = t;
    }
    auto whole = [&](double x) {
      const int32_t r = (int32_t)__builtin_floor(__builtin_fabs(x) * amplitude + 0.5);
      return (x < 0) != ((quarter & 2) != 0) ? -r : r;
    };
    table[i] = make_int2(whole(c), whole(s));
  }
}

struct TurnArgs {
  const int2* table;
  uint32_t head_dim, pairs;  // pairs that are turned; the dims behind them stay
  uint32_t shift;
  int32_t limit;             // 0: none, the result is taken mod P
  uint32_t n;                // sequences of this launch
  struct {
    const uint32_t* x;
    uint32_t* y;
    uint32_t heads;  // 0: no such matrix
  } m[2];
  struct {
    uint32_t row0, position;  // its first row in this launch, and that row's position
  } e[kTurnSeqs];
};
// t / 2^shift as a word of the field.
__device__ __forceinline__ uint32_t turn_word(int64_t t, uint32_t shift, int64_t half, int32_t limit) {
  const int64_t sign = t >> 63;
  uint64_t size = (uint64_t)(((t ^ sign) - sign) + half) >> shift;
  if (limit) size = size < (uint64_t)limit ? size : (uint64_t)limit;
  const uint32_t r = m31_reduce64(size);
  return sign ? m31_neg(r) : r;
}

// Grid: a row, and 256 units of it; a unit is four pairs (or up to eight dims
// that stay).  A thread's loads are whole 16 bytes, also where a head's size is
// no multiple of four: words may lie on any word's boundary.  A row's heads share
// its line of the table through the caches.
template <bool INTERLEAVED>
static __global__ void __launch_bounds__(256) k_turn(TurnArgs a, uint64_t row_base) {
  const uint32_t row = blockIdx.x;
  uint32_t i = 0;
  // The last sequence that begins at or before this row: a lane looks at four of them
  // (halving, a load behind the other, took 0.6 us more for 64).
  if (a.n > 1) {
#pragma unroll
    for (uint32_t j = 0; j < kTurnSeqs / 64; j++) {
      const uint32_t e = 64 * j + (threadIdx.x & 63);
      i += (uint32_t)__popcll(__ballot(e < a.n && a.e[e].row0 <= row));
    }
    i = __builtin_amdgcn_readfirstlane(i - 1);
  }
  const uint32_t position = a.e[i].position + (row - a.e[i].row0);
  const uint32_t rest = a.head_dim - 2 * a.pairs, turning = (a.pairs + 3) / 4, units = turning + (rest + 7) / 8;
  uint32_t u = blockIdx.y * 256 + threadIdx.x, which = 0;
  if (u >= a.m[0].heads * units) {
    u -= a.m[0].heads * units;
    which = 1;
    if (u >= a.m[1].heads * units) return;
  }
  const uint32_t head = u / units, unit = u - head * units;
  const uint64_t at = ((row_base + row) * a.m[which].heads + head) * a.head_dim;
  const uint32_t* const x = a.m[which].x + at;
  uint32_t* const y = a.m[which].y + at;
  if (unit >= turning) {  // dims that stay
    if (x == y) return;
    const uint32_t d0 = 2 * a.pairs + 8 * (unit - turning), d1 = d0 + 8 < a.head_dim ? d0 + 8 : a.head_dim;
    if (d1 - d0 == 8) {
      const v4i_word lo = *(const v4i_word*)(x + d0), hi = *(const v4i_word*)(x + d0 + 4);
      *(v4i_word*)(y + d0) = lo;
      *(v4i_word*)(y + d0 + 4) = hi;
    } else {
      for (uint32_t d = d0; d < d1; d++) y[d] = x[d];
    }
    return;
  }
  const int64_t half = a.shift ? 1ll << (a.shift - 1) : 0;
  const uint32_t p0 = 4 * unit;
  const int2* const cs = a.table + (uint64_t)position * a.pairs + p0;
  auto turn = [&](uint32_t x0, uint32_t x1, int2 t, uint32_t& y0, uint32_t& y1) {
    const int64_t v0 = center_m31(x0), v1 = center_m31(x1);
    y0 = turn_word(v0 * t.x - v1 * t.y, a.shift, half, a.limit);
    y1 = turn_word(v1 * t.x + v0 * t.y, a.shift, half, a.limit);
  };
  if (p0 + 4 <= a.pairs) {
    typedef int v4i_pair __attribute__((ext_vector_type(4), aligned(8)));
    const v4i_pair t0 = *(const v4i_pair*)cs, t1 = *(const v4i_pair*)(cs + 2);
    const int2 t[4] = {make_int2(t0[0], t0[1]), make_int2(t0[2], t0[3]), make_int2(t1[0], t1[1]), make_int2(t1[2], t1[3])};
    const uint32_t at0 = INTERLEAVED ? 2 * p0 : p0, at1 = INTERLEAVED ? at0 + 4 : p0 + a.pairs;
    const v4i_word w0 = *(const v4i_word*)(x + at0), w1 = *(const v4i_word*)(x + at1);
    v4i_word o0, o1;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      uint32_t y0, y1;
      if constexpr (INTERLEAVED) {
        const v4i_word& w = j < 2 ? w0 : w1;
        turn((uint32_t)w[2 * (j & 1)], (uint32_t)w[2 * (j & 1) + 1], t[j], y0, y1);
        v4i_word& o = j < 2 ? o0 : o1;
        o[2 * (j & 1)] = (int)y0;
        o[2 * (j & 1) + 1] = (int)y1;
      } else {
        turn((uint32_t)w0[j], (uint32_t)w1[j], t[j], y0, y1);
        o0[j] = (int)y0;
        o1[j] = (int)y1;
      }
    }
    *(v4i_word*)(y + at0) = o0;
    *(v4i_word*)(y + at1) = o1;
  } else {
    for (uint32_t p = p0; p < a.pairs; p++) {
      const uint32_t i0 = INTERLEAVED ? 2 * p : p, i1 = INTERLEAVED ? i0 + 1 : p + a.pairs;
      uint32_t y0, y1;
      turn(x[i0], x[i1], cs[p - p0], y0, y1);
      y[i0] = y0;
      y[i1] = y1;
    }
  }
}

}  // namespace gkr
