// Rotary positions: the angle of a pair at a position, its cosine and sine, and the
// turned values, for the kernels that turn rows in place of a table of every angle.
//
// Pair i of a row at position t is turned by t f_i.  The caller hands over each frequency
// as a whole number of 2^-64 turns, F_i = 2^64 (f_i / 2 pi mod 1): t F_i mod 2^64 is then
// the exact fraction of a turn at every 32-bit position, negative ones too, where t f_i in
// fp32 would be off by whole radians far out (2^-24 of 100000 radians).  The fraction is
// split into the nearest quarter turn and a rest of at most 1/8 turn, whose sine and
// cosine are their Taylor polynomials to x^9 and x^8 (off by x^11/11! < 2e-9 and
// x^10/10! < 2.5e-8, below fp32's half step next to 1).
#pragma once
#include "common.hpp"
#include "kernels.hpp"

namespace tia {

__device__ __forceinline__ void turn_of(uint64_t f, int64_t t, float amplitude, float& cosine, float& sine) {
  const uint64_t at = uint64_t(t) * f;
  const uint32_t hi = uint32_t(at >> 32), quarter = (hi + 0x20000000u) >> 30;
  const int32_t rest = int32_t(hi - (quarter << 30));
  // (The low word counts where the rest is small: a slow pair near position 0.)
  const float x = fmaf(float(uint32_t(at)), 0x1p-32f, float(rest)) * 1.4629180792671596e-9f;  // 2 pi / 2^32
  const float y = x * x;
  const float s = fmaf(x * y, fmaf(y, fmaf(y, fmaf(y, 1.f / 362880, -1.f / 5040), 1.f / 120), -1.f / 6), x);
  const float c = fmaf(y, fmaf(y, fmaf(y, fmaf(y, 1.f / 40320, -1.f / 720), 1.f / 24), -0.5f), 1.f);
  const float a = quarter & 1 ? s : c, b = quarter & 1 ? c : s;
  cosine = amplitude * ((quarter + 1) & 2 ? -a : a);
  sine = amplitude * (quarter & 2 ? -b : b);
}

// A lane's share of a row: 16 values, two pieces of 8, as 8 pairs.  Half layout: pieces
// 8 u and R / 2 + 8 u; interleaved: 16 u and 16 u + 8.  From R on: the plain 16 u, 16 u + 8.
struct RowUnit {
  int first, second;  // where the pieces start
  bool turned;
};
__device__ __forceinline__ RowUnit row_unit(const RotaryArgs& r, int u) {
  const bool turned = 16 * u < r.rotated;
  if (turned && !r.interleaved) return {8 * u, (r.rotated >> 1) + 8 * u, true};
  return {16 * u, 16 * u + 8, turned};
}

struct Turns {
  float c[8], s[8];
  // Those of pairs 8 u .. 8 u + 7.
  __device__ __forceinline__ Turns(const RotaryArgs& r, int u, int64_t t) {
#pragma unroll
    for (int e = 0; e < 8; ++e) turn_of(r.turns[8 * u + e], t, r.amplitude, c[e], s[e]);
  }
};

__device__ __forceinline__ half8_t load_half8(const uint16_t* p) {  // (any even address)
  half8_t x;
  __builtin_memcpy(&x, p, 16);
  return x;
}
__device__ __forceinline__ void store_half8(uint16_t* p, half8_t x) { __builtin_memcpy(p, &x, 16); }

// A pair's two values, rounded to fp16 once.  (Which product is fused with the sum is written
// down, so every kernel gives the same bits.)
__device__ __forceinline__ void turn_pair(float c, float s, f16& a, f16& b) {
  const float x = float(a), y = float(b);
  a = f16r(fmaf(x, c, -(y * s)));
  b = f16r(fmaf(x, s, y * c));
}
__device__ __forceinline__ void turn_unit(const Turns& t, bool interleaved, half8_t& first, half8_t& second) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (interleaved) {
      half8_t& x = e < 4 ? first : second;
      f16 a = x[2 * e & 7], b = x[(2 * e & 7) + 1];
      turn_pair(t.c[e], t.s[e], a, b);
      x[2 * e & 7] = a;
      x[(2 * e & 7) + 1] = b;
    } else {
      f16 a = first[e], b = second[e];
      turn_pair(t.c[e], t.s[e], a, b);
      first[e] = a;
      second[e] = b;
    }
  }
}

// A lane's unit of heads [h0, h1) of a row from x to y (each given at head 0, y at the
// first piece, its second one y_second behind), HC heads at a time: their loads are on the
// way while the angles, or the heads in front of them, are worked on.
template <int HC>
__device__ __forceinline__ void turn_heads(const RotaryArgs& r, RowUnit unit, int u, int64_t t, const uint16_t* x, int64_t x_step,
                                           uint16_t* y, int64_t y_step, int y_second, int h0, int h1) {
  half8_t p[HC], q[HC];
  const auto load = [&](int h) {
#pragma unroll
    for (int i = 0; i < HC; ++i) {
      const uint16_t* at = x + int64_t(min(h + i, h1 - 1)) * x_step;
      p[i] = load_half8(at + unit.first);
      q[i] = load_half8(at + unit.second);
    }
  };
  const auto store = [&](int h) {
#pragma unroll
    for (int i = 0; i < HC; ++i) {
      if (h + i >= h1) break;
      store_half8(y + int64_t(h + i) * y_step, p[i]);
      store_half8(y + int64_t(h + i) * y_step + y_second, q[i]);
    }
  };
  load(h0);
  if (!unit.turned) {
    for (int h = h0;;) {
      store(h);
      if ((h += HC) >= h1) return;
      load(h);
    }
  }
  const Turns turns(r, u, t);
  for (int h = h0;;) {
#pragma unroll
    for (int i = 0; i < HC; ++i) turn_unit(turns, r.interleaved, p[i], q[i]);
    store(h);
    if ((h += HC) >= h1) return;
    load(h);
  }
}

}  // namespace tia
