// The rotation by position, as the kernels before the attention and in front of the paged cache apply it.
//
// Pair i of a head is turned by the angle position * inv_freq[i].  The angle is a product in 64 bits, taken in turns and
// reduced to half a turn either way there, far angles with the rests that 64 bits leave of the product and of 1 / (2 pi), and
// only then a 32-bit number: its error stays below 2^-24 of a turn for every position that 64 bits tell from the next (up to 2^53)
// and every angle up to 2^70 turns.  (In 32 bits a position of 10^6 is off by 0.06 rad; in 64 bits without the rests one of 2^40 by
// 2 * 10^-4, one of 2^52 by 0.8.)
//
// A row of D elements is the work of G lanes (8 up to 64 elements, 16 up to 128), 8 elements to a lane in two groups of
// four: lane u < rotary / 8 holds pairs 4u to 4u+3, the lanes behind hold the elements 8u to 8u+7 that are not turned.
// Pairs are (i, i + rotary / 2), or (2i, 2i + 1) where `interleaved`; a lane needs no element of another's either way,
// and the lanes of a row read whole cache lines.
#pragma once
#include "common.h"

namespace moba {

struct RowPlace {
  int a, b;     // first elements of the lane's two groups of four
  bool active;  // the row has elements for this lane
  bool turned;
};
__device__ __forceinline__ RowPlace row_place(int u, int D, int rotary, bool interleaved) {
  RowPlace p;
  p.active = 8 * u < D;
  p.turned = 8 * u < rotary;
  p.a = p.turned && !interleaved ? 4 * u : 8 * u;
  p.b = p.turned && !interleaved ? rotary / 2 + 4 * u : 8 * u + 4;
  return p;
}

// cos and sin of the angle of a pair at a position
__device__ __forceinline__ void turn_of(double position, float inv_freq, float& c, float& s) {
  constexpr double kOver2Pi = 0x1.45f306dc9c883p-3, kOver2PiRest = -0x1.6b01ec5417056p-57;
  const double f = inv_freq, angle = position * f, near = angle * kOver2Pi;
  double turns = near - rint(near);
  if (fabs(near) > 0x1p26) {   // (up to there the two roundings are off by 2^-26 of a turn; both rests everywhere: 1 % of an append)
    const double rest = fma(position, f, -angle);
    turns = fma(angle, kOver2Pi, -rint(near)) + fma(angle, kOver2PiRest, rest * kOver2Pi);
    turns -= rint(turns);
  }
  sincospif(2.f * (float)turns, &s, &c);
}

// The angles of a lane's four pairs.
struct Turn {
  float c[4], s[4];
  bool turned;  // (not turned: c and s mean nothing; a turn by 0 would spread an infinity or a NaN to the element beside it)
};
// x[0..3], x[4..7]: a lane's two groups.  kBack: by the angles' negatives, which is the transpose.
template <bool kBack = false>
__device__ __forceinline__ void turn_row(float (&x)[8], const Turn& t, bool interleaved) {
  if (!t.turned) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float s = kBack ? -t.s[i] : t.s[i];
    float& lo = interleaved ? x[2 * i] : x[i];
    float& hi = interleaved ? x[2 * i + 1] : x[i + 4];
    const float a = lo, b = hi;
    lo = a * t.c[i] - b * s;
    hi = b * t.c[i] + a * s;
  }
}

// A lane's two groups of a row, at addresses of 8-byte alignment.
template <class E>
__device__ __forceinline__ void load_row(const typename E::elem* row, const RowPlace& p, float (&x)[8]) {
  const typename E::elem4 a = *reinterpret_cast<const typename E::elem4*>(row + p.a);
  const typename E::elem4 b = *reinterpret_cast<const typename E::elem4*>(row + p.b);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[i] = (float)a[i];
    x[i + 4] = (float)b[i];
  }
}
template <class E>
__device__ __forceinline__ void store_row(typename E::elem* row, const RowPlace& p, const float (&x)[8]) {
  *reinterpret_cast<u32x2*>(row + p.a) = u32x2{pack2<E>(x[0], x[1]), pack2<E>(x[2], x[3])};
  *reinterpret_cast<u32x2*>(row + p.b) = u32x2{pack2<E>(x[4], x[5]), pack2<E>(x[6], x[7])};
}

// sum over the G lanes of a row, in every one of them (G = 8 or 16 neighbouring lanes)
template <int G>
__device__ __forceinline__ float row_sum(float x) {
  auto add = [](float v, int u) { return v + __builtin_bit_cast(float, u); };
  x = add(x, __builtin_amdgcn_update_dpp(0, (int)float_bits(x), 0xB1, 0xf, 0xf, false));   // lanes 1 0 3 2
  x = add(x, __builtin_amdgcn_update_dpp(0, (int)float_bits(x), 0x4E, 0xf, 0xf, false));   // lanes 2 3 0 1
  x = add(x, __builtin_amdgcn_update_dpp(0, (int)float_bits(x), 0x141, 0xf, 0xf, false));  // the other four of eight
  if constexpr (G == 16) x = add(x, __builtin_amdgcn_update_dpp(0, (int)float_bits(x), 0x140, 0xf, 0xf, false));  // the other eight
  return x;
}

}  // namespace moba
