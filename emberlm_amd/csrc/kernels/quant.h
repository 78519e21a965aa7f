// The one rule by which groups of fp32 values are held in few bits (kv4.hip,
// q8.hip).  A group keeps lo, its smallest value, and
//   step = (largest - smallest) / TOP, rounded to fp32   (TOP = 15 or 255),
// and per value the whole code nearest (x - lo) / step, which reads back as
// fma(code, step, lo).  The error is at most step / 2 and the roundings of
// step and of the read-back.  A group of equal values has step 0 and reads
// back exactly; a group with an infinity or a NaN reads back as NaN throughout
// (lo = step = NaN, codes 0).
//
// The quotient is the one that fp64 gives: rounded to fp32 along the way it puts
// about one value in a million on the other side of a border between two
// codes, and a value off by a whole step then looks like an error of the store.  A
// wave forms it in fp32 first, whose error is below kNear, and again in fp64
// only where some value of its lies that near a border (2 kNear of a wave's 512
// values: a wave in 8 of 255 steps, in 140 of 15): all in fp64, with two fp64 divisions a group,
// quantising 32768 x 2048 values took 90 us, so 67 (5.1 TB/s).
#pragma once

#include "common.h"

namespace ember {

struct QuantGrid {
  float lo, step;
  float inv;  // near 1 / step; 0 where step is 0, NaN where only fp64 will do
};

// x is Inf or NaN.
__device__ __forceinline__ bool not_finite(float x) {
  return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u;
}

// The grid of a group spread over LPG lanes (aligned blocks of LPG lanes, a
// power of two; every lane of the wave takes part): lo, hi and bad are this
// lane's bounds and whether it holds a value that is not finite.
template <int LPG, int TOP>
__device__ __forceinline__ QuantGrid quant_grid(float lo, float hi, bool bad) {
#pragma unroll
  for (int o = LPG / 2; o > 0; o >>= 1) {
    lo = fminf(lo, __shfl_xor(lo, o, kWave));
    hi = fmaxf(hi, __shfl_xor(hi, o, kWave));
  }
  const int lane = threadIdx.x & (kWave - 1);
  constexpr unsigned long long kMask = LPG == 64 ? ~0ull : (1ull << (LPG & 63)) - 1;
  QuantGrid g;
  if ((__ballot(bad) >> (lane & ~(LPG - 1))) & kMask) {
    g.lo = g.step = g.inv = __uint_as_float(0x7fc00000u);
    return g;
  }
  g.lo = lo;
  // d / TOP, the product with 1 / TOP corrected by its remainder
  const double d = static_cast<double>(hi) - static_cast<double>(lo);
  const double q = d * (1.0 / TOP);
  g.step = static_cast<float>(fma(fma(-q, static_cast<double>(TOP), d), 1.0 / TOP, q));
  // Outside of these steps the fp32 quotient leaves its range or its error bound.
  g.inv = g.step >= 0x1p-126f && g.step <= 0x1p125f ? __builtin_amdgcn_rcpf(g.step)
          : g.step == 0.f                           ? 0.f
                                                    : __uint_as_float(0x7fc00000u);
  return g;
}

// The codes of a lane's eight values (whole waves call this; values of lanes
// that hold none are any finite ones).
template <int TOP>
__device__ __forceinline__ void quant_codes(const QuantGrid& g, const float (&x)[8],
                                            unsigned (&code)[8]) {
  // x - lo rounds by 2^-24 of it, rcp by 2^-23, the product by 2^-24; twice that
  constexpr float kNear = TOP * 0x1p-21f;
  bool near = false;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float t = (x[e] - g.lo) * g.inv, r = __builtin_rintf(t);
    near |= !(fabsf(t - r) < 0.5f - kNear);  // and where t is NaN
    code[e] = static_cast<unsigned>(r);
  }
  if (!__any(near)) return;
  const bool none = !(g.step > 0.f);  // 0 or NaN: every code is 0
  const double inv = 1.0 / static_cast<double>(g.step);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const double t =
        __builtin_rint((static_cast<double>(x[e]) - static_cast<double>(g.lo)) * inv);
    // Above TOP only where a subnormal step was rounded down by much.
    code[e] = none ? 0u : static_cast<unsigned>(t > TOP ? static_cast<double>(TOP) : t);
  }
}

}  // namespace ember
