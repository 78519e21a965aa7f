// The one rule by which groups of fp32 values are held in few bits (kv4.hip,
// q8.hip).  A group keeps lo, its smallest value, and
//   step = (largest - smallest) / TOP, rounded to fp32   (TOP = 15 or 255),
// and per value the whole code nearest (x - lo) / step, which reads back as
// fma(code, step, lo).  The error is at most step / 2 and the roundings of
// step and of the read-back.  A group of equal values has step 0 and reads
// back exactly; a group with an infinity or a NaN reads back as NaN throughout
// (lo = step = NaN, codes 0).
//
// The quotient is formed in fp64: in fp32 the rounding of x - lo and of 1 / step
// (together up to 3 * 2^-24 of it) puts about one value in a million on the other
// side of a border between two codes, and a value off by a whole step then
// looks like an error of the store.  The fp64 work runs under the memory
// traffic: see q8_quantize_kernel's figures.
#pragma once

#include "common.h"

namespace ember {

struct QuantGrid {
  float lo, step;
  double inv;  // 1 / step; 0 where step is 0 or NaN
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
    g.lo = g.step = __uint_as_float(0x7fc00000u);
    g.inv = 0.0;
    return g;
  }
  g.lo = lo;
  g.step = static_cast<float>((static_cast<double>(hi) - static_cast<double>(lo)) /
                              static_cast<double>(TOP));
  g.inv = g.step > 0.f ? 1.0 / static_cast<double>(g.step) : 0.0;
  return g;
}

// The code of x (finite, unless the group is NaN throughout).
template <int TOP>
__device__ __forceinline__ unsigned quant_code(const QuantGrid& g, float x) {
  const double t =
      __builtin_rint((static_cast<double>(x) - static_cast<double>(g.lo)) * g.inv);
  // Above TOP only where a subnormal step was rounded down by much.
  return g.inv == 0.0 ? 0u : static_cast<unsigned>(t > TOP ? static_cast<double>(TOP) : t);
}

}  // namespace ember
