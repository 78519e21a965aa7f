// Weights held in microscaled 4-bit floating point: the form in memory and the
// device helpers that mx4.hip (store, lookup) and mx4_linear.hip (products)
// share.
//
// A weight [N, K] is cut along its rows into groups of 32 values.  A group
// keeps one byte b, its scale 2^(b - 127) (255: NaN), and per value a 4-bit
// code: a sign above one of the sizes 0, 1/2, 1, 3/2, 2, 3, 4, 6.  The scale is
// the smallest power of two that 7 times reaches the group's largest size:
// every value is then within half a step of a code, 6 to 7 included (the step
// below 6 is 2), where a scale of 6 would cost a bit of the next octave.
//
// The form is the matrix cores' own operand: a tile of 32 rows by 64 columns is
// 1 KB, lane 32 * h + r of a v_mfma_scale_f32_32x32x64_f8f6f4 holding the 16
// bytes of columns 32 h .. 32 h + 31 of row r; a row of tiles lies in order of
// the columns.  Scales come in blocks of 32 rows by 256 columns: lane 32 * h +
// r holds four bytes, one for each of the four tiles, which is the register
// (and the byte selects) that these four MFMAs take.  So a wave loads a tile
// in one 1 KB access and feeds it without a shuffle or a conversion.
#pragma once

#include "common.h"

namespace ember {

constexpr int kMx4TileBytes = 1024;
constexpr int kMx4ScaleBytes = 256;  // per 32 rows by 256 columns

// Tiles along N, tiles along K, scale blocks along K.
inline int64_t mx4_row_tiles(int64_t N) { return (N + 31) / 32; }
inline int64_t mx4_col_tiles(int64_t K) { return (K + 63) / 64; }
inline int64_t mx4_col_blocks(int64_t K) { return (K + 255) / 256; }

// Sizes the entries take: columns that an int holds with room to round up, and
// a weight whose values can be counted in 62 bits.
inline bool mx4_sizes_ok(int64_t N, int64_t K) {
  return N >= 0 && K >= 1 && N <= 0x7fffffff && K <= (int64_t(1) << 30);
}

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// The scale's byte of a group whose largest size has these bits: its exponent
// less 2, or less 1 where its mantissa is above 1.75; at least 0 (2^-127).
__device__ __forceinline__ unsigned mx4_scale_byte(unsigned top) {
  if (top >= 0x7f800000u) return 255u;  // an infinity or a NaN: the group reads back as NaN
  const int e = static_cast<int>((top + 0x1fffffu) >> 23) - 2;
  return static_cast<unsigned>(e > 0 ? e : 0);
}

// The code of x in a group of this scale byte.  Below 2 the codes' sizes lie 1/2
// apart, below 4 they lie 1 apart, above 2; rint takes ties to the even code, as
// each octave begins at one.
__device__ __forceinline__ unsigned mx4_code(float x, int byte) {
  const float q = __builtin_ldexpf(fabsf(x), 127 - byte);
  const float r = q < 2.f   ? __builtin_rintf(q + q)
                  : q < 4.f ? __builtin_rintf(q) + 2.f
                            : __builtin_rintf(0.5f * q) + 4.f;
  return static_cast<unsigned>(fminf(r, 7.f)) | (__float_as_uint(x) >> 28 & 8u);
}

// The four values of a group's codes in the low 16 bits of `codes`.
__device__ __forceinline__ f32x4 mx4_values(unsigned codes, int byte) {
  const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.f, 0);
  const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.f, 1);
  const float nan = __uint_as_float(0x7fc00000u);
  const int e = byte - 127;
  return byte == 255 ? f32x4{nan, nan, nan, nan}
                     : f32x4{__builtin_ldexpf(a.x, e), __builtin_ldexpf(a.y, e),
                             __builtin_ldexpf(b.x, e), __builtin_ldexpf(b.y, e)};
}

}  // namespace ember
