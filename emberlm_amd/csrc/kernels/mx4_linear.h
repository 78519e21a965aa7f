// What the entry points of the products with 4-bit weights (mx4_linear.hip)
// share with their kernels.
#pragma once

#include <cmath>

#include "mx4.h"

namespace ember {

constexpr int kMx4MaxSeg = 3;  // weights of one ember_mx4_linear call

struct Mx4Weight {
  const uint32_t* codes;
  const uint32_t* scales;
};

// One call's products.  SwiGLU (gate): weights 0 and 1 are the gate's and the
// up projection's, both of N[0] rows, y[0] the output.
struct Mx4Call {
  const float* x;
  const float* norm_w;  // NULL: x as it is
  float eps;
  int64_t M, K;
  int64_t kb, ks;  // tiles and scale blocks along K
  Mx4Weight W[kMx4MaxSeg];
  const float* res[kMx4MaxSeg];
  float* y[kMx4MaxSeg];
  int64_t N[kMx4MaxSeg];
  int nseg;
  bool x_vec;  // rows of x and the norm's weight are whole aligned float4s
};

// The segment and its block of a workgroup that takes block b of all segments'
// column blocks (first[i]: the first of segment i).
struct Mx4Blocks {
  int64_t first[kMx4MaxSeg + 1];
};
__device__ __forceinline__ int mx4_segment(const Mx4Blocks& bl, int nseg, int64_t& b) {
  int seg = 0;
  while (seg + 1 < nseg && b >= bl.first[seg + 1]) ++seg;
  b -= bl.first[seg];
  return seg;
}

// A launch holds fewer than 2^32 threads.
inline bool mx4_launch_ok(int64_t blocks, int threads) {
  return blocks <= 0xffffffffll / threads;
}

// silu(g) u.  With q = e^-|g| the sigmoid is 1 / (1 + q), or q / (1 + q) left of 0: nothing
// overflows, and a reciprocal of 1 to 2 and an exponential whose argument keeps its
// second word (log2 e in two) are each off by two half steps.  e^g below 2^-126 counts as
// 0.  (14 instructions for the 36 of expf and a division: 2048 rows to 2 x 6144 columns 149.7
// -> 145.4 us.)
__device__ __forceinline__ float mx4_silu_mul(float g, float u) {
  constexpr float kLog2eHi = 1.44269502f, kLog2eLo = 1.92596303e-8f, kLn2 = 0.693147181f;
  const float a = fminf(fabsf(g), 200.f);
  const float t = -kLog2eHi * a;
  const float rest = __builtin_fmaf(-kLog2eHi, a, -t) - kLog2eLo * a;
  const float q = __builtin_amdgcn_exp2f(t) * __builtin_fmaf(rest, kLn2, 1.f);
  const float top = g < 0.f ? g * q : g;
  return top * __builtin_amdgcn_rcpf(1.f + q) * u;
}

// Calls of few rows (mx4_few.hip).  Each of its workgroups cuts all of x into digits
// for itself, which for an x of many values takes longer than a launch that does it
// once.  With N = 2048, there and in mx4_many.hip: 8 rows of K = 8192 22.5 us and 11.4,
// 8 of 4096 11.4 and 10.7, 4 of 6144 9.7 and 11, 8 of 2048 7.6 and 8.5.
constexpr int kMx4FewRows = 8;
inline bool mx4_few(int64_t M, int64_t K) {
  return M <= 3 || (M <= kMx4FewRows && M * K <= 30000);
}
int mx4_few_rows(const Mx4Call& c, bool gate, hipStream_t st);
// Calls of more (mx4_many.hip), and the workspace they take.
size_t mx4_many_rows_bytes(int64_t M, int64_t K);
int mx4_many_rows(const Mx4Call& c, bool gate, void* workspace, hipStream_t st);

}  // namespace ember
