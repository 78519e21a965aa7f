// Products with weights in microscaled 4-bit floating point (the form is in
// mx4.h): y = W xn (+ residual) for up to three weights, and the input half of
// a SwiGLU block, xn = x or RMSNorm(x).  The reference's counterparts are
// Linear::forward, RMSNorm::forward and MLP::forward over fp32 weights.
#include "mx4_linear.h"

using namespace ember;

namespace {

// A workgroup takes 16 rows of x and 64 columns of y: thread (i, j) column j and
// rows 4 i .. 4 i + 3, the weights' values as they are read, a tile's 64 columns
// of x at a time through LDS.
constexpr int kThreads = 256;
constexpr int kRows = 16;
constexpr int kCols = 64;

template <bool GATE>
__global__ __launch_bounds__(kThreads) void mx4_linear_kernel(Mx4Call sg, Mx4Blocks bl) {
  __shared__ float xs[kRows][64];
  const int j = threadIdx.x % kCols, i = threadIdx.x / kCols;
  const float* x = sg.x;
  const float* norm_w = sg.norm_w;
  const int64_t M = sg.M, K = sg.K;
  int64_t blk = blockIdx.x;
  const int seg = GATE ? 0 : mx4_segment(bl, sg.nseg, blk);
  const int64_t N = sg.N[seg];
  const int64_t n = blk * kCols + j;
  const int64_t m0 = static_cast<int64_t>(blockIdx.y) * kRows;
  const int64_t kb = sg.kb, ks = sg.ks;
  const int64_t nb = n / 32, r = n % 32;
  float acc[2][4] = {}, ss[4] = {};
  for (int64_t t = 0; t < kb; ++t) {
    float part[2][4] = {};  // a tile's sums, so that the long one has K / 64 terms
    __syncthreads();
    for (int e = threadIdx.x; e < kRows * 64; e += kThreads) {
      const int64_t m = m0 + e / 64, k = t * 64 + e % 64;
      xs[e / 64][e % 64] = m < M && k < K ? x[m * K + k] : 0.f;
    }
    __syncthreads();
    for (int h = 0; h < 2; ++h) {
      for (int q = 0; q < 8; ++q) {
        f32x4 w[2] = {};
        for (int s = 0; s < (GATE ? 2 : 1); ++s) {
          if (n < N) {
            const Mx4Weight& W = sg.W[seg + s];
            const unsigned word = W.codes[(nb * kb + t) * 256 + (32 * h + r) * 4 + q / 2];
            const unsigned sc = W.scales[(nb * ks + t / 4) * 64 + 32 * h + r];
            w[s] = mx4_values(word >> (16 * (q % 2)), sc >> (8 * (t % 4)) & 255u);
          }
        }
        for (int e = 0; e < 4; ++e) {
          const int c = 32 * h + 4 * q + e;
          const int64_t k = t * 64 + c;
          if (k >= K) break;
          const float nw = norm_w ? norm_w[k] : 1.f;
          for (int m = 0; m < 4; ++m) {
            const float xv = xs[4 * i + m][c];
            ss[m] += xv * xv;
            for (int s = 0; s < (GATE ? 2 : 1); ++s) part[s][m] += w[s][e] * (xv * nw);
          }
        }
      }
    }
    for (int m = 0; m < 4; ++m)
      for (int s = 0; s < 2; ++s) acc[s][m] += part[s][m];
  }
  if (n >= N) return;
  for (int m = 0; m < 4; ++m) {
    const int64_t row = m0 + 4 * i + m;
    if (row >= M) break;
    const float sc = norm_w ? 1.0f / sqrtf(ss[m] / static_cast<float>(K) + sg.eps) : 1.0f;
    const float v = acc[0][m] * sc;
    float* y = sg.y[seg] + row * N + n;
    if (GATE) *y = mx4_silu_mul(v, acc[1][m] * sc);
    else *y = sg.res[seg] ? sg.res[seg][row * N + n] + v : v;
  }
}

// Rows of x and all the weights' rows a call takes: a launch's grid, and outputs
// whose offsets are counted in 64 bits.
bool rows_ok(int64_t M, int64_t K) { return M >= 0 && M <= 0x7fffffff && mx4_sizes_ok(0, K); }

template <bool GATE>
int launch(const Mx4Call& c, hipStream_t st) {
  Mx4Blocks bl{};
  for (int i = 0; i < c.nseg; ++i) bl.first[i + 1] = bl.first[i] + (c.N[i] + kCols - 1) / kCols;
  for (int64_t m = 0; m < c.M; m += int64_t(kRows) * 65535) {
    Mx4Call part = c;
    part.x += m * c.K;
    part.M = c.M - m < int64_t(kRows) * 65535 ? c.M - m : int64_t(kRows) * 65535;
    for (int i = 0; i < c.nseg; ++i) {
      part.y[i] += m * c.N[i];
      if (part.res[i]) part.res[i] += m * c.N[i];
    }
    const dim3 grid(static_cast<unsigned>(bl.first[GATE ? 1 : c.nseg]),
                    static_cast<unsigned>((part.M + kRows - 1) / kRows));
    mx4_linear_kernel<GATE><<<grid, kThreads, 0, st>>>(part, bl);
    const int rc = launch_status();
    if (rc != EMBER_OK) return rc;
  }
  return EMBER_OK;
}

// The parts of a call that do not depend on its kind.
Mx4Call call_of(const float* x, int64_t M, int64_t K, const float* norm_w, float eps) {
  Mx4Call c{};
  c.x = x;
  c.norm_w = norm_w;
  c.eps = eps;
  c.M = M;
  c.K = K;
  c.kb = mx4_col_tiles(K);
  c.ks = mx4_col_blocks(K);
  c.x_vec = K % 4 == 0 && aligned16(x) && (!norm_w || aligned16(norm_w));
  return c;
}

}  // namespace

extern "C" size_t ember_mx4_workspace_bytes(int64_t M, int64_t K, int64_t N) {
  (void)M, (void)K, (void)N;
  return 0;
}

extern "C" int ember_mx4_linear(const float* x, int64_t M, int64_t K, const float* norm_w,
                                float eps, int nseg, const void* const* codes,
                                const void* const* scales, const int64_t* N, float* const* y,
                                const float* const* residual, void* workspace,
                                size_t workspace_bytes, ember_stream_t s) {
  (void)workspace, (void)workspace_bytes;
  if (!rows_ok(M, K) || nseg < 1 || nseg > kMx4MaxSeg || !codes || !scales || !N || !y)
    return EMBER_EINVAL;
  Mx4Call c = call_of(x, M, K, norm_w, eps);
  c.nseg = nseg;
  for (int i = 0; i < nseg; ++i) {
    if (N[i] < 1 || !mx4_sizes_ok(N[i], K)) return EMBER_EINVAL;
    if (M == 0) continue;
    if (!codes[i] || !scales[i] || !y[i]) return EMBER_EINVAL;
    if (!aligned16(codes[i]) || !aligned16(scales[i])) return EMBER_EALIGN;
    c.W[i] = {static_cast<const uint32_t*>(codes[i]), static_cast<const uint32_t*>(scales[i])};
    c.y[i] = y[i];
    c.res[i] = residual ? residual[i] : nullptr;
    c.N[i] = N[i];
  }
  if (M == 0) return EMBER_OK;
  if (!x) return EMBER_EINVAL;
  if (M <= kMx4FewRows) return mx4_few_rows(c, false, as_stream(s));
  return launch<false>(c, as_stream(s));
}

extern "C" int ember_mx4_gateup(const float* x, int64_t M, int64_t K, const float* norm_w,
                                float eps, const void* gate_codes, const void* gate_scales,
                                const void* up_codes, const void* up_scales, int64_t I, float* out,
                                void* workspace, size_t workspace_bytes, ember_stream_t s) {
  (void)workspace, (void)workspace_bytes;
  if (!rows_ok(M, K) || I < 1 || !mx4_sizes_ok(I, K)) return EMBER_EINVAL;
  if (M == 0) return EMBER_OK;
  if (!x || !gate_codes || !gate_scales || !up_codes || !up_scales || !out) return EMBER_EINVAL;
  for (const void* p : {gate_codes, gate_scales, up_codes, up_scales})
    if (!aligned16(p)) return EMBER_EALIGN;
  Mx4Call c = call_of(x, M, K, norm_w, eps);
  c.nseg = 2;
  c.W[0] = {static_cast<const uint32_t*>(gate_codes), static_cast<const uint32_t*>(gate_scales)};
  c.W[1] = {static_cast<const uint32_t*>(up_codes), static_cast<const uint32_t*>(up_scales)};
  c.y[0] = out;
  c.N[0] = c.N[1] = I;
  if (M <= kMx4FewRows) return mx4_few_rows(c, true, as_stream(s));
  return launch<true>(c, as_stream(s));
}
