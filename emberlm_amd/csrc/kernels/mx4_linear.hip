// Products with weights in microscaled 4-bit floating point (the form is in
// mx4.h): y = W xn (+ residual) for up to three weights, and the input half of
// a SwiGLU block, xn = x or RMSNorm(x).  The reference's counterparts are
// Linear::forward, RMSNorm::forward and MLP::forward over fp32 weights.
#include "mx4_linear.h"

using namespace ember;

namespace {

// Rows of x that a call takes: counted in 31 bits.
bool rows_ok(int64_t M, int64_t K) { return M >= 0 && M <= 0x7fffffff && mx4_sizes_ok(0, K); }

// Columns of a SwiGLU input half: of few rows, 32 a workgroup of 512 threads.
constexpr int64_t kMostInner = int64_t(1) << 27;

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

int run(const Mx4Call& c, bool gate, void* workspace, size_t workspace_bytes, hipStream_t st) {
  if (mx4_few(c.M, c.K)) return mx4_few_rows(c, gate, st);
  if (!workspace || workspace_bytes < mx4_many_rows_bytes(c.M, c.K)) return EMBER_EWORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) & 255u) return EMBER_EALIGN;
  return mx4_many_rows(c, gate, workspace, st);
}

}  // namespace

extern "C" size_t ember_mx4_workspace_bytes(int64_t M, int64_t K, int64_t N) {
  if (!rows_ok(M, K) || N < 0 || mx4_few(M, K)) return 0;
  return mx4_many_rows_bytes(M, K);
}

extern "C" int ember_mx4_linear(const float* x, int64_t M, int64_t K, const float* norm_w,
                                float eps, int nseg, const void* const* codes,
                                const void* const* scales, const int64_t* N, float* const* y,
                                const float* const* residual, void* workspace,
                                size_t workspace_bytes, ember_stream_t s) {
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
  return run(c, false, workspace, workspace_bytes, as_stream(s));
}

extern "C" int ember_mx4_gateup(const float* x, int64_t M, int64_t K, const float* norm_w,
                                float eps, const void* gate_codes, const void* gate_scales,
                                const void* up_codes, const void* up_scales, int64_t I, float* out,
                                void* workspace, size_t workspace_bytes, ember_stream_t s) {
  if (!rows_ok(M, K) || I < 1 || I > kMostInner || !mx4_sizes_ok(I, K)) return EMBER_EINVAL;
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
  return run(c, true, workspace, workspace_bytes, as_stream(s));
}
