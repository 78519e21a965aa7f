// Rows of fp32 held in 8 bits: the saved inputs of checkpointed blocks.
//
// Groups of 128 values along a row (the last may be shorter), by the rule of
// quant.h with 255 steps.  codes [rows][round_up(H, 16)] bytes (the padding is
// written as 0), params [rows][ceil(H / 128)][2] = {lo, step}.  The reference
// keeps every block's fp32 input (CheckpointNode, src/core/autograd.cu:327-363)
// and has no counterpart to these.
#include <cmath>

#include "common.h"
#include "quant.h"

using namespace ember;

namespace {

constexpr int kThreads = 256;
constexpr int kGroup = 128;
constexpr int kLpg = kGroup / 8;  // lanes per group, 8 values each

inline int64_t row_groups(int64_t H) { return (H + kGroup - 1) / kGroup; }
__host__ __device__ inline int64_t row_bytes(int64_t H) { return (H + 15) / 16 * 16; }

// Eight values of a row from column c0 (those at or past H are not read).
template <bool VEC>
__device__ __forceinline__ void load8(const float* __restrict__ row, int64_t c0, int64_t H,
                                      float (&x)[8]) {
  if (VEC && c0 + 8 <= H) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(row + c0);
    const f32x4 b = *reinterpret_cast<const f32x4*>(row + c0 + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = a[e];
      x[4 + e] = b[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = c0 + e < H ? row[c0 + e] : 0.f;
  }
}

// One group per 16 lanes, eight values a lane.
template <bool VEC>
__global__ __launch_bounds__(kThreads) void q8_quantize_kernel(const float* __restrict__ x,
                                                               uint8_t* __restrict__ codes,
                                                               float* __restrict__ params,
                                                               int64_t rows, int64_t H,
                                                               int64_t ngroups) {
  const int64_t total = rows * ngroups;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (kThreads / kLpg);
  const int64_t hp = row_bytes(H);
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * (kThreads / kLpg); base < total;
       base += step) {
    const int64_t gi = base + threadIdx.x / kLpg;
    const bool live = gi < total;
    const int64_t row = live ? gi / ngroups : 0, grp = live ? gi % ngroups : 0;
    const int64_t c0 = grp * kGroup + 8 * (threadIdx.x % kLpg);
    float v[8];
    load8<VEC>(x + row * H, c0, live ? H : 0, v);
    float lo = INFINITY, hi = -INFINITY;
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c0 + e < H) {
        lo = fminf(lo, v[e]);
        hi = fmaxf(hi, v[e]);
        bad |= not_finite(v[e]);
      }
    const QuantGrid g = quant_grid<kLpg, 255>(lo, hi, bad);
    if (!live) continue;
    uint2 w = {0u, 0u};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (c0 + e < H) w.x |= quant_code<255>(g, v[e]) << (8 * e);
      if (c0 + 4 + e < H) w.y |= quant_code<255>(g, v[4 + e]) << (8 * e);
    }
    if (c0 < hp) *reinterpret_cast<uint2*>(codes + row * hp + c0) = w;
    if (threadIdx.x % kLpg == 0)
      *reinterpret_cast<float2*>(params + 2 * gi) = float2{g.lo, g.step};
  }
}

// The eight values held from column c0 of a row.
__device__ __forceinline__ void held8(const uint8_t* __restrict__ codes,
                                      const float* __restrict__ params, int64_t row, int64_t c0,
                                      int64_t hp, int64_t ngroups, float (&x)[8]) {
  const uint2 w = *reinterpret_cast<const uint2*>(codes + row * hp + c0);
  const float2 p = *reinterpret_cast<const float2*>(params + 2 * (row * ngroups + c0 / kGroup));
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[e] = fmaf(static_cast<float>((w.x >> (8 * e)) & 255u), p.y, p.x);
    x[4 + e] = fmaf(static_cast<float>((w.y >> (8 * e)) & 255u), p.y, p.x);
  }
}

template <bool VEC>
__device__ __forceinline__ void store8(float* __restrict__ row, int64_t c0, int64_t H,
                                       const float (&x)[8]) {
  if (VEC && c0 + 8 <= H) {
    *reinterpret_cast<f32x4*>(row + c0) = f32x4{x[0], x[1], x[2], x[3]};
    *reinterpret_cast<f32x4*>(row + c0 + 4) = f32x4{x[4], x[5], x[6], x[7]};
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c0 + e < H) row[c0 + e] = x[e];
  }
}

template <bool VEC>
__global__ __launch_bounds__(kThreads) void q8_dequantize_kernel(
    const uint8_t* __restrict__ codes, const float* __restrict__ params, float* __restrict__ x,
    int64_t rows, int64_t H, int64_t ngroups) {
  const int64_t per = (H + 7) / 8, hp = row_bytes(H);
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kThreads;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < rows * per;
       i += stride) {
    const int64_t row = i / per, c0 = 8 * (i % per);
    float v[8];
    held8(codes, params, row, c0, hp, ngroups, v);
    store8<VEC>(x + row * H, c0, H, v);
  }
}

// The restored rows and their RMSNorm, a block per row.
template <bool VEC>
__global__ __launch_bounds__(kThreads) void q8_dequantize_rmsnorm_kernel(
    const uint8_t* __restrict__ codes, const float* __restrict__ params,
    const float* __restrict__ w, float* __restrict__ x, float* __restrict__ y,
    float* __restrict__ rstd, int64_t H, int64_t ngroups, float eps) {
  __shared__ float red[kThreads / kWave];
  const int64_t row = blockIdx.x, hp = row_bytes(H);
  float ss = 0.f;
  for (int64_t c0 = 8 * threadIdx.x; c0 < H; c0 += 8 * kThreads) {
    float v[8];
    held8(codes, params, row, c0, hp, ngroups, v);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c0 + e < H) ss = fmaf(v[e], v[e], ss);
    store8<VEC>(x + row * H, c0, H, v);
  }
  ss = block_sum(ss, red);
  const float s = 1.0f / sqrtf(ss / static_cast<float>(H) + eps);
  if (rstd && threadIdx.x == 0) rstd[row] = s;
  for (int64_t c0 = 8 * threadIdx.x; c0 < H; c0 += 8 * kThreads) {
    float v[8], wv[8];
    held8(codes, params, row, c0, hp, ngroups, v);
    load8<VEC>(w, c0, H, wv);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = v[e] * s * wv[e];
    store8<VEC>(y + row * H, c0, H, v);
  }
}

bool aligned8(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7u) == 0; }

}  // namespace

extern "C" size_t ember_q8_code_bytes(int64_t rows, int64_t H) {
  return rows > 0 && H > 0 ? static_cast<size_t>(rows * row_bytes(H)) : 0;
}

extern "C" size_t ember_q8_param_bytes(int64_t rows, int64_t H) {
  return rows > 0 && H > 0 ? static_cast<size_t>(rows * row_groups(H)) * 2 * sizeof(float) : 0;
}

extern "C" int ember_q8_quantize(const float* x, void* codes, float* params, int64_t rows,
                                 int64_t H, ember_stream_t s) {
  if (rows < 0 || H < 0) return EMBER_EINVAL;
  if (rows == 0 || H == 0) return EMBER_OK;
  if (!x || !codes || !params) return EMBER_EINVAL;
  if (!aligned16(codes) || !aligned8(params)) return EMBER_EALIGN;
  auto* c = static_cast<uint8_t*>(codes);
  const int64_t ng = row_groups(H);
  const unsigned grid = grid_1d(rows * ng, kThreads / kLpg);
  if (H % 4 == 0 && aligned16(x))
    q8_quantize_kernel<true><<<grid, kThreads, 0, as_stream(s)>>>(x, c, params, rows, H, ng);
  else
    q8_quantize_kernel<false><<<grid, kThreads, 0, as_stream(s)>>>(x, c, params, rows, H, ng);
  return launch_status();
}

extern "C" int ember_q8_dequantize(const void* codes, const float* params, float* x, int64_t rows,
                                   int64_t H, ember_stream_t s) {
  if (rows < 0 || H < 0) return EMBER_EINVAL;
  if (rows == 0 || H == 0) return EMBER_OK;
  if (!x || !codes || !params) return EMBER_EINVAL;
  if (!aligned16(codes) || !aligned8(params)) return EMBER_EALIGN;
  const auto* c = static_cast<const uint8_t*>(codes);
  const int64_t ng = row_groups(H);
  const unsigned grid = grid_1d(rows * ((H + 7) / 8), kThreads);
  if (H % 4 == 0 && aligned16(x))
    q8_dequantize_kernel<true><<<grid, kThreads, 0, as_stream(s)>>>(c, params, x, rows, H, ng);
  else
    q8_dequantize_kernel<false><<<grid, kThreads, 0, as_stream(s)>>>(c, params, x, rows, H, ng);
  return launch_status();
}

extern "C" int ember_q8_dequantize_rmsnorm(const void* codes, const float* params, const float* w,
                                           float* x, float* y, float* rstd, int64_t rows,
                                           int64_t H, float eps, ember_stream_t s) {
  if (rows < 0 || H < 0 || rows > 0x7fffffff) return EMBER_EINVAL;
  if (rows == 0 || H == 0) return EMBER_OK;
  if (!x || !y || !w || !codes || !params) return EMBER_EINVAL;
  if (!aligned16(codes) || !aligned8(params)) return EMBER_EALIGN;
  const auto* c = static_cast<const uint8_t*>(codes);
  const int64_t ng = row_groups(H);
  const unsigned grid = static_cast<unsigned>(rows);
  if (H % 4 == 0 && aligned16(x) && aligned16(y) && aligned16(w))
    q8_dequantize_rmsnorm_kernel<true>
        <<<grid, kThreads, 0, as_stream(s)>>>(c, params, w, x, y, rstd, H, ng, eps);
  else
    q8_dequantize_rmsnorm_kernel<false>
        <<<grid, kThreads, 0, as_stream(s)>>>(c, params, w, x, y, rstd, H, ng, eps);
  return launch_status();
}
