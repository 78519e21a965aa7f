// Rows of fp32 held in 8 bits: the saved inputs of checkpointed blocks.
//
// Groups of 128 values along a row (the last may be shorter), by the rule of
// quant.h with 255 steps.  codes [rows][round_up(H, 16)] bytes (the padding is
// written as 0), params [rows][ceil(H / 128)][2] = {lo, step}.  The reference
// keeps every block's fp32 input (CheckpointNode, src/core/autograd.cu:327-363)
// and has no counterpart to these.
//
// All three kernels are bound by HBM: quantising moves 4 + 1 1/16 bytes a
// value, restoring 1 1/16 + 4, restoring with the norm 1 1/16 + 8 (a restore and
// ember_rmsnorm_fwd after it, 13 1/16).  fp32 rows may start at any float: their
// 16-byte accesses need 4-byte alignment only, so a width of 1001 runs at the
// rate of 1000.
#include <cmath>

#include "common.h"
#include "quant.h"

using namespace ember;

namespace {

constexpr int kThreads = 256;
constexpr int kGroup = 128;
constexpr int kLpg = kGroup / 8;  // lanes per group when quantising, 8 values each

inline int64_t row_groups(int64_t H) { return (H + kGroup - 1) / kGroup; }
__host__ __device__ inline int64_t row_bytes(int64_t H) { return (H + 15) / 16 * 16; }

// Four floats at any float's address.
typedef f32x4 f32x4_any __attribute__((aligned(4)));

// Columns c .. c + 3 of a row of H (those past it read as 0, and are not stored).
// ONCE: rows that are read once (non-temporal).
template <bool ONCE>
__device__ __forceinline__ f32x4 load4(const float* __restrict__ row, int64_t c, int64_t H) {
  const f32x4_any* p = reinterpret_cast<const f32x4_any*>(row + c);
  if (c + 4 <= H) return ONCE ? __builtin_nontemporal_load(p) : *p;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int e = 0; e < 3; ++e)
    if (c + e < H) v[e] = row[c + e];
  return v;
}
__device__ __forceinline__ void store4(float* __restrict__ row, int64_t c, int64_t H, f32x4 v) {
  if (c + 4 <= H) {
    *reinterpret_cast<f32x4_any*>(row + c) = v;
  } else {
#pragma unroll
    for (int e = 0; e < 3; ++e)
      if (c + e < H) row[c + e] = v[e];
  }
}

// One group per 16 lanes: lane l holds columns 4 l .. and 64 + 4 l .., so that
// the lanes' loads lie side by side.  Rows and groups advance by the grid's
// stride without a division.
__global__ __launch_bounds__(kThreads) void q8_quantize_kernel(const float* __restrict__ x,
                                                               uint8_t* __restrict__ codes,
                                                               float* __restrict__ params,
                                                               int64_t rows, int64_t H,
                                                               int64_t ngroups) {
  const int64_t hp = row_bytes(H);
  const int64_t step = static_cast<int64_t>(gridDim.x) * (kThreads / kLpg);
  const int64_t step_rows = step / ngroups, step_groups = step % ngroups;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (kThreads / kLpg) + threadIdx.x / kLpg;
  int64_t row = first / ngroups, grp = first % ngroups;
  // the wave's first group decides when the whole wave is done
  int64_t wave_first = first - (threadIdx.x & (kWave - 1)) / kLpg;
  for (; wave_first < rows * ngroups; wave_first += step) {
    const bool live = row < rows;
    const int64_t c = grp * kGroup + 4 * (threadIdx.x % kLpg);
    const float* src = x + (live ? row : 0) * H;
    const int64_t end = live ? H : 0;
    float v[8];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const f32x4 t = load4<true>(src, c + 64 * u, end);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 * u + e] = t[e];
    }
    float lo = INFINITY, hi = -INFINITY;
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + 64 * (e / 4) + e % 4 < end) {
        lo = fminf(lo, v[e]);
        hi = fmaxf(hi, v[e]);
        bad |= not_finite(v[e]);
      }
    const QuantGrid g = quant_grid<kLpg, 255>(lo, hi, bad);
    unsigned code[8];
    quant_codes<255>(g, v, code);
    if (live) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int64_t cu = c + 64 * u;
        unsigned w = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) w |= (cu + e < H ? code[4 * u + e] : 0u) << (8 * e);
        if (cu < hp) __builtin_nontemporal_store(w, reinterpret_cast<unsigned*>(codes + row * hp + cu));
      }
      if (threadIdx.x % kLpg == 0)
        *reinterpret_cast<float2*>(params + 2 * (row * ngroups + grp)) = float2{g.lo, g.step};
    }
    row += step_rows;
    grp += step_groups;
    if (grp >= ngroups) {
      grp -= ngroups;
      ++row;
    }
  }
}

// The four values held from column c (a multiple of 4, below the padded width).
__device__ __forceinline__ f32x4 held4(const uint8_t* __restrict__ codes,
                                       const float* __restrict__ params, int64_t c) {
  const unsigned w = __builtin_nontemporal_load(reinterpret_cast<const unsigned*>(codes + c));
  const float2 p = *reinterpret_cast<const float2*>(params + 2 * (c / kGroup));
  f32x4 x;
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = fmaf(static_cast<float>((w >> (8 * e)) & 255u), p.y, p.x);
  return x;
}

// LPR lanes per row, four columns a lane at a time.
template <int LPR>
__global__ __launch_bounds__(kThreads) void q8_dequantize_kernel(
    const uint8_t* __restrict__ codes, const float* __restrict__ params, float* __restrict__ x,
    int64_t rows, int64_t H, int64_t ngroups) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / LPR) + threadIdx.x / LPR;
  if (row >= rows) return;
  const uint8_t* rc = codes + row * row_bytes(H);
  const float* rp = params + 2 * row * ngroups;
#pragma unroll 4
  for (int64_t c = 4 * (threadIdx.x % LPR); c < H; c += 4 * LPR)
    store4(x + row * H, c, H, held4(rc, rp, c));
}

// The restored rows and their RMSNorm, the row held in registers between the
// two: LPR lanes, MAXC pieces of four columns each.  32768 x 2048: 130 us, 4.7
// TB/s (a large copy reaches 5.2); a block per row that reads the codes twice
// takes 7 more.
template <int LPR, int MAXC>
__global__ __launch_bounds__(kThreads) void q8_dequantize_rmsnorm_reg(
    const uint8_t* __restrict__ codes, const float* __restrict__ params,
    const float* __restrict__ w, float* __restrict__ x, float* __restrict__ y,
    float* __restrict__ rstd, int64_t rows, int H, int ngroups, float eps) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / LPR) + threadIdx.x / LPR;
  const int sub = threadIdx.x % LPR;
  const bool live = row < rows;
  const uint8_t* rc = codes + (live ? row : 0) * row_bytes(H);
  const float* rp = params + 2 * (live ? row : 0) * ngroups;
  float* xr = x + row * H;
  float* yr = y + row * H;
  f32x4 v[MAXC];
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < MAXC; ++j) {
    const int c = 4 * (sub + j * LPR);
    v[j] = live && c < H ? held4(rc, rp, c) : f32x4{0.f, 0.f, 0.f, 0.f};
    if (c + 4 > H) {  // the row's last piece: no padding in the sum
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (c + e >= H) v[j][e] = 0.f;
    }
  }
#pragma unroll
  for (int j = 0; j < MAXC; ++j) {
    const int c = 4 * (sub + j * LPR);
    if (live && c < H) store4(xr, c, H, v[j]);
  }
#pragma unroll
  for (int j = 0; j < MAXC; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) ss = fmaf(v[j][e], v[j][e], ss);
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o, kWave);
  if (!live) return;
  const float s = 1.0f / sqrtf(ss / static_cast<float>(H) + eps);
  if (rstd && sub == 0) rstd[row] = s;
#pragma unroll
  for (int j = 0; j < MAXC; ++j) {
    const int c = 4 * (sub + j * LPR);
    if (c >= H) break;
    const f32x4 ww = load4<false>(w, c, H);
    f32x4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = v[j][e] * s * ww[e];
    store4(yr, c, H, o);
  }
}

// The same a block per row, the codes read twice: for rows of any width, and
// for so few rows that a wave each would leave most of the GPU idle (511 x 576:
// 3.7 against 3.9 us, 300 x 2048: 4.8 against 6.1; at 1500 x 2048 already 9.2
// against 8.6, at 2048 x 2048 11.8 both).
__global__ __launch_bounds__(kThreads) void q8_dequantize_rmsnorm_wide(
    const uint8_t* __restrict__ codes, const float* __restrict__ params,
    const float* __restrict__ w, float* __restrict__ x, float* __restrict__ y,
    float* __restrict__ rstd, int64_t H, int64_t ngroups, float eps) {
  __shared__ float red[kThreads / kWave];
  const int64_t row = blockIdx.x;
  const uint8_t* rc = codes + row * row_bytes(H);
  const float* rp = params + 2 * row * ngroups;
  float ss = 0.f;
  for (int64_t c = 4 * threadIdx.x; c < H; c += 4 * kThreads) {
    const f32x4 v = held4(rc, rp, c);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (c + e < H) ss = fmaf(v[e], v[e], ss);
    store4(x + row * H, c, H, v);
  }
  ss = block_sum(ss, red);
  const float s = 1.0f / sqrtf(ss / static_cast<float>(H) + eps);
  if (rstd && threadIdx.x == 0) rstd[row] = s;
  for (int64_t c = 4 * threadIdx.x; c < H; c += 4 * kThreads) {
    f32x4 v = held4(rc, rp, c);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (c + e < H) v[e] = v[e] * s * w[c + e];
    store4(y + row * H, c, H, v);
  }
}

// Lanes per row: enough for its pieces of four columns, up to a wave.
int lanes_per_row(int64_t H) {
  int lpr = 8;
  while (lpr < kWave && 4 * lpr < H) lpr <<= 1;
  return lpr;
}

constexpr int64_t kFewRows = 2048;

// A launch holds fewer than 2^32 threads: a block per row, 2^24 of them, would not fit.
constexpr int64_t kLaunchRows = int64_t{1} << 22;

// run(first row, rows) for all rows, kLaunchRows at most at a time.
template <typename Run>
int by_launches(int64_t rows, Run run) {
  for (int64_t r = 0; r < rows; r += kLaunchRows) {
    run(r, rows - r < kLaunchRows ? rows - r : kLaunchRows);
    if (const int rc = launch_status()) return rc;
  }
  return EMBER_OK;
}

// Blocks that quantise: several groups each, to keep the loads of some waves beside
// the arithmetic of others.
constexpr int64_t kQuantizeBlocks = 4096;

// The rows' size in bytes, and that of their codes and pairs, are 64-bit numbers.
bool sizes_fit(int64_t rows, int64_t H) {
  return H <= INT64_MAX / 32 && fits64(rows, H + 16, sizeof(float));
}

bool aligned8(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7u) == 0; }

}  // namespace

extern "C" size_t ember_q8_code_bytes(int64_t rows, int64_t H) {
  return rows > 0 && H > 0 && sizes_fit(rows, H) ? static_cast<size_t>(rows * row_bytes(H)) : 0;
}

extern "C" size_t ember_q8_param_bytes(int64_t rows, int64_t H) {
  return rows > 0 && H > 0 && sizes_fit(rows, H)
             ? static_cast<size_t>(rows * row_groups(H)) * 2 * sizeof(float)
             : 0;
}

extern "C" int ember_q8_quantize(const float* x, void* codes, float* params, int64_t rows,
                                 int64_t H, ember_stream_t s) {
  if (rows < 0 || H < 0 || rows > 0x7fffffff) return EMBER_EINVAL;  // what can be restored
  if (rows == 0 || H == 0) return EMBER_OK;
  if (!sizes_fit(rows, H)) return EMBER_EINVAL;
  if (!x || !codes || !params) return EMBER_EINVAL;
  if (!aligned16(codes) || !aligned8(params)) return EMBER_EALIGN;
  const int64_t ng = row_groups(H);
  const unsigned grid = grid_1d(rows * ng, kThreads / kLpg, kQuantizeBlocks);
  q8_quantize_kernel<<<grid, kThreads, 0, as_stream(s)>>>(x, static_cast<uint8_t*>(codes), params,
                                                          rows, H, ng);
  return launch_status();
}

extern "C" int ember_q8_dequantize(const void* codes, const float* params, float* x, int64_t rows,
                                   int64_t H, ember_stream_t s) {
  if (rows < 0 || H < 0 || rows > 0x7fffffff) return EMBER_EINVAL;
  if (rows == 0 || H == 0) return EMBER_OK;
  if (!sizes_fit(rows, H)) return EMBER_EINVAL;
  if (!x || !codes || !params) return EMBER_EINVAL;
  if (!aligned16(codes) || !aligned8(params)) return EMBER_EALIGN;
  const auto* c = static_cast<const uint8_t*>(codes);
  const int64_t ng = row_groups(H);
  auto launch = [&](auto lanes) {
    constexpr int LPR = decltype(lanes)::value;
    constexpr int RPB = kThreads / LPR;
    return by_launches(rows, [&](int64_t r, int64_t n) {
      q8_dequantize_kernel<LPR><<<static_cast<unsigned>((n + RPB - 1) / RPB), kThreads, 0,
                                  as_stream(s)>>>(c + r * row_bytes(H), params + 2 * r * ng,
                                                  x + r * H, n, H, ng);
    });
  };
  switch (lanes_per_row(H)) {
    case 8: return launch(std::integral_constant<int, 8>{});
    case 16: return launch(std::integral_constant<int, 16>{});
    case 32: return launch(std::integral_constant<int, 32>{});
    default: return launch(std::integral_constant<int, 64>{});
  }
}

extern "C" int ember_q8_dequantize_rmsnorm(const void* codes, const float* params, const float* w,
                                           float* x, float* y, float* rstd, int64_t rows,
                                           int64_t H, float eps, ember_stream_t s) {
  if (rows < 0 || H < 0 || rows > 0x7fffffff) return EMBER_EINVAL;
  if (rows == 0 || H == 0) return EMBER_OK;
  if (!sizes_fit(rows, H)) return EMBER_EINVAL;
  if (!x || !y || !w || !codes || !params) return EMBER_EINVAL;
  if (!aligned16(codes) || !aligned8(params)) return EMBER_EALIGN;
  const auto* c = static_cast<const uint8_t*>(codes);
  const int64_t ng = row_groups(H);
  if (rows < kFewRows || H > 4 * 64 * 16)
    return by_launches(rows, [&](int64_t r, int64_t n) {
      q8_dequantize_rmsnorm_wide<<<static_cast<unsigned>(n), kThreads, 0, as_stream(s)>>>(
          c + r * row_bytes(H), params + 2 * r * ng, w, x + r * H, y + r * H,
          rstd ? rstd + r : nullptr, H, ng, eps);
    });
  auto launch = [&](auto lanes, auto pieces) {
    constexpr int LPR = decltype(lanes)::value, MAXC = decltype(pieces)::value;
    constexpr int RPB = kThreads / LPR;
    return by_launches(rows, [&](int64_t r, int64_t n) {
      q8_dequantize_rmsnorm_reg<LPR, MAXC>
          <<<static_cast<unsigned>((n + RPB - 1) / RPB), kThreads, 0, as_stream(s)>>>(
              c + r * row_bytes(H), params + 2 * r * ng, w, x + r * H, y + r * H,
              rstd ? rstd + r : nullptr, n, static_cast<int>(H), static_cast<int>(ng), eps);
    });
  };
  using std::integral_constant;
  switch (lanes_per_row(H)) {
    case 8: return launch(integral_constant<int, 8>{}, integral_constant<int, 1>{});
    case 16: return launch(integral_constant<int, 16>{}, integral_constant<int, 1>{});
    case 32: return launch(integral_constant<int, 32>{}, integral_constant<int, 1>{});
    default: break;
  }
  using W = integral_constant<int, 64>;
  if (H <= 4 * 64 * 4) return launch(W{}, integral_constant<int, 4>{});
  if (H <= 4 * 64 * 8) return launch(W{}, integral_constant<int, 8>{});
  return launch(W{}, integral_constant<int, 16>{});
}
