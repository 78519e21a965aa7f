// A KV cache held in 4 bits, and attention over it.
//
// Layout: codes [B, Hk, S, D/8] 32-bit words, eight 4-bit codes each with the
// first of them in the lowest bits, and params [B, Hk, S, 2] = {lo, step}: one
// group (quant.h, 15 steps) per head row of D values, so a row of D = 128 takes
// 72 bytes where the fp32 cache (kvcache.hip) takes 512.  Rows are otherwise as
// in that cache: one KV head's rows are contiguous.
//
// Over a row of codes c the score of a query is
//   q . k = step (q . c) + lo sum(q),
// and a value row adds p lo + (p step) c to the output.
#include <cmath>

#include "common.h"
#include "quant.h"

using namespace ember;

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kMaxD = 256;  // of write and read; the attention takes 64 and 128

// ------------------------------------------------------------ write, read
// src rows [B,T,Hk,D] (blockIdx.y: keys or values) -> cache rows pos + t.
// LPR lanes per row (a power of two >= D/8), eight values a lane.
struct WriteArgs {
  const float* src[2];
  uint32_t* codes[2];
  float* params[2];
  int64_t rows, T, Hk, S, pos;
  int words;  // D / 8
};

template <int LPR>
__global__ __launch_bounds__(kThreads) void kv4_write_kernel(WriteArgs a) {
  const int z = blockIdx.y;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (kThreads / LPR);
  const int w = threadIdx.x % LPR;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * (kThreads / LPR); base < a.rows;
       base += step) {
    const int64_t r = base + threadIdx.x / LPR;
    const bool live = r < a.rows && w < a.words;
    float v[8] = {};
    if (live) {
      const f32x4* p =
          reinterpret_cast<const f32x4*>(a.src[z] + (r * a.words + w) * 8);
      const f32x4 x = p[0], y = p[1];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = x[e];
        v[4 + e] = y[e];
      }
    }
    float lo = INFINITY, hi = -INFINITY;
    bool bad = false;
    if (live) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        lo = fminf(lo, v[e]);
        hi = fmaxf(hi, v[e]);
        bad |= not_finite(v[e]);
      }
    }
    const QuantGrid g = quant_grid<LPR, 15>(lo, hi, bad);
    if (!live) continue;
    uint32_t word = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) word |= quant_code<15>(g, v[e]) << (4 * e);
    const int64_t h = r % a.Hk, t = r / a.Hk % a.T, b = r / (a.Hk * a.T);
    const int64_t row = (b * a.Hk + h) * a.S + a.pos + t;
    a.codes[z][row * a.words + w] = word;
    if (w == 0) *reinterpret_cast<float2*>(a.params[z] + 2 * row) = float2{g.lo, g.step};
  }
}

__device__ __forceinline__ void held8(uint32_t word, float2 p, float (&x)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e)
    x[e] = fmaf(static_cast<float>((word >> (4 * e)) & 15u), p.y, p.x);
}

// Cache rows [0, L) -> out [B, Hk*group, L, D]; a thread reads one word and
// writes its eight values to every head of the group.
__global__ __launch_bounds__(kThreads) void kv4_read_expanded_kernel(
    const uint32_t* __restrict__ codes, const float* __restrict__ params, float* __restrict__ out,
    int64_t n, int64_t group, int64_t L, int64_t S, int words) {
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kThreads;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < n;
       i += stride) {
    const int64_t w = i % words, j = i / words % L, bh = i / (words * L);
    const int64_t row = bh * S + j;
    float x[8];
    held8(codes[row * words + w], *reinterpret_cast<const float2*>(params + 2 * row), x);
    for (int64_t h = 0; h < group; ++h) {
      f32x4* o = reinterpret_cast<f32x4*>(out) + (((bh * group + h) * L + j) * words + w) * 2;
      o[0] = f32x4{x[0], x[1], x[2], x[3]};
      o[1] = f32x4{x[4], x[5], x[6], x[7]};
    }
  }
}

// ---------------------------------------------------------------- attention
// Query rows of a KV head: r -> (t = r / G, h = hk*G + r % G), G = H / Hk.
constexpr int kRowTile = 4;
constexpr int kMinKeysPerSplit = 32;
constexpr int kTargetBlocks = 512;
constexpr int kMaxSplits = 1024;

struct AttnArgs {
  const float* q;  // [B, T, H, D]
  const uint32_t* kc;
  const float* kp;
  const uint32_t* vc;
  const float* vp;
  float* o;        // [B, T, H, D]
  float* part_o;   // [B*T*H, nsplit, D]: each split's unnormalised sums
  float* part_ml;  // [B*T*H, nsplit, 2]: its maximum (log2 units) and weight sum
  int64_t T, H, Hk, L, pos, S;
  int64_t kps;  // keys per split
  int nsplit, row_tiles;
  float qscale;  // scale * log2(e)
};

// A workgroup owns one (batch, KV head, row tile, key split); a key's words
// lie over D/8 lanes, which form one group with an online softmax of its own.
template <int D>
__global__ __launch_bounds__(kThreads) void attn_kv4_kernel(AttnArgs a) {
  constexpr int LPK = D / 8, KPW = kWave / LPK, NG = kWaves * KPW;
  __shared__ float s_ml[NG][kRowTile][2];
  __shared__ float s_o[NG][kRowTile][D];
  const int lane = threadIdx.x & (kWave - 1), wv = threadIdx.x / kWave;
  const int w = lane % LPK, gid = wv * KPW + lane / LPK;
  const int64_t G = a.H / a.Hk, R = G * a.T;
  const int64_t split = blockIdx.x % a.nsplit, rest = blockIdx.x / a.nsplit;
  const int64_t r0 = rest % a.row_tiles * kRowTile, bh = rest / a.row_tiles;
  const int64_t hk = bh % a.Hk, b = bh / a.Hk;
  const int64_t ks = split * a.kps, ke = ks + a.kps < a.L ? ks + a.kps : a.L;
  const int nr = static_cast<int>(R - r0 < kRowTile ? R - r0 : kRowTile);

  float q[kRowTile][8], acc[kRowTile][8], m[kRowTile], l[kRowTile], qsum[kRowTile];
  int64_t lim[kRowTile], jend = ks;
#pragma unroll
  for (int r = 0; r < kRowTile; ++r) {
    m[r] = -INFINITY;
    l[r] = qsum[r] = 0.f;
    lim[r] = ks;
#pragma unroll
    for (int e = 0; e < 8; ++e) q[r][e] = acc[r][e] = 0.f;
    if (r < nr) {
      const int64_t t = (r0 + r) / G, h = hk * G + (r0 + r) % G;
      const float* p = a.q + ((b * a.T + t) * a.H + h) * D + 8 * w;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        q[r][e] = p[e] * a.qscale;
        qsum[r] += q[r][e];
      }
      const int64_t c = a.pos + t + 1;
      lim[r] = c < ke ? c : ke;
      jend = lim[r] > jend ? lim[r] : jend;
    }
  }
  for (int64_t j = ks + gid; j < jend; j += NG) {
    const int64_t row = bh * a.S + j;
    const uint32_t kw = a.kc[row * LPK + w], vw = a.vc[row * LPK + w];
    const float2 kp = *reinterpret_cast<const float2*>(a.kp + 2 * row);
    const float2 vp = *reinterpret_cast<const float2*>(a.vp + 2 * row);
    float kx[8], vx[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) kx[e] = static_cast<float>((kw >> (4 * e)) & 15u);
    held8(vw, vp, vx);
#pragma unroll
    for (int r = 0; r < kRowTile; ++r) {
      float d = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) d = fmaf(q[r][e], kx[e], d);
      float sc = fmaf(d, kp.y, qsum[r] * kp.x);
#pragma unroll
      for (int o = LPK / 2; o > 0; o >>= 1) sc += __shfl_xor(sc, o, kWave);
      if (j < lim[r]) {
        const float mx = fmaxf(m[r], sc);
        const float c = exp2f(m[r] - mx), p = exp2f(sc - mx);
        l[r] = l[r] * c + p;
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[r][e] = acc[r][e] * c + p * vx[e];
        m[r] = mx;
      }
    }
  }
#pragma unroll
  for (int r = 0; r < kRowTile; ++r) {
#pragma unroll
    for (int e = 0; e < 8; ++e) s_o[gid][r][8 * w + e] = acc[r][e];
    if (w == 0) {
      s_ml[gid][r][0] = m[r];
      s_ml[gid][r][1] = l[r];
    }
  }
  __syncthreads();
  for (int it = threadIdx.x; it < nr * D; it += kThreads) {
    const int r = it / D, d = it % D;
    float M = -INFINITY;
    for (int g = 0; g < NG; ++g) M = fmaxf(M, s_ml[g][r][0]);
    float ls = 0.f, os = 0.f;
    for (int g = 0; g < NG; ++g) {
      const float e = s_ml[g][r][0] == -INFINITY ? 0.f : exp2f(s_ml[g][r][0] - M);
      ls += s_ml[g][r][1] * e;
      os += s_o[g][r][d] * e;
    }
    const int64_t t = (r0 + r) / G, h = hk * G + (r0 + r) % G;
    const int64_t orow = (b * a.T + t) * a.H + h;
    if (a.nsplit == 1) {
      a.o[orow * D + d] = os / ls;
    } else {
      a.part_o[(orow * a.nsplit + split) * D + d] = os;
      if (d == 0) {
        a.part_ml[(orow * a.nsplit + split) * 2] = M;
        a.part_ml[(orow * a.nsplit + split) * 2 + 1] = ls;
      }
    }
  }
}

// Merges a row's splits in split order: a block per row, D threads.
__global__ void attn_kv4_combine(const float* __restrict__ part_o,
                                 const float* __restrict__ part_ml, float* __restrict__ o,
                                 int nsplit, int D) {
  const int64_t row = blockIdx.x;
  const float* ml = part_ml + row * nsplit * 2;
  float M = -INFINITY;
  for (int s = 0; s < nsplit; ++s) M = fmaxf(M, ml[2 * s]);
  float ls = 0.f, os = 0.f;
  for (int s = 0; s < nsplit; ++s) {
    const float e = ml[2 * s] == -INFINITY ? 0.f : exp2f(ml[2 * s] - M);
    ls += ml[2 * s + 1] * e;
    os += part_o[(row * nsplit + s) * D + threadIdx.x] * e;
  }
  o[row * D + threadIdx.x] = os / ls;
}

struct Plan {
  int nsplit, row_tiles;
  int64_t kps;
};

Plan attn_plan(int64_t B, int64_t T, int64_t H, int64_t Hk, int64_t L) {
  const int64_t tiles = (H / Hk * T + kRowTile - 1) / kRowTile;
  const int64_t heads = B * Hk * tiles;
  int64_t want = (kTargetBlocks + heads - 1) / heads;
  const int64_t most = (L + kMinKeysPerSplit - 1) / kMinKeysPerSplit;
  if (want > most) want = most;
  if (want > kMaxSplits) want = kMaxSplits;
  const int64_t kps = (L + want - 1) / want;
  return Plan{static_cast<int>((L + kps - 1) / kps), static_cast<int>(tiles), kps};
}

bool aligned8(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7u) == 0; }

}  // namespace

extern "C" int ember_kv4_write(const float* k, const float* v, uint32_t* k_codes, float* k_params,
                               uint32_t* v_codes, float* v_params, int64_t B, int64_t T,
                               int64_t Hk, int64_t D, int64_t S, int64_t pos, ember_stream_t s) {
  if (B < 0 || T < 0 || Hk < 0 || pos < 0 || T > S || pos > S - T) return EMBER_EINVAL;
  if (D < 8 || D > kMaxD || D % 8) return EMBER_EINVAL;
  if (B * T * Hk == 0) return EMBER_OK;
  if (!k || !v || !k_codes || !k_params || !v_codes || !v_params) return EMBER_EINVAL;
  if (!aligned16(k) || !aligned16(v) || !aligned16(k_codes) || !aligned16(v_codes) ||
      !aligned8(k_params) || !aligned8(v_params))
    return EMBER_EALIGN;
  WriteArgs a{{k, v}, {k_codes, v_codes}, {k_params, v_params}, B * T * Hk, T, Hk, S, pos,
              static_cast<int>(D / 8)};
  auto launch = [&](auto lpr) {
    constexpr int LPR = decltype(lpr)::value;
    const dim3 grid(grid_1d(a.rows, kThreads / LPR), 2);
    kv4_write_kernel<LPR><<<grid, kThreads, 0, as_stream(s)>>>(a);
  };
  if (a.words <= 8)
    launch(std::integral_constant<int, 8>{});
  else if (a.words <= 16)
    launch(std::integral_constant<int, 16>{});
  else
    launch(std::integral_constant<int, 32>{});
  return launch_status();
}

extern "C" int ember_kv4_read_expanded(const uint32_t* codes, const float* params, float* out,
                                       int64_t B, int64_t Hk, int64_t group, int64_t L, int64_t D,
                                       int64_t S, ember_stream_t s) {
  if (B < 0 || Hk < 0 || group <= 0 || L < 0 || L > S) return EMBER_EINVAL;
  if (D < 8 || D > kMaxD || D % 8) return EMBER_EINVAL;
  const int64_t n = B * Hk * L * (D / 8);
  if (n == 0) return EMBER_OK;
  if (!codes || !params || !out) return EMBER_EINVAL;
  if (!aligned16(codes) || !aligned16(out) || !aligned8(params)) return EMBER_EALIGN;
  kv4_read_expanded_kernel<<<grid_1d(n, kThreads), kThreads, 0, as_stream(s)>>>(
      codes, params, out, n, group, L, S, static_cast<int>(D / 8));
  return launch_status();
}

extern "C" size_t ember_attn_kv4_workspace_bytes(int64_t B, int64_t T, int64_t H, int64_t Hk,
                                                 int64_t D, int64_t L) {
  if (B <= 0 || T <= 0 || H <= 0 || Hk <= 0 || H % Hk || D <= 0 || L <= 0) return 0;
  const Plan p = attn_plan(B, T, H, Hk, L);
  if (p.nsplit == 1) return 0;
  return static_cast<size_t>(B * T * H) * p.nsplit * (D + 2) * sizeof(float);
}

extern "C" int ember_attn_kv4(const float* q, const uint32_t* k_codes, const float* k_params,
                              const uint32_t* v_codes, const float* v_params, float* o, int64_t B,
                              int64_t T, int64_t H, int64_t Hk, int64_t D, int64_t L, int64_t pos,
                              int64_t S, float scale, void* workspace, size_t workspace_bytes,
                              ember_stream_t s) {
  if (B < 0 || T < 0 || H <= 0 || Hk <= 0 || H % Hk != 0 || pos < 0) return EMBER_EINVAL;
  if (D != 64 && D != 128) return EMBER_EINVAL;
  if (B == 0 || T == 0) return EMBER_OK;
  if (L < 1 || L > S || S > 0x7fffffff) return EMBER_EINVAL;
  if (!q || !k_codes || !k_params || !v_codes || !v_params || !o) return EMBER_EINVAL;
  if (!aligned16(q) || !aligned16(o) || !aligned16(k_codes) || !aligned16(v_codes) ||
      !aligned8(k_params) || !aligned8(v_params))
    return EMBER_EALIGN;
  const Plan p = attn_plan(B, T, H, Hk, L);
  const int64_t blocks = B * Hk * p.row_tiles * p.nsplit;
  if (blocks > 0x7fffffff) return EMBER_EINVAL;
  const size_t need = ember_attn_kv4_workspace_bytes(B, T, H, Hk, D, L);
  if (need && (!workspace || workspace_bytes < need)) return EMBER_EWORKSPACE;
  if (need && !aligned16(workspace)) return EMBER_EALIGN;
  const int64_t rows = B * T * H;
  AttnArgs a{};
  a.q = q;
  a.kc = k_codes;
  a.kp = k_params;
  a.vc = v_codes;
  a.vp = v_params;
  a.o = o;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = need ? a.part_o + rows * p.nsplit * D : nullptr;
  a.T = T;
  a.H = H;
  a.Hk = Hk;
  a.L = L;
  a.pos = pos;
  a.S = S;
  a.kps = p.kps;
  a.nsplit = p.nsplit;
  a.row_tiles = p.row_tiles;
  a.qscale = scale * 1.4426950408889634f;
  hipStream_t st = as_stream(s);
  const unsigned grid = static_cast<unsigned>(blocks);
  if (D == 128)
    attn_kv4_kernel<128><<<grid, kThreads, 0, st>>>(a);
  else
    attn_kv4_kernel<64><<<grid, kThreads, 0, st>>>(a);
  const int rc = launch_status();
  if (rc || p.nsplit == 1) return rc;
  attn_kv4_combine<<<static_cast<unsigned>(rows), static_cast<unsigned>(D), 0, st>>>(
      a.part_o, a.part_ml, o, p.nsplit, static_cast<int>(D));
  return launch_status();
}
