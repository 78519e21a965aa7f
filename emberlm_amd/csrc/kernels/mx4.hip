// Weights in microscaled 4-bit floating point (the form is in mx4.h): brought
// into it, read back, and looked up by row.  All three are bound by the fp32
// side's HBM traffic (4 bytes a value against 17/32): a table of 151936 x 2048 is
// brought into it in 263-305 us and read back in 259-272 (4.6 to 5.4 TB/s), 4096 of its
// rows looked up in 12.2 (lines of 128 bytes for runs of 16, mx4_embedding_kernel).  The reference holds its weights
// in fp32 only.
#include "mx4.h"

using namespace ember;

namespace {

constexpr int kThreads = 256;
constexpr int kCols = 256;  // columns of a workgroup's block: one block of scales
constexpr int64_t kMaxGrid = int64_t(1) << 20;  // workgroups; more blocks loop

// Columns [c, c + 4) of a row of K floats; zeros past its end.  VEC: rows are
// whole aligned float4s.
template <bool VEC>
__device__ __forceinline__ f32x4 load4(const float* __restrict__ row, int64_t c, int64_t K) {
  if constexpr (VEC) {
    return c < K ? *reinterpret_cast<const f32x4*>(row + c) : f32x4{0.f, 0.f, 0.f, 0.f};
  } else {
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = c + e < K ? row[c + e] : 0.f;
    return v;
  }
}

template <bool VEC>
__device__ __forceinline__ void store4(float* __restrict__ row, int64_t c, int64_t K, f32x4 v) {
  if constexpr (VEC) {
    if (c < K) *reinterpret_cast<f32x4*>(row + c) = v;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (c + e < K) row[c + e] = v[e];
  }
}

// 32 rows by 256 columns a workgroup: eight lanes a row, four values of a group
// each, so that a wave's load takes eight whole 128-byte lines.  Two groups'
// codes are traded between neighbouring lanes: the even one then stores four
// bytes of the first, the odd one four of the second.
template <bool VEC>
__global__ __launch_bounds__(kThreads) void mx4_quantize_kernel(
    const float* __restrict__ w, uint32_t* __restrict__ codes, uint32_t* __restrict__ scales,
    int64_t N, int64_t K, int64_t kb, int64_t ks, int64_t blocks) {
  const int r = threadIdx.x / 8, c8 = threadIdx.x % 8;
  for (int64_t blk = blockIdx.x; blk < blocks; blk += gridDim.x) {
    const int64_t nb = blk / ks, kc = blk % ks;
    const int64_t n = nb * 32 + r;
    const float* row = w + n * K;
    f32x4 v[8];
#pragma unroll
    for (int g = 0; g < 8; ++g)
      v[g] = n < N ? load4<VEC>(row, kc * kCols + 32 * g + 4 * c8, K) : f32x4{0.f, 0.f, 0.f, 0.f};
    uint32_t sc[2] = {0, 0};  // of halves 0 and 1 of the four tiles
    uint32_t mine[8];
#pragma unroll
    for (int g = 0; g < 8; ++g) {
      unsigned top = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(v[g][e]) & 0x7fffffffu);
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) top = max(top, __shfl_xor(top, o, kWave));
      const unsigned byte = mx4_scale_byte(top);
      sc[g % 2] |= byte << (8 * (g / 2));
      mine[g] = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        mine[g] |= mx4_code(v[g][e], static_cast<int>(byte)) << (4 * e);
      if (byte == 255u) mine[g] = 0;
    }
    const bool odd = c8 & 1;
#pragma unroll
    for (int t = 0; t < 4; ++t) {  // tile t of the block: groups 2t (h = 0) and 2t + 1
      const uint32_t got = __shfl_xor(odd ? mine[2 * t] : mine[2 * t + 1], 1, kWave);
      const uint32_t word = odd ? got | mine[2 * t + 1] << 16 : mine[2 * t] | got << 16;
      if (kc * 4 + t < kb)
        codes[(nb * kb + kc * 4 + t) * (kMx4TileBytes / 4) + (32 * odd + r) * 4 + c8 / 2] = word;
    }
    if (c8 < 2) scales[blk * (kMx4ScaleBytes / 4) + 32 * c8 + r] = sc[c8];
  }
}

// The reverse: a lane reads four bytes of a group, gives its neighbour the half
// that is not its own, and stores four values of either half's group.
template <bool VEC>
__global__ __launch_bounds__(kThreads) void mx4_dequantize_kernel(
    const uint32_t* __restrict__ codes, const uint32_t* __restrict__ scales, float* __restrict__ w,
    int64_t N, int64_t K, int64_t kb, int64_t ks, int64_t blocks) {
  const int r = threadIdx.x / 8, c8 = threadIdx.x % 8;
  const bool odd = c8 & 1;
  for (int64_t blk = blockIdx.x; blk < blocks; blk += gridDim.x) {
    const int64_t nb = blk / ks, kc = blk % ks;
    const int64_t n = nb * 32 + r;
    const uint32_t sc[2] = {scales[blk * (kMx4ScaleBytes / 4) + r],
                            scales[blk * (kMx4ScaleBytes / 4) + 32 + r]};
    uint32_t word[4];
#pragma unroll
    for (int t = 0; t < 4; ++t)
      word[t] = kc * 4 + t < kb ? codes[(nb * kb + kc * 4 + t) * (kMx4TileBytes / 4) +
                                        (32 * odd + r) * 4 + c8 / 2]
                                : 0u;
    float* row = w + n * K;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint32_t got = __shfl_xor(odd ? word[t] & 0xffffu : word[t] >> 16, 1, kWave);
      const uint32_t of0 = odd ? got : word[t], of1 = odd ? word[t] >> 16 : got;
      const int64_t c = kc * kCols + 64 * t + 4 * c8;
      if (n < N) {
        store4<VEC>(row, c, K, mx4_values(of0, sc[0] >> (8 * t) & 255u));
        store4<VEC>(row, c + 32, K, mx4_values(of1, sc[1] >> (8 * t) & 255u));
      }
    }
  }
}

// One wave per (id, BLOCKS blocks of 256 columns): lane i takes columns 4 i of each.
// A row of the table lies in runs of 16 bytes, two a tile, and of 4 for the scales, each
// in a line of 128 that its neighbours share: for 1088 bytes of a row of 2048 columns some
// 10 KB cross the caches beside the 8 KB that are written.
template <bool VEC, int BLOCKS>
__global__ __launch_bounds__(kThreads) void mx4_embedding_kernel(
    const int64_t* __restrict__ ids, const uint16_t* __restrict__ codes,
    const uint8_t* __restrict__ scales, float* __restrict__ out, int64_t n, int64_t K, int64_t V,
    int64_t kb, int64_t ks) {
  const int lane = threadIdx.x & (kWave - 1);
  constexpr int kWaves = kThreads / kWave;
  const int64_t groups = (ks + BLOCKS - 1) / BLOCKS;
  for (int64_t it = static_cast<int64_t>(blockIdx.x) * kWaves + threadIdx.x / kWave;
       it < n * groups; it += static_cast<int64_t>(gridDim.x) * kWaves) {
    const int64_t i = it / groups, first = it % groups * BLOCKS;
    const int64_t id = ids[i];
    const bool known = id >= 0 && id < V;
    const int64_t nb = id / 32, r = id % 32;
    const int t = lane / 16, h = lane / 8 % 2;
    unsigned byte[BLOCKS], code[BLOCKS];
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
      const int64_t kc = first + b;
      byte[b] = code[b] = 0;
      if (!known || kc * kCols + 4 * lane >= K) continue;
      byte[b] = scales[(nb * ks + kc) * kMx4ScaleBytes + (32 * h + r) * 4 + t];
      code[b] = codes[(nb * kb + kc * 4 + t) * (kMx4TileBytes / 2) + (32 * h + r) * 8 + lane % 8];
    }
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b)
      store4<VEC>(out + i * K, (first + b) * kCols + 4 * lane, K,
                  mx4_values(code[b], static_cast<int>(byte[b])));
  }
}

// A lookup of more blocks than the GPU has room for waves takes two of them a wave, whose
// loads go out together (32768 rows of K = 2048 113.6 -> 96.0 us, four a wave 97.6; 2048
// rows 8.1 -> 7.5, and 8.5).
constexpr int kWide = 2;
constexpr int64_t kManyBlocks = 8192;

bool vec(const float* w, int64_t K) { return K % 4 == 0 && aligned16(w); }

unsigned grid_of(int64_t blocks) {
  return static_cast<unsigned>(blocks < kMaxGrid ? blocks : kMaxGrid);
}

}  // namespace

extern "C" size_t ember_mx4_code_bytes(int64_t N, int64_t K) {
  if (!mx4_sizes_ok(N, K)) return 0;
  return static_cast<size_t>(mx4_row_tiles(N) * mx4_col_tiles(K)) * kMx4TileBytes;
}

extern "C" size_t ember_mx4_scale_bytes(int64_t N, int64_t K) {
  if (!mx4_sizes_ok(N, K)) return 0;
  return static_cast<size_t>(mx4_row_tiles(N) * mx4_col_blocks(K)) * kMx4ScaleBytes;
}

extern "C" int ember_mx4_quantize(const float* w, void* codes, void* scales, int64_t N, int64_t K,
                                  ember_stream_t s) {
  if (!mx4_sizes_ok(N, K)) return EMBER_EINVAL;
  if (N == 0) return EMBER_OK;
  if (!w || !codes || !scales) return EMBER_EINVAL;
  if (!aligned16(codes) || !aligned16(scales)) return EMBER_EALIGN;
  const int64_t kb = mx4_col_tiles(K), ks = mx4_col_blocks(K), blocks = mx4_row_tiles(N) * ks;
  auto* kernel = vec(w, K) ? mx4_quantize_kernel<true> : mx4_quantize_kernel<false>;
  kernel<<<grid_of(blocks), kThreads, 0, as_stream(s)>>>(w, static_cast<uint32_t*>(codes),
                                                         static_cast<uint32_t*>(scales), N, K, kb,
                                                         ks, blocks);
  return launch_status();
}

extern "C" int ember_mx4_dequantize(const void* codes, const void* scales, float* w, int64_t N,
                                    int64_t K, ember_stream_t s) {
  if (!mx4_sizes_ok(N, K)) return EMBER_EINVAL;
  if (N == 0) return EMBER_OK;
  if (!w || !codes || !scales) return EMBER_EINVAL;
  if (!aligned16(codes) || !aligned16(scales)) return EMBER_EALIGN;
  const int64_t kb = mx4_col_tiles(K), ks = mx4_col_blocks(K), blocks = mx4_row_tiles(N) * ks;
  auto* kernel = vec(w, K) ? mx4_dequantize_kernel<true> : mx4_dequantize_kernel<false>;
  kernel<<<grid_of(blocks), kThreads, 0, as_stream(s)>>>(static_cast<const uint32_t*>(codes),
                                                         static_cast<const uint32_t*>(scales), w, N,
                                                         K, kb, ks, blocks);
  return launch_status();
}

extern "C" int ember_mx4_embedding(const int64_t* ids, const void* codes, const void* scales,
                                   float* out, int64_t n, int64_t K, int64_t V,
                                   ember_stream_t s) {
  if (!mx4_sizes_ok(V, K) || n < 0 || n > 0x7fffffff) return EMBER_EINVAL;
  if (n == 0) return EMBER_OK;
  if (!ids || !out || (V > 0 && (!codes || !scales))) return EMBER_EINVAL;
  if (!aligned16(codes) || !aligned16(scales)) return EMBER_EALIGN;
  const int64_t kb = mx4_col_tiles(K), ks = mx4_col_blocks(K);
  constexpr int kWaves = kThreads / kWave;
  const bool wide = n * ks >= kManyBlocks;
  auto* kernel = vec(out, K) ? wide ? mx4_embedding_kernel<true, kWide> : mx4_embedding_kernel<true, 1>
                 : wide      ? mx4_embedding_kernel<false, kWide>
                             : mx4_embedding_kernel<false, 1>;
  const int64_t groups = wide ? (ks + kWide - 1) / kWide : ks;
  kernel<<<grid_of((n * groups + kWaves - 1) / kWaves), kThreads, 0, as_stream(s)>>>(
      ids, static_cast<const uint16_t*>(codes), static_cast<const uint8_t*>(scales), out, n, K, V,
      kb, ks);
  return launch_status();
}
