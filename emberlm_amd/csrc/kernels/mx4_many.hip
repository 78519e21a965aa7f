// Products of many rows of x with weights in microscaled 4-bit floating point
// (the form is in mx4.h): prompts.  Bound by the block-scaled matrix cores.
//
// x enters as five signed base-32 digits a value, a group of 32 values sharing
// one exponent: with s the group's scale, |x| / s < 16, digit 0 is x / s
// rounded to a whole number, digit 1 what is left times 32 rounded, and so on:
// x to 2^-24 of the group's largest.  A whole number up to 16 is an eighth of it
// in e2m3, whose codes to 16 / 8 are the number itself beside a sign; 6-bit
// operands run at the rate of 4-bit ones (5978 TFLOP/s here on random operands;
// 8-bit 3334), the codes beside them are read once for the five.  So a product
// costs five MFMAs' share, 1196 TFLOP/s of fp32-accurate product at that
// rate where bf16 splits of x would have 428 of the library's 1285.
//
// mx4_split_kernel cuts x into digits once a call, times the norm's weight
// where there is one, in the form of the matrix cores' operand: a tile of 32 rows
// by 64 columns is, for each digit, 64 lanes of 16 bytes and then 64 of 8; scales
// lie as the weights' do.  It also leaves each row's sums of squares (per 256
// columns) from which the product's store takes the norm's factor.
//
// Sums: a digit's products and their sums of 64 are exact in the MFMA (8 bits,
// whole numbers of one unit a group); what it adds to is a running fp32 sum, and
// there terms below 2^-27 of the largest are dropped, downwards.  Digits 0 and 1
// and digits 2 to 4 have sums of their own, so that the small ones meet no large
// sum before the end.
#include <algorithm>

#include "mfma_sched.h"
#include "mx4_linear.h"

using namespace ember;

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

constexpr int kDigits = 5;
constexpr int kDigitBytes = 1536;                  // a digit of 32 rows by 64 columns
constexpr int kTileBytes = kDigits * kDigitBytes;  // all of them
constexpr int kSplitThreads = 256;

// Workspace of R rows (whole tiles of 32) by K columns.
struct Space {
  uint8_t* digits;   // [R / 32][kb][kDigits][kDigitBytes]
  uint32_t* scales;  // [R / 32][ks][64]
  float* squares;    // [R][ks]
};
constexpr size_t round256(size_t n) { return (n + 255) / 256 * 256; }
size_t digit_bytes(int64_t tiles, int64_t kb) { return static_cast<size_t>(tiles * kb) * kTileBytes; }
size_t space_bytes(int64_t tiles, int64_t kb, int64_t ks) {
  return round256(digit_bytes(tiles, kb)) + round256(static_cast<size_t>(tiles * ks) * 256) +
         round256(static_cast<size_t>(tiles * 32 * ks) * 4);
}

// v of eight neighbouring lanes combined, in each of them: lane ^ 1, ^ 2, ^ 7.
template <typename F>
__device__ __forceinline__ unsigned over_8(unsigned v, F f) {
  v = f(v, static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, true)));
  v = f(v, static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, true)));
  return f(v, static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, true)));
}

__device__ __forceinline__ f32x4 load_x(const float* __restrict__ row, int64_t c, int64_t K,
                                        bool vec) {
  if (vec) return c < K ? *reinterpret_cast<const f32x4*>(row + c) : f32x4{0.f, 0.f, 0.f, 0.f};
  f32x4 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = c + e < K ? row[c + e] : 0.f;
  return v;
}

// 32 rows by 256 columns a workgroup, eight lanes a row and four values of a group
// each.  Four lanes' 24 bits of a digit are three words: lane j < 3 of four takes
// the rest of its own and the beginning of its neighbour's.
__global__ __launch_bounds__(kSplitThreads) void mx4_split_kernel(Mx4Call c, Space sp,
                                                                  int64_t blocks) {
  const int r = threadIdx.x / 8, c8 = threadIdx.x % 8, j = c8 % 4;
  const int word = 3 * (c8 / 4) + j;  // of a lane's six
  for (int64_t blk = blockIdx.x; blk < blocks; blk += gridDim.x) {
    const int64_t mb = blk / c.ks, kc = blk % c.ks;
    const int64_t m = mb * 32 + r;
    f32x4 v[8];
#pragma unroll
    for (int g = 0; g < 8; ++g)
      v[g] = m < c.M ? load_x(c.x + m * c.K, kc * 256 + 32 * g + 4 * c8, c.K, c.x_vec)
                     : f32x4{0.f, 0.f, 0.f, 0.f};
    if (c.norm_w) {
      float ss = 0.f;
#pragma unroll
      for (int g = 0; g < 8; ++g) {
        ss += v[g].x * v[g].x + v[g].y * v[g].y + v[g].z * v[g].z + v[g].w * v[g].w;
        v[g] *= load_x(c.norm_w, kc * 256 + 32 * g + 4 * c8, c.K, c.x_vec);
      }
      ss = __uint_as_float(over_8(__float_as_uint(ss), [](unsigned a, unsigned b) {
        return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
      }));
      if (c8 == 0) sp.squares[m * c.ks + kc] = ss;
    }
    uint32_t sc[2] = {0, 0};
#pragma unroll
    for (int g = 0; g < 8; ++g) {
      unsigned top = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(v[g][e]) & 0x7fffffffu);
      top = over_8(top, [](unsigned a, unsigned b) { return max(a, b); });
      // 255: a group that is not finite makes its row NaN; 23 and up leave room for
      // the digits' factors 2^-5 .. 2^-20 (and the eighths')
      const int byte = top >= 0x7f800000u ? 255 : max(static_cast<int>(top >> 23), 23);
      sc[g % 2] |= static_cast<uint32_t>(byte) << (8 * (g / 2));
      f32x4 t;
#pragma unroll
      for (int e = 0; e < 4; ++e) t[e] = __builtin_ldexpf(v[g][e], 130 - byte);
      const int64_t kb = kc * 4 + g / 2;
      uint8_t* tile = sp.digits + (mb * c.kb + kb) * kTileBytes;
      const int lane = 32 * (g % 2) + r;
      uint32_t* out = reinterpret_cast<uint32_t*>(
          tile + (word < 4 ? 16 * lane + 4 * word : 1024 + 8 * lane + 4 * (word - 4)));
#pragma unroll
      for (int p = 0; p < kDigits; ++p) {
        unsigned bits = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float d = __builtin_rintf(t[e]);
          const unsigned code = static_cast<unsigned>(fabsf(d)) | (__float_as_uint(d) >> 26 & 32u);
          bits |= code << (6 * e);
          t[e] = (t[e] - d) * 32.f;
        }
        const unsigned next = static_cast<unsigned>(
            __builtin_amdgcn_update_dpp(0, (int)bits, 0xF9, 0xf, 0xf, true));  // lane + 1 of four
        if (j < 3 && kb < c.kb)
          out[p * (kDigitBytes / 4)] = bits >> (8 * j) | next << (24 - 8 * j);
      }
    }
    if (c8 < 2) sp.scales[blk * 64 + 32 * c8 + r] = sc[c8];
  }
}

// A workgroup's WM x WN waves take 32 rows by 32 TN columns each, WK of them the
// same ones at every WK-th tile of K (their sums are joined at the end).  Tiles
// go from global memory to LDS without registers, a ring of three stages of WK
// tiles of K, two ahead, one barrier a stage.
// GATE: half of a wave's TN column tiles are the gate's, half the up
// projection's at the same columns.
template <int WM_, int WN_, int TN_, int WK_, bool GATE_>
struct Shape {
  static constexpr int WM = WM_, WN = WN_, TN = TN_, WK = WK_;
  static constexpr bool GATE = GATE_;
  static constexpr int kWaves = WM * WN * WK;
  static constexpr int kThreads = kWaves * kWave;
  static constexpr int kRowTiles = WM;                       // of x, 32 rows each
  static constexpr int kColTiles = WN * TN;                  // of the weights
  static constexpr int kOutTiles = kColTiles / (GATE ? 2 : 1);
  static constexpr int kABytes = WM * kTileBytes;            // a tile of K
  static constexpr int kTileK = kABytes + kColTiles * kMx4TileBytes;
  static constexpr int kCopies = (WK * kTileK + 1023) / 1024;  // of 1 KB
  static constexpr int kPerWave = (kCopies + kWaves - 1) / kWaves;
  static constexpr int kStage = kPerWave * kWaves * 1024;    // room for every wave's copies
  static constexpr int kStages = 3;
  static_assert(kStages * kStage <= 160 * 1024, "LDS");
};

template <class S>
__global__ __launch_bounds__(S::kThreads) void mx4_gemm_kernel(Mx4Call c, Space sp, Mx4Blocks bl,
                                                               int64_t col_blocks) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[S::kStages * S::kStage];
  constexpr bool GATE = S::GATE;
  const int lane = threadIdx.x & (kWave - 1);
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wk = w % S::WK, wm = w / S::WK % S::WM, wn = w / (S::WK * S::WM);
  // Blocks go round the eight XCDs: each takes a run of tiles, columns first, whose
  // rows of digits stay in its L2.
  const int64_t total = gridDim.x, xcd = blockIdx.x % 8, each = total / 8, more = total % 8;
  const int64_t at = xcd * each + (xcd < more ? xcd : more) + blockIdx.x / 8;
  const int64_t mt = at / col_blocks;
  int64_t nblk = at % col_blocks;
  const int seg = GATE ? 0 : mx4_segment(bl, c.nseg, nblk);
  const int64_t N = c.N[seg];
  const int64_t last_n = (N - 1) / 32, last_m = (c.M - 1) / 32;

  // Column tile q of the block (wave wn's are wn TN .. wn TN + TN - 1); past the end
  // the last one again, not stored.
  auto col_tile = [&](int q) {
    const int64_t t = GATE ? nblk * S::kOutTiles + q / S::TN * (S::TN / 2) + q % S::TN % (S::TN / 2)
                           : nblk * S::kOutTiles + q;
    return t < last_n ? t : last_n;
  };
  auto weight = [&](int q) -> const Mx4Weight& {
    return c.W[GATE ? q % S::TN / (S::TN / 2) : seg];
  };

  // This lane's part of the wave's copies of a stage: 16 bytes each, of the tile of K
  // number `step` of the stage; what lies behind the last one is copied as the first
  // (into room that is not read).
  const uint8_t* src[S::kPerWave];
  int step[S::kPerWave], stride[S::kPerWave];
#pragma unroll
  for (int i = 0; i < S::kPerWave; ++i) {
    int u = ((w + i * S::kWaves) * 64 + lane) * 16;
    if (u >= S::WK * S::kTileK) u = 0;
    step[i] = u / S::kTileK;
    const int in = u % S::kTileK;
    if (in < S::kABytes) {
      const int64_t mb = mt * S::WM + in / kTileBytes;
      src[i] = sp.digits + (mb < last_m ? mb : last_m) * c.kb * kTileBytes + in % kTileBytes;
      stride[i] = kTileBytes;
    } else {
      const int q = (in - S::kABytes) / kMx4TileBytes;
      src[i] = reinterpret_cast<const uint8_t*>(weight(q).codes) +
               col_tile(q) * c.kb * kMx4TileBytes + (in - S::kABytes) % kMx4TileBytes;
      stride[i] = kMx4TileBytes;
    }
  }
  const int64_t kb = c.kb, stages = (kb + S::WK - 1) / S::WK;
  auto issue = [&](int64_t stage, uint8_t* to) {
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
    for (int i = 0; i < S::kPerWave; ++i) {
      int64_t k = stage * S::WK + step[i];
      k = k < kb ? k : kb - 1;  // not read there
      __builtin_amdgcn_global_load_lds(
          reinterpret_cast<const uint32_t*>(src[i] + k * stride[i]),
          (__attribute__((address_space(3))) void*)(to + (w + i * S::kWaves) * 1024), 16, 0, 0);
    }
#endif
  };

  // Scales: one word a lane covers 256 columns.
  const uint32_t* sa_at = sp.scales + (std::min(mt * S::WM + wm, last_m) * c.ks) * 64 + lane;
  const uint32_t* sb_at[S::TN];
#pragma unroll
  for (int t = 0; t < S::TN; ++t)
    sb_at[t] = weight(wn * S::TN + t).scales + col_tile(wn * S::TN + t) * c.ks * 64 + lane;

  f32x16 hi[S::TN] = {}, lo[S::TN] = {};
  int sa[kDigits], sb[S::TN];
  auto load_scales = [&](int64_t ks, uint32_t& a, uint32_t (&b)[S::TN]) {
    a = sa_at[ks * 64];
#pragma unroll
    for (int t = 0; t < S::TN; ++t) b[t] = sb_at[t][ks * 64];
  };

  // The products of one tile of K: byte J of the scales.
  auto compute = [&](const uint8_t* from, auto byte) {
    constexpr int J = decltype(byte)::value;
    const uint8_t* a_at = from + wm * kTileBytes;
    const uint8_t* b_at = from + S::kABytes + wn * S::TN * kMx4TileBytes + lane * 16;
    i32x8 b[S::TN];
#pragma unroll
    for (int t = 0; t < S::TN; ++t) {
      const u32x4 q = *reinterpret_cast<const u32x4*>(b_at + t * kMx4TileBytes);
      b[t] = i32x8{(int)q.x, (int)q.y, (int)q.z, (int)q.w, 0, 0, 0, 0};
    }
#pragma unroll
    for (int p = kDigits - 1; p >= 0; --p) {
      const u32x4 q = *reinterpret_cast<const u32x4*>(a_at + p * kDigitBytes + lane * 16);
      const u32x2 e = *reinterpret_cast<const u32x2*>(a_at + p * kDigitBytes + 1024 + lane * 8);
      const i32x8 a = {(int)q.x, (int)q.y, (int)q.z, (int)q.w, (int)e.x, (int)e.y, 0, 0};
#pragma unroll
      for (int t = 0; t < S::TN; ++t) {
        f32x16& acc = p < 2 ? hi[t] : lo[t];
        acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b[t], acc, 2, 4, J, sa[p], J,
                                                              sb[t]);
      }
    }
  };

  issue(0, lds);
  issue(stages > 1 ? 1 : 0, lds + S::kStage);
  uint32_t next_a, next_b[S::TN];
  load_scales(0, next_a, next_b);
  uint8_t *cur = lds, *nxt = lds + S::kStage, *far = lds + 2 * S::kStage;
  auto stage = [&](int64_t st, auto byte) {
    wait_vm_lgkm0<S::kPerWave>();  // all copies but the next stage's are here
    block_barrier();
    issue(st + 2 < stages ? st + 2 : stages - 1, far);
    if (S::WK == 1 || st * S::WK + wk < kb) compute(cur + wk * S::kTileK, byte);
    uint8_t* t = cur;
    cur = nxt, nxt = far, far = t;
  };
  for (int64_t ks = 0; ks < c.ks; ++ks) {
    const int shift = S::WK == 4 ? 8 * wk : 0;  // this wave's byte to the bottom
#pragma unroll
    for (int t = 0; t < S::TN; ++t) sb[t] = static_cast<int>(next_b[t] >> shift);
#pragma unroll
    for (int p = 0; p < kDigits; ++p)  // no byte is below 23: nothing is borrowed
      sa[p] = static_cast<int>((next_a - 0x05050505u * p) >> shift);
    load_scales(ks + 1 < c.ks ? ks + 1 : ks, next_a, next_b);
    if constexpr (S::WK == 4) {
      stage(ks, std::integral_constant<int, 0>{});
    } else {
      stage(4 * ks, std::integral_constant<int, 0>{});
      if (4 * ks + 1 < kb) stage(4 * ks + 1, std::integral_constant<int, 1>{});
      if (4 * ks + 2 < kb) stage(4 * ks + 2, std::integral_constant<int, 2>{});
      if (4 * ks + 3 < kb) stage(4 * ks + 3, std::integral_constant<int, 3>{});
    }
  }

  wait_vm_lgkm0<0>();  // no copy is under way when the LDS is given back or used again
#pragma unroll
  for (int t = 0; t < S::TN; ++t) hi[t] += lo[t];
  if constexpr (S::WK > 1) {
    // The waves of one place add up over LDS, in their order.
    block_barrier();
    float* red = reinterpret_cast<float*>(lds) + (wn * S::WM + wm) * (S::TN * 1024) + lane;
    for (int q = 1; q < S::WK; ++q) {
      if (wk == q) {
#pragma unroll
        for (int t = 0; t < S::TN; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i) red[(t * 16 + i) * 64] = hi[t][i];
      }
      __syncthreads();
      if (wk == 0) {
#pragma unroll
        for (int t = 0; t < S::TN; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i) hi[t][i] += red[(t * 16 + i) * 64];
      }
      __syncthreads();
    }
    if (wk != 0) return;
  }

  // Lane: column lane % 32 of a tile, rows 8 (i / 4) + 4 (lane / 32) + i % 4.
  const int64_t m0 = (mt * S::WM + wm) * 32;
  float rstd = 1.f;
  if (c.norm_w) {
    const int64_t m = std::min(m0 + lane % 32, c.M - 1);
    float sum = 0.f;
    for (int64_t k = 0; k < c.ks; ++k) sum += sp.squares[m * c.ks + k];
    rstd = 1.0f / sqrtf(sum / static_cast<float>(c.K) + c.eps);
  }
  constexpr int kOutT = GATE ? S::TN / 2 : S::TN;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int r = 8 * (i / 4) + 4 * (lane / 32) + i % 4;
    const float f = c.norm_w ? __shfl(rstd, r, kWave) : 1.f;
    const int64_t m = m0 + r;
    if (m >= c.M) continue;
#pragma unroll
    for (int t = 0; t < kOutT; ++t) {
      const int64_t n = (nblk * S::kOutTiles + wn * kOutT + t) * 32 + lane % 32;
      if (n >= N) continue;
      float* y = c.y[seg] + m * N + n;
      const float v = hi[t][i] * f;
      if constexpr (GATE) *y = mx4_silu_mul(v, hi[kOutT + t][i] * f);
      else *y = c.res[seg] ? c.res[seg][m * N + n] + v : v;
    }
  }
}

template <class S>
int launch_gemm(const Mx4Call& c, const Space& sp, hipStream_t st) {
  Mx4Blocks bl{};
  for (int i = 0; i < c.nseg; ++i)
    bl.first[i + 1] = bl.first[i] + (mx4_row_tiles(c.N[i]) + S::kOutTiles - 1) / S::kOutTiles;
  const int64_t cols = bl.first[S::GATE ? 1 : c.nseg];
  const int64_t rows = (mx4_row_tiles(c.M) + S::WM - 1) / S::WM;
  if (cols * rows > 0x7fffffff) return EMBER_EINVAL;
  mx4_gemm_kernel<S><<<static_cast<unsigned>(cols * rows), S::kThreads, 0, st>>>(c, sp, bl, cols);
  return launch_status();
}

// Rows whose digits take a quarter of a GB, whole blocks of 256: a longer x is taken
// in pieces of that many.
int64_t piece_rows(int64_t M, int64_t kb) {
  const int64_t fit = (int64_t(1) << 28) / (kb * (kTileBytes / 32)) / 256 * 256;
  return std::min((M + 31) / 32 * 32, std::max<int64_t>(fit, 256));
}

}  // namespace

size_t ember::mx4_many_rows_bytes(int64_t M, int64_t K) {
  const int64_t kb = mx4_col_tiles(K);
  return space_bytes(piece_rows(M, kb) / 32, kb, mx4_col_blocks(K));
}

int ember::mx4_many_rows(const Mx4Call& call, bool gate, void* workspace, hipStream_t st) {
  const int64_t rows = piece_rows(call.M, call.kb), tiles = rows / 32;
  Space sp;
  sp.digits = static_cast<uint8_t*>(workspace);
  uint8_t* p = sp.digits + round256(digit_bytes(tiles, call.kb));
  sp.scales = reinterpret_cast<uint32_t*>(p);
  p += round256(static_cast<size_t>(tiles * call.ks) * 256);
  sp.squares = reinterpret_cast<float*>(p);
  for (int64_t m = 0; m < call.M; m += rows) {
    Mx4Call c = call;
    c.M = std::min(rows, call.M - m);
    c.x += m * c.K;
    for (int i = 0; i < (gate ? 1 : c.nseg); ++i) {
      c.y[i] += m * c.N[i];
      if (c.res[i]) c.res[i] += m * c.N[i];
    }
    const int64_t blocks = mx4_row_tiles(c.M) * c.ks;
    mx4_split_kernel<<<static_cast<unsigned>(std::min<int64_t>(blocks, 1 << 20)), kSplitThreads, 0,
                       st>>>(c, sp, blocks);
    int rc = launch_status();
    if (rc != EMBER_OK) return rc;
    rc = gate ? launch_gemm<Shape<4, 2, 4, 1, true>>(c, sp, st)
              : launch_gemm<Shape<4, 2, 4, 1, false>>(c, sp, st);
    if (rc != EMBER_OK) return rc;
  }
  return EMBER_OK;
}
