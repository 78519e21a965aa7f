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
// by 64 columns is, for each digit, 64 lanes of 16 bytes and then 64 of 8 (two such
// tiles, 15 KB, lie together: whole copies of 1 KB); scales lie as the weights' do.
// It also leaves each row's sums of squares (per 256 columns) from which the
// product's store takes the norm's factor.
//
// Sums: a digit's products with a group's 32 codes and their sum are exact in the
// MFMA (8 bits, whole numbers of the group's unit).  Its two groups, each of its own
// unit, are added to the running sum one after the other, as fp32 additions that first drop,
// downwards, what lies below 2^-27 of the larger one: groups 2^16 apart in a row cost
// what they cost an fp32 sum.  Digits 0 and 1 and digits 2 to 4 have sums of their own,
// so that the small ones meet no large sum before the end.
//
// Measured: 2048 rows of K = 2048 to the SwiGLU half of 2 x 6144 columns 139-145 us with
// the norm, of them 12.8 for the digits (730 TFLOP/s in all, 800 in the product); 4096 rows
// of K = 6144 to 2048 columns 163, of them 42-46 for the digits (630 and 870).  In the product
// the matrix cores are busy half of the cycles, at 1.89 GHz.  Power is part of it (on
// zeros the call is a fifth faster, a bare loop of these MFMAs 1.56 times); the rest is
// latency, LDS traffic and some 8 us of a round of tiles before its first and behind its
// last product.
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

// Workspace of R rows (whole blocks of 64) by K columns.
struct Space {
  uint8_t* digits;   // [R / 64][kb][2][kDigits][kDigitBytes]: 15 KB for 64 rows by 64 columns
  uint8_t* scales;   // [R / 32][ks][64][4]
  float* squares;    // [R][ks]
  float* parts;      // [kMostParts][2][16][64]: sums of splits of K (the small kernel's)
};
constexpr int kMostParts = 256;  // workgroups of a launch that splits K
constexpr size_t round256(size_t n) { return (n + 255) / 256 * 256; }
size_t digit_bytes(int64_t tiles, int64_t kb) { return static_cast<size_t>(tiles * kb) * kTileBytes; }
size_t space_bytes(int64_t tiles, int64_t kb, int64_t ks) {
  return round256(digit_bytes(tiles, kb)) + round256(static_cast<size_t>(tiles * ks) * 256) +
         round256(static_cast<size_t>(tiles * 32 * ks) * 4) + kMostParts * 8192;
}

// v of eight neighbouring lanes combined, in each of them: lane ^ 1, ^ 2, ^ 7.
template <typename F>
__device__ __forceinline__ unsigned over_8(unsigned v, F f) {
  v = f(v, static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, true)));
  v = f(v, static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, true)));
  return f(v, static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, true)));
}

// Four columns of a row; zeros past its end.  once: past the caches.
__device__ __forceinline__ f32x4 load_x(const float* __restrict__ row, int64_t c, int64_t K,
                                        bool vec, bool once) {
  if (vec) {
    const f32x4* at = reinterpret_cast<const f32x4*>(row + c);
    return c >= K ? f32x4{0.f, 0.f, 0.f, 0.f} : once ? __builtin_nontemporal_load(at) : *at;
  }
  f32x4 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = c + e < K ? row[c + e] : 0.f;
  return v;
}

// Eight rows by 256 columns a workgroup, a tile of 64 columns a wave: eight lanes a
// row, and four values of each of its two groups.  (32 rows a workgroup, a third
// as many of them, took 8.3 us where x is small for 4.3.)  Four lanes' 24 bits of a
// digit are three words: lane j < 3 of four takes the rest of its own and the
// beginning of its neighbour's.  Rows past M are left as they are (what is
// multiplied with them is not stored).
__global__ __launch_bounds__(kSplitThreads) void mx4_split_kernel(Mx4Call c, Space sp,
                                                                  int64_t blocks, bool once) {
  __shared__ float sums[8][4];
  const int q = threadIdx.x / kWave, r = threadIdx.x % kWave / 8, c8 = threadIdx.x % 8, j = c8 % 4;
  const int word = 3 * (c8 / 4) + j;  // of a lane's six
  for (int64_t blk = blockIdx.x; blk < blocks; blk += gridDim.x) {
    const int64_t m = blk / c.ks * 8 + r, kc = blk % c.ks;
    const int64_t row = m < c.M ? m : c.M - 1, kb = kc * 4 + q;
    f32x4 v[2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
      v[h] = load_x(c.x + row * c.K, kb * 64 + 32 * h + 4 * c8, c.K, c.x_vec, once);
    if (c.norm_w) {
      float ss = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        ss += v[h].x * v[h].x + v[h].y * v[h].y + v[h].z * v[h].z + v[h].w * v[h].w;
        v[h] *= load_x(c.norm_w, kb * 64 + 32 * h + 4 * c8, c.K, c.x_vec, false);
      }
      ss = __uint_as_float(over_8(__float_as_uint(ss), [](unsigned a, unsigned b) {
        return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
      }));
      if (c8 == 0) sums[r][q] = ss;
      __syncthreads();
      if (q == 0 && c8 == 0 && m < c.M)
        sp.squares[m * c.ks + kc] = sums[r][0] + sums[r][1] + (sums[r][2] + sums[r][3]);
      __syncthreads();
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      unsigned top = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(v[h][e]) & 0x7fffffffu);
      top = over_8(top, [](unsigned a, unsigned b) { return max(a, b); });
      // 255: a group that is not finite makes its row NaN; 23 and up leave room for
      // the digits' factors 2^-5 .. 2^-20 (and the eighths')
      const int byte = top >= 0x7f800000u ? 255 : max(static_cast<int>(top >> 23), 23);
      f32x4 t;
#pragma unroll
      for (int e = 0; e < 4; ++e) t[e] = byte == 255 ? 0.f : __builtin_ldexpf(v[h][e], 130 - byte);
      const int64_t mb = m / 32;
      const int lane = 32 * h + static_cast<int>(m % 32);
      uint8_t* tile = sp.digits + ((mb / 2 * c.kb + kb) * 2 + mb % 2) * kTileBytes;
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
        if (j < 3 && kb < c.kb && m < c.M)
          out[p * (kDigitBytes / 4)] = bits >> (8 * j) | next << (24 - 8 * j);
      }
      if (c8 == 0 && m < c.M)
        sp.scales[(mb * c.ks + kc) * 256 + 4 * lane + q] = static_cast<uint8_t>(byte);
    }
  }
}

// A row's factor 1 / rms from its squares, eight loads at a time.
__device__ __forceinline__ float row_factor(const Mx4Call& c, const Space& sp, int64_t m) {
  const float* at = sp.squares + m * c.ks;
  float sum = 0.f;
  for (int64_t k = 0; k < c.ks; k += 8) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = at[std::min(k + j, c.ks - 1)];
#pragma unroll
    for (int j = 0; j < 8; ++j) sum += k + j < c.ks ? v[j] : 0.f;
  }
  return 1.0f / sqrtf(sum / static_cast<float>(c.K) + c.eps);
}

// A workgroup's WM x WN waves take 32 rows by 32 TN columns each.  Tiles go from
// global memory to LDS without registers, a ring of four stages of a tile of K
// each, two to three ahead, one barrier a stage.
// GATE: half of a wave's TN column tiles are the gate's, half the up
// projection's at the same columns.
template <int WM_, int WN_, int TN_, bool GATE_>
struct Shape {
  static constexpr int WM = WM_, WN = WN_, TN = TN_;
  static constexpr bool GATE = GATE_;
  static constexpr int kWaves = WM * WN;
  static constexpr int kThreads = kWaves * kWave;
  static constexpr int kRowTiles = WM;                       // of x, 32 rows each
  static constexpr int kColTiles = WN * TN;                  // of the weights
  static constexpr int kOutTiles = kColTiles / (GATE ? 2 : 1);
  static constexpr int kACopies = WM / 2 * 15;               // of 1 KB, a tile of K
  static constexpr int kCopies = kACopies + kColTiles;
  static constexpr int kABytes = kACopies * 1024;
  static_assert(WM % 2 == 0, "digits lie in blocks of 64 rows");
  static constexpr int kPerWave = (kCopies + kWaves - 1) / kWaves;
  static constexpr int kStage = kCopies * 1024;
  static constexpr int kSpare = kPerWave * kWaves - kCopies;  // copies of nothing, to a room of their own
  static constexpr int kStages = 4;
  static constexpr int kLds = kStages * kStage + kSpare * 1024;
  static_assert(kLds <= 160 * 1024, "LDS");
};

template <class S>
__global__ __launch_bounds__(S::kThreads) void mx4_gemm_kernel(Mx4Call c, Space sp, Mx4Blocks bl,
                                                               unsigned col_blocks) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[S::kLds];
  constexpr bool GATE = S::GATE;
  const int lane = threadIdx.x & (kWave - 1);
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wm = w % S::WM, wn = w / S::WM;
  // Blocks go round the eight XCDs: each takes a run of tiles, columns first, whose
  // rows of digits stay in its L2.
  const unsigned xcd = blockIdx.x % 8, each = gridDim.x / 8, more = gridDim.x % 8;
  const unsigned at = xcd * each + (xcd < more ? xcd : more) + blockIdx.x / 8;
  const unsigned mt = at / col_blocks;
  int64_t nblk = at % col_blocks;
  const int seg = GATE ? 0 : mx4_segment(bl, c.nseg, nblk);
  const int64_t N = c.N[seg];
  const int64_t last_n = (N - 1) / 32, last_m = (c.M - 1) / 32;
  const int kb = static_cast<int>(c.kb);
  const int blocks = static_cast<int>(c.ks);

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

  // The wave's copies of a stage, 1 KB each: where they begin, and how far the next
  // stage is.
  const uint8_t* src[S::kPerWave];
  int stride[S::kPerWave];
#pragma unroll
  for (int i = 0; i < S::kPerWave; ++i) {
    const int in = w + i * S::kWaves < S::kCopies ? w + i * S::kWaves : 0;
    if (in < S::kACopies) {
      const int64_t mb = std::min<int64_t>(int64_t(mt) * (S::WM / 2) + in / 15, last_m / 2);
      src[i] = sp.digits + mb * kb * (2 * kTileBytes) + in % 15 * 1024;
      stride[i] = 2 * kTileBytes;
    } else {
      src[i] = reinterpret_cast<const uint8_t*>(weight(in - S::kACopies).codes) +
               col_tile(in - S::kACopies) * kb * kMx4TileBytes;
      stride[i] = kMx4TileBytes;
    }
  }
  // Copy i of stage k to LDS at `to`.
  auto copy = [&](int i, int k, uint8_t* to) {
#if defined(__HIP_DEVICE_COMPILE__)
    k = std::min(k, kb - 1);  // past the end: not read
    const int chunk = w + i * S::kWaves;
    uint8_t* at_lds = chunk < S::kCopies ? to + chunk * 1024
                                         : lds + S::kStages * S::kStage + (chunk - S::kCopies) * 1024;
    __builtin_amdgcn_global_load_lds(
        reinterpret_cast<const uint32_t*>(src[i] + int64_t(k) * stride[i] + lane * 16u),
        (__attribute__((address_space(3))) void*)at_lds, 16, 0, 0);
#endif
  };
  auto issue = [&](int stage, uint8_t* to) {
#pragma unroll
    for (int i = 0; i < S::kPerWave; ++i) copy(i, stage, to);
  };

  // Scales: one word a lane covers 256 columns.
  const uint32_t* sa_at = reinterpret_cast<const uint32_t*>(sp.scales) +
                          std::min<int64_t>(mt * S::WM + wm, last_m) * c.ks * 64 + lane;
  const uint32_t* sb_at[S::TN];
#pragma unroll
  for (int t = 0; t < S::TN; ++t)
    sb_at[t] = weight(wn * S::TN + t).scales + col_tile(wn * S::TN + t) * c.ks * 64 + lane;

  f32x16 hi[S::TN] = {}, lo[S::TN] = {};
  int sa[kDigits], sb[S::TN];
  auto load_scales = [&](int ks, uint32_t& a, uint32_t (&b)[S::TN]) {
    a = sa_at[int64_t(ks) * 64];
#pragma unroll
    for (int t = 0; t < S::TN; ++t) b[t] = sb_at[t][int64_t(ks) * 64];
  };

  auto read_a = [&](const uint8_t* from, int p) {
    const uint8_t* a_at = from + wm * kTileBytes + p * kDigitBytes;
    const u32x4 q = *reinterpret_cast<const u32x4*>(a_at + lane * 16);
    const u32x2 e = *reinterpret_cast<const u32x2*>(a_at + 1024 + lane * 8);
    return i32x8{(int)q.x, (int)q.y, (int)q.z, (int)q.w, (int)e.x, (int)e.y, 0, 0};
  };
  auto read_b = [&](const uint8_t* from, int t) {
    const u32x4 q = *reinterpret_cast<const u32x4*>(
        from + S::kABytes + (wn * S::TN + t) * kMx4TileBytes + lane * 16);
    return i32x8{(int)q.x, (int)q.y, (int)q.z, (int)q.w, 0, 0, 0, 0};
  };
  auto scales_of = [&](uint32_t a, const uint32_t (&b)[S::TN]) {
#pragma unroll
    for (int t = 0; t < S::TN; ++t) sb[t] = static_cast<int>(b[t]);
#pragma unroll
    for (int p = 0; p < kDigits; ++p)  // no byte is below 23: nothing is borrowed
      sa[p] = static_cast<int>(a - 0x05050505u * p);
  };

  uint32_t next_a, next_b[S::TN];
  load_scales(0, next_a, next_b);
  // One tile of K a stage, four stages in the ring, so that a stage's place in it
  // is its scales' byte.  The barrier lies before a stage's last digit: the
  // products of that one cover the reads of the next stage's first operands.  The
  // wave's copies of a stage are spread over five digits' products, as many as
  // the memory pipe takes without holding the wave up: the first goes out behind
  // the barrier, three stages ahead, the others in the next stage's products.
  auto spread = [&](int gap, int stage, int place) {
#pragma unroll
    for (int i = gap; i < S::kPerWave; i += kDigits) copy(i, stage, lds + place % 4 * S::kStage);
  };
  i32x8 a[2], b[2][S::TN];
  issue(0, lds);
  issue(1, lds + S::kStage);
  spread(0, 2, 2);
  wait_vm_lgkm0<S::kPerWave>();
  block_barrier();
  a[0] = read_a(lds, kDigits - 1);
#pragma unroll
  for (int t = 0; t < S::TN; ++t) b[0][t] = read_b(lds, t);
  auto stage = [&](int st, auto byte) {
    constexpr int J = decltype(byte)::value;
    const uint8_t* from = lds + J * S::kStage;
    const uint8_t* next = lds + (J + 1) % 4 * S::kStage;
    auto& bj = b[J % 2];
    auto& bn = b[(J + 1) % 2];
#pragma unroll
    for (int p = kDigits - 1; p >= 0; --p) {
      // five digits a stage: which of the two registers alternates with the stages too
      auto& ap = a[(J + kDigits - 1 - p) % 2];
      auto& an = a[(J + kDigits - p) % 2];
      if (p == 0) {
        // The next stage is here; of the one behind it all copies may be under way.
        // (Reads of this stage may be too: its place is not written before the next
        // barrier.)
        wait_vm<S::kPerWave>();
        block_barrier();
      }
#pragma unroll
      for (int t = 0; t < S::TN; ++t) {
        f32x16& acc = p < 2 ? hi[t] : lo[t];
        acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(ap, bj[t], acc, 2, 4, J, sa[p], J,
                                                              sb[t]);
        if (t > 0) continue;
        // The next digit's reads go out behind the first product, so that what the
        // next wait waits for is old by then (the compiler would put them right
        // before their own, and waits for all that are under way).
        __builtin_amdgcn_sched_barrier(0);
        if (p > 0) {
          an = read_a(from, p - 1);
        } else {
          an = read_a(next, kDigits - 1);
#pragma unroll
          for (int q = 0; q < S::TN; ++q) bn[q] = read_b(next, q);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if (p == 0) spread(0, st + 3, J + 3);
      else spread(kDigits - p, st + 2, J + 2);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  int ks = 0;
  for (; ks < kb / 4; ++ks) {
    scales_of(next_a, next_b);
    load_scales(std::min(ks + 1, blocks - 1), next_a, next_b);
    stage(4 * ks, std::integral_constant<int, 0>{});
    stage(4 * ks + 1, std::integral_constant<int, 1>{});
    stage(4 * ks + 2, std::integral_constant<int, 2>{});
    stage(4 * ks + 3, std::integral_constant<int, 3>{});
  }
  if (4 * ks < kb) {
    scales_of(next_a, next_b);
    stage(4 * ks, std::integral_constant<int, 0>{});
    if (4 * ks + 1 < kb) stage(4 * ks + 1, std::integral_constant<int, 1>{});
    if (4 * ks + 2 < kb) stage(4 * ks + 2, std::integral_constant<int, 2>{});
  }

  wait_vm_lgkm0<0>();  // no copy is under way when the LDS is given back or used again
#pragma unroll
  for (int t = 0; t < S::TN; ++t) hi[t] += lo[t];

  // Lane: column lane % 32 of a tile, rows 8 (i / 4) + 4 (lane / 32) + i % 4.
  const int64_t m0 = (int64_t(mt) * S::WM + wm) * 32;
  if (c.norm_w) {
    const float rstd = row_factor(c, sp, std::min(m0 + lane % 32, c.M - 1));
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float f = __shfl(rstd, 8 * (i / 4) + 4 * (lane / 32) + i % 4, kWave);
#pragma unroll
      for (int t = 0; t < S::TN; ++t) hi[t][i] *= f;
    }
  }
  constexpr int kOutT = GATE ? S::TN / 2 : S::TN;
  float* y = c.y[seg];
  if (const float* res = GATE ? nullptr : c.res[seg]) {
    // All loads before the first store and without branches (past the end of the last row
    // and column), or each would wait for its own and for the store before it.
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int64_t m = std::min(m0 + 8 * (i / 4) + 4 * (lane / 32) + i % 4, c.M - 1);
#pragma unroll
      for (int t = 0; t < kOutT; ++t) {
        const int64_t n = (nblk * S::kOutTiles + wn * kOutT + t) * 32 + lane % 32;
        lo[t][i] = res[m * N + std::min(n, N - 1)];
      }
    }
#pragma unroll
    for (int t = 0; t < kOutT; ++t) hi[t] += lo[t];
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int64_t m = m0 + 8 * (i / 4) + 4 * (lane / 32) + i % 4;
    if (m >= c.M) continue;
#pragma unroll
    for (int t = 0; t < kOutT; ++t) {
      const int64_t n = (nblk * S::kOutTiles + wn * kOutT + t) * 32 + lane % 32;
      if (n >= N) continue;
      if constexpr (GATE) y[m * N + n] = mx4_silu_mul(hi[t][i], hi[kOutT + t][i]);
      else y[m * N + n] = hi[t][i];
    }
  }
}

// Few tiles: a workgroup takes 32 rows by 32 columns (GATE: of the gate's and the
// up projection's both), its eight waves an eighth of K each, operands straight
// from memory to registers; the waves' sums are joined over LDS.  What bounds it is a
// CU's path to its L2 (8.7 KB a tile of K, 64 bytes a cycle), so where the tiles are few
// and K is long, several workgroups take a tile, each a part of K, and leave their sums
// in the workspace, which mx4_join_kernel adds up in their order and stores.  (8 rows of K =
// 8192, N = 2048 18.1 -> 11.4 us; joined by the last workgroup to arrive, 13.2.)
constexpr int kSmallWaves = 8;

template <bool GATE>
__global__ __launch_bounds__(kSmallWaves* kWave) void mx4_small_kernel(Mx4Call c, Space sp,
                                                                       Mx4Blocks bl,
                                                                       unsigned col_blocks,
                                                                       int splits) {
  constexpr int TN = GATE ? 2 : 1;
  __shared__ float red[kSmallWaves][TN][16][kWave];
  __shared__ float factor[32];
  const int lane = threadIdx.x & (kWave - 1);
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const unsigned tile = blockIdx.x / splits, split = blockIdx.x % splits;
  const int64_t mb = tile / col_blocks;
  int64_t nblk = tile % col_blocks;
  const int seg = GATE ? 0 : mx4_segment(bl, c.nseg, nblk);
  const int kb = static_cast<int>(c.kb);
  const uint8_t* a_at = sp.digits + (mb / 2 * kb * 2 + mb % 2) * int64_t(kTileBytes) + lane * 16;
  const uint32_t* sa_at = reinterpret_cast<const uint32_t*>(sp.scales) + mb * c.ks * 64 + lane;
  const uint32_t* b_at[TN];
  const uint32_t* sb_at[TN];
#pragma unroll
  for (int t = 0; t < TN; ++t) {
    b_at[t] = c.W[seg + t].codes + nblk * kb * (kMx4TileBytes / 4) + lane * 4;
    sb_at[t] = c.W[seg + t].scales + nblk * c.ks * 64 + lane;
  }
  struct Operands {
    u32x4 a16[kDigits], b[TN];
    u32x2 a8[kDigits];
    uint32_t sa, sb[TN];
  };
  auto load = [&](Operands& o, int k) {
    const uint8_t* a = a_at + int64_t(k) * (2 * kTileBytes);
#pragma unroll
    for (int t = 0; t < TN; ++t) {
      o.b[t] = *reinterpret_cast<const u32x4*>(b_at[t] + int64_t(k) * (kMx4TileBytes / 4));
      o.sb[t] = sb_at[t][k / 4 * 64];
    }
    o.sa = sa_at[k / 4 * 64];
#pragma unroll
    for (int p = 0; p < kDigits; ++p) {
      o.a16[p] = *reinterpret_cast<const u32x4*>(a + p * kDigitBytes);
      o.a8[p] = *reinterpret_cast<const u32x2*>(a + p * kDigitBytes + 1024 - lane * 8);
    }
  };
  f32x16 hi[TN] = {}, lo[TN] = {};
  Operands next;
  const int step = kSmallWaves * splits, first = kSmallWaves * split + w;
  if (first < kb) load(next, first);
  for (int k = first; k < kb; k += step) {
    const Operands o = next;
    if (k + step < kb) load(next, k + step);
    const int shift = k % 4 * 8;
#pragma unroll
    for (int p = kDigits - 1; p >= 0; --p) {
      const i32x8 a = {(int)o.a16[p].x, (int)o.a16[p].y, (int)o.a16[p].z, (int)o.a16[p].w,
                       (int)o.a8[p].x,  (int)o.a8[p].y,  0,               0};
#pragma unroll
      for (int t = 0; t < TN; ++t) {
        const i32x8 b = {(int)o.b[t].x, (int)o.b[t].y, (int)o.b[t].z, (int)o.b[t].w, 0, 0, 0, 0};
        f32x16& acc = p < 2 ? hi[t] : lo[t];
        acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
            a, b, acc, 2, 4, 0, static_cast<int>((o.sa >> shift) - 5 * p), 0,
            static_cast<int>(o.sb[t] >> shift));
      }
    }
  }
#pragma unroll
  for (int t = 0; t < TN; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) red[w][t][i][lane] = hi[t][i] + lo[t][i];
  if (c.norm_w && threadIdx.x < 32)
    factor[lane] = row_factor(c, sp, std::min(mb * 32 + lane, c.M - 1));
  __syncthreads();
  // Two of the 16 accumulator registers a wave; the waves' parts in their order.
  float sum[2][TN];
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int t = 0; t < TN; ++t) {
      sum[j][t] = 0.f;
#pragma unroll
      for (int u = 0; u < kSmallWaves; ++u) sum[j][t] += red[u][t][2 * w + j][lane];
    }
  if (splits > 1) {
    // [tile][split][t][16][64]
    float* parts = sp.parts + static_cast<size_t>(blockIdx.x) * (TN * 1024) + lane;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int t = 0; t < TN; ++t) parts[(t * 16 + 2 * w + j) * 64] = sum[j][t];
    return;
  }
  const int64_t N = c.N[seg], n = nblk * 32 + lane % 32;
  float extra[2] = {};
  if (const float* res = GATE ? nullptr : c.res[seg]) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int i = 2 * w + j;
      const int64_t m = std::min(mb * 32 + 8 * (i / 4) + 4 * (lane / 32) + i % 4, c.M - 1);
      extra[j] = res[m * N + std::min(n, N - 1)];
    }
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int i = 2 * w + j, r = 8 * (i / 4) + 4 * (lane / 32) + i % 4;
    const int64_t m = mb * 32 + r;
    if (m >= c.M || n >= N) continue;
    float v[TN];
#pragma unroll
    for (int t = 0; t < TN; ++t) v[t] = c.norm_w ? sum[j][t] * factor[r] : sum[j][t];
    float* y = c.y[seg] + m * N + n;
    if constexpr (GATE) *y = mx4_silu_mul(v[0], v[1]);
    else *y = extra[j] + v[0];
  }
}

// The sums of a tile's splits, a quarter of the tile a workgroup.
template <bool GATE>
__global__ __launch_bounds__(256) void mx4_join_kernel(Mx4Call c, Space sp, Mx4Blocks bl,
                                                       unsigned col_blocks, int splits) {
  constexpr int TN = GATE ? 2 : 1;
  const int lane = threadIdx.x % kWave, i = blockIdx.x % 4 * 4 + threadIdx.x / kWave;
  const unsigned tile = blockIdx.x / 4;
  const int64_t mb = tile / col_blocks;
  int64_t nblk = tile % col_blocks;
  const int seg = GATE ? 0 : mx4_segment(bl, c.nseg, nblk);
  const int64_t N = c.N[seg], n = nblk * 32 + lane % 32;
  const int64_t m = mb * 32 + 8 * (i / 4) + 4 * (lane / 32) + i % 4;
  if (m >= c.M || n >= N) return;
  float v[TN] = {};
  for (int u = 0; u < splits; ++u)
#pragma unroll
    for (int t = 0; t < TN; ++t)
      v[t] += sp.parts[((static_cast<size_t>(tile) * splits + u) * TN + t) * 1024 + i * 64 + lane];
  if (c.norm_w) {
    const float rstd = row_factor(c, sp, m);
#pragma unroll
    for (int t = 0; t < TN; ++t) v[t] *= rstd;
  }
  float* y = c.y[seg] + m * N + n;
  if constexpr (GATE) *y = mx4_silu_mul(v[0], v[1]);
  else *y = c.res[seg] ? c.res[seg][m * N + n] + v[0] : v[0];
}

// How many workgroups of the small kernel share a tile: as many as the GPU has CUs for, four
// at most, and four tiles of K a wave at least (at K = 2048 two took 10.7 us for one's 9.9).
int64_t small_splits(int64_t tiles, int64_t kb) {
  const int64_t splits = std::min<int64_t>(kMostParts / std::max<int64_t>(tiles, 1), kb / 32);
  return std::max<int64_t>(std::min<int64_t>(splits, 4), 1);
}

template <bool GATE>
int launch_small(const Mx4Call& c, const Space& sp, hipStream_t st) {
  Mx4Blocks bl{};
  for (int i = 0; i < c.nseg; ++i) bl.first[i + 1] = bl.first[i] + mx4_row_tiles(c.N[i]);
  const int64_t cols = bl.first[GATE ? 1 : c.nseg], rows = mx4_row_tiles(c.M);
  const int64_t splits = small_splits(cols * rows, c.kb);
  if (!mx4_launch_ok(cols * rows * splits, kSmallWaves * kWave)) return EMBER_EINVAL;
  mx4_small_kernel<GATE><<<static_cast<unsigned>(cols * rows * splits), kSmallWaves * kWave, 0,
                           st>>>(c, sp, bl, static_cast<unsigned>(cols),
                                 static_cast<int>(splits));
  const int rc = launch_status();
  if (rc != EMBER_OK || splits == 1) return rc;
  mx4_join_kernel<GATE><<<static_cast<unsigned>(4 * cols * rows), 256, 0, st>>>(
      c, sp, bl, static_cast<unsigned>(cols), static_cast<int>(splits));
  return launch_status();
}

template <class S>
int launch_gemm(const Mx4Call& c, const Space& sp, hipStream_t st) {
  Mx4Blocks bl{};
  for (int i = 0; i < c.nseg; ++i)
    bl.first[i + 1] = bl.first[i] + (mx4_row_tiles(c.N[i]) + S::kOutTiles - 1) / S::kOutTiles;
  const int64_t cols = bl.first[S::GATE ? 1 : c.nseg];
  const int64_t rows = (mx4_row_tiles(c.M) + S::WM - 1) / S::WM;
  if (!mx4_launch_ok(cols * rows, S::kThreads)) return EMBER_EINVAL;
  mx4_gemm_kernel<S><<<static_cast<unsigned>(cols * rows), S::kThreads, 0, st>>>(c, sp, bl,
                                                                  static_cast<unsigned>(cols));
  return launch_status();
}

// The kernel of a call, by what each is expected to take, in microseconds, from its
// count of workgroups and K (fitted on Qwen3-1.7B's and SmolLM2's products of 16 to
// 4096 rows, which it is within a quarter of):
//   tiles of 128 x 256 run at 0.72 us a tile of K where few run at once (the MFMAs'
//   latency) and 1.17 where each CU has one (power), 6 before the first and behind
//   the last;
//   tiles of 64 x 128 take 0.38 a CU, so 1.3 times as long a value, in smaller
//   rounds;
//   the small kernel's 32 x 32 take 0.105, 2.5 times as long a value, but an eighth
//   of K's latency, or less where several workgroups share a tile.
// Linear K = 2048, N = 4096 in the order small, 64 x 128, 128 x 256: 128 rows 13.8,
// 17.4, 33.7 us; 512 rows 35.1, 26.6, 37.3; 2048 rows 118, 65.9, 57.2.
enum class Kernel { kSmall, kMid, kLarge };
Kernel kernel_of(const Mx4Call& c, bool gate) {
  const int n = gate ? 1 : c.nseg, twice = gate ? 2 : 1;
  double small = 0, mid = 0, large = 0;  // workgroups
  for (int i = 0; i < n; ++i) {
    const int64_t cols = mx4_row_tiles(c.N[i]);
    small += cols;
    mid += (cols * twice + 3) / 4;
    large += (cols * twice + 7) / 8;
  }
  small *= mx4_row_tiles(c.M);
  mid *= (c.M + 63) / 64;
  large *= (c.M + 127) / 128;
  const double kb = static_cast<double>(c.kb);
  const double rounds = std::floor(large / 256), rest = large / 256 - rounds;
  const double splits = static_cast<double>(small_splits(static_cast<int64_t>(small), c.kb));
  const double t_small = 1 + 2.5 * std::ceil(small / 768) + (splits > 1 ? 2.5 : 0) +
                         0.105 * twice * kb * std::max(small / 256, 1.0 / splits);
  const double t_mid = 5 + 0.38 * kb * std::ceil(mid / 256);
  const double t_large = rounds * (6 + 1.17 * kb) + (rest > 0 ? 6 + (0.72 + 0.45 * rest) * kb : 0);
  if (t_small <= t_mid && t_small <= t_large) return Kernel::kSmall;
  return t_mid <= t_large ? Kernel::kMid : Kernel::kLarge;
}

// An x of more values than these is read past the caches, which its digits then have to
// themselves until the product reads them (4096 x 6144, 100 MB: 195 -> 178 us when it was built); a
// smaller one may still be there when the product's residual or the caller wants it (2048 x
// 6144: 102 us, read past them 105).
constexpr int64_t kKeep = int64_t(1) << 24;

// Rows whose digits take a quarter of a GB, whole blocks of 256: a longer x is taken
// in pieces of that many.
int64_t piece_rows(int64_t M, int64_t kb) {
  const int64_t fit = (int64_t(1) << 28) / (kb * (kTileBytes / 32)) / 256 * 256;
  return std::min((M + 63) / 64 * 64, std::max<int64_t>(fit, 256));
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
  sp.scales = p;
  p += round256(static_cast<size_t>(tiles * call.ks) * 256);
  sp.squares = reinterpret_cast<float*>(p);
  p += round256(static_cast<size_t>(tiles * 32 * call.ks) * 4);
  sp.parts = reinterpret_cast<float*>(p);
  for (int64_t m = 0; m < call.M; m += rows) {
    Mx4Call c = call;
    c.M = std::min(rows, call.M - m);
    c.x += m * c.K;
    for (int i = 0; i < (gate ? 1 : c.nseg); ++i) {
      c.y[i] += m * c.N[i];
      if (c.res[i]) c.res[i] += m * c.N[i];
    }
    const int64_t blocks = (c.M + 7) / 8 * c.ks;
    mx4_split_kernel<<<static_cast<unsigned>(std::min<int64_t>(blocks, 1 << 20)), kSplitThreads, 0,
                       st>>>(c, sp, blocks, c.M * c.K > kKeep);
    int rc = launch_status();
    if (rc != EMBER_OK) return rc;
    switch (kernel_of(c, gate)) {
      case Kernel::kSmall:
        rc = gate ? launch_small<true>(c, sp, st) : launch_small<false>(c, sp, st);
        break;
      case Kernel::kMid:
        rc = gate ? launch_gemm<Shape<2, 2, 2, true>>(c, sp, st)
                  : launch_gemm<Shape<2, 2, 2, false>>(c, sp, st);
        break;
      default:
        rc = gate ? launch_gemm<Shape<4, 2, 4, true>>(c, sp, st)
                  : launch_gemm<Shape<4, 2, 4, false>>(c, sp, st);
    }
    if (rc != EMBER_OK) return rc;
  }
  return EMBER_OK;
}
