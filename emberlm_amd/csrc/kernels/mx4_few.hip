// Products of at most eight rows of x with weights in microscaled 4-bit
// floating point: decode steps.  Bound by the weights' bytes (17/32 a value)
// where they are many, by a launch's latency where they are few.
//
// The weights go from memory into the matrix cores as they are held (mx4.h).
// x comes to them in digits: with s the scale of a group of 32 values, |x| / s <
// 16, digit 0 is x / s rounded to a whole number, digit 1 what is left times 32
// rounded, and so on; five hold a value to 2^-24 of its group's largest, as a
// fp32 that the group shared the exponent of.  Whole numbers to 16 are exact
// in e4m3, and so are their products with the codes and the sums of these:
// eight bits each.  (Pieces that use e4m3's own exponents, which would hold
// small values beside large ones in full, lose them: within a group the instruction
// drops a product 2^-14 of its neighbour.  Groups, of unlike scales, are added up as
// in fp32.)  Digit p of row m is row 5 m + p of the 16
// that v_mfma_scale_f32_16x16x128_f8f6f4 takes: three rows of x an
// instruction, and every digit has a sum of its own, so that nothing small
// meets anything large before the end, where they are added from the smallest up.
//
// A wave takes 256 columns (one register of scales a lane) of 16 NT weight rows
// at a time, the waves of a workgroup every 256 columns in turn.  It asks for
// its x and then its weights (loads come back in order), and cuts up x while the
// weights come; its part of x goes through its own LDS, so that no wave waits for
// another before the sums are joined.  A norm's factor 1 / rms is the row's, so it
// waits for the end: the products take x times the norm's weight.
//
// In a row of calls: an LM head of 151936 x 2048 32.0 us of one row (5.2 TB/s), 41.1 of
// eight (cutting x and adding up its digits); the SwiGLU half of 2 x 6144 x 2048 4.9
// of one row and 10.1 of eight; QKV of 960 x 576 in all 3.5, of which an empty launch
// takes 2.4.
#include <algorithm>
#include <type_traits>

#include "mx4_linear.h"

using namespace ember;

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kBlockCols = 256;
constexpr int kDigits = 5;
constexpr int kTokens = 3;               // rows of x in a 16-row tile
constexpr int kRowBytes = kBlockCols + 16;  // a row of digits: 16 rows at one column in 16 banks
constexpr int kTileLds = 16 * kRowBytes;

// The largest of eight neighbouring lanes' values, in each of them.
__device__ __forceinline__ unsigned max_of_8(unsigned v) {
  v = max(v, static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0xB1, 0xf,
                                                               0xf, true)));  // lane ^ 1
  v = max(v, static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x4E, 0xf,
                                                               0xf, true)));  // lane ^ 2
  return max(v, static_cast<unsigned>(__builtin_amdgcn_update_dpp(
                    0, static_cast<int>(v), 0x141, 0xf, 0xf, true)));  // lane ^ 7
}

// The sum over a wave's lanes, in each of them, without LDS.
__device__ __forceinline__ float sum_of_64(float v) {
  const auto dpp = [](float x, auto ctrl) {
    return __uint_as_float(static_cast<unsigned>(__builtin_amdgcn_update_dpp(
        0, static_cast<int>(__float_as_uint(x)), decltype(ctrl)::value, 0xf, 0xf, true)));
  };
  v += dpp(v, std::integral_constant<int, 0xB1>{});   // lane ^ 1
  v += dpp(v, std::integral_constant<int, 0x4E>{});   // lane ^ 2
  v += dpp(v, std::integral_constant<int, 0x141>{});  // lane ^ 7
  v += dpp(v, std::integral_constant<int, 0x140>{});  // lane ^ 15
  return sum_over_rows(v);
}

// LDS accesses of one wave run in order; this keeps the compiler from moving a
// lane's read over another lane's write.
__device__ __forceinline__ void wave_lds_order() { asm volatile("" ::: "memory"); }

// One lane's operand of NT tiles of 16 weight rows by 256 columns; a word of scales
// holds the bytes for its half of the groups at bits 8 (g / 2) and 16 above.  (Shifted
// when used: a shift behind the load would wait for it.)
template <int NT>
struct Operand {
  u32x4 code[NT][2];
  uint32_t scale[NT];
};

template <int NT>
__device__ __forceinline__ void load_weights(Operand<NT>& o, const Mx4Weight (&W)[NT],
                                             const int64_t (&tile)[NT], int64_t kblk, int64_t kb,
                                             int64_t ks) {
  const int lane = threadIdx.x & (kWave - 1);
  const int n = lane & 15, g = lane >> 4;  // lane n of row group g holds columns 32 g .. + 31
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int64_t nb = tile[t] >> 1;
    const int at = 32 * (g & 1) + 16 * (tile[t] & 1) + n;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      // Past the end the last tile again: x's digits are 0 there.
      const int64_t k = std::min(4 * kblk + 2 * s + (g >> 1), kb - 1);
      o.code[t][s] = *reinterpret_cast<const u32x4*>(W[t].codes + ((nb * kb + k) * 64 + at) * 4);
    }
    o.scale[t] = W[t].scales[(nb * ks + kblk) * 64 + at];
  }
}

// What a workgroup holds in LDS.
template <int TT, int NT, int W>
struct Shared {
  __attribute__((aligned(16))) uint8_t digits[W][TT * kTileLds];  // and a wave's sums
  uint8_t scale[W][TT * kTokens * 8];
  float parts[W][NT][kMx4FewRows][16];
  float squares[W][kMx4FewRows];
};

// A lane's four columns of x's rows, and of the norm's weight: of rows and columns past
// the end the last ones, so that no load waits for a branch.
template <int TT>
struct Columns {
  f32x4 x[TT * kTokens], nw;
};
template <int TT, bool VEC>
__device__ __forceinline__ void load_columns_as(const Mx4Call& c, int64_t col, Columns<TT>& o) {
  const auto load = [&](const float* __restrict__ row) {
    if constexpr (VEC) return *reinterpret_cast<const f32x4*>(row + std::min(col, c.K - 4));
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = row[std::min(col + e, c.K - 1)];
    return v;
  };
#pragma unroll
  for (int m = 0; m < TT * kTokens; ++m) o.x[m] = load(c.x + std::min<int64_t>(m, c.M - 1) * c.K);
  o.nw = load(c.norm_w ? c.norm_w : c.x);
}
template <int TT>
__device__ __forceinline__ void load_columns(const Mx4Call& c, int64_t kblk, Columns<TT>& o) {
  const int64_t col = kblk * kBlockCols + 4 * (threadIdx.x & (kWave - 1));
  if (c.x_vec) load_columns_as<TT, true>(c, col, o);
  else load_columns_as<TT, false>(c, col, o);
}

// Cuts 256 columns of x's rows (times the norm's weight) into digits in the wave's
// part of LDS; adds up the rows' squares in ss.
template <int TT>
__device__ __forceinline__ void cut_x(const Mx4Call& c, int64_t kblk, const Columns<TT>& in,
                                      uint8_t* mine, uint8_t* scale, float (&ss)[TT * kTokens]) {
  const int lane = threadIdx.x & (kWave - 1), M = static_cast<int>(c.M);
  const int64_t col = kblk * kBlockCols + 4 * lane;
#pragma unroll
  for (int m = 0; m < TT * kTokens; ++m) {
    if (m >= M) continue;
    f32x4 t;
#pragma unroll
    for (int e = 0; e < 4; ++e) t[e] = col + e < c.K ? in.x[m][e] : 0.f;
    if (c.norm_w) {
      ss[m] += t.x * t.x + t.y * t.y + t.z * t.z + t.w * t.w;
      t *= in.nw;
    }
    unsigned top = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(t[e]) & 0x7fffffffu);
    top = max_of_8(top);
    // 255: a group that is not finite makes its row NaN; 20 and up leave room for
    // the digits' factors 2^-5 .. 2^-20
    const int byte = top >= 0x7f800000u ? 255 : max(static_cast<int>(top >> 23) - 3, 20);
#pragma unroll
    for (int e = 0; e < 4; ++e) t[e] = byte == 255 ? 0.f : __builtin_ldexpf(t[e], 127 - byte);
    uint8_t* row = mine + (m / kTokens) * kTileLds + (m % kTokens) * kDigits * kRowBytes;
#pragma unroll
    for (int p = 0; p < kDigits; ++p) {
      f32x4 d;
#pragma unroll
      for (int e = 0; e < 4; ++e) d[e] = __builtin_rintf(t[e]);
      int word = __builtin_amdgcn_cvt_pk_fp8_f32(d.x, d.y, 0, false);
      word = __builtin_amdgcn_cvt_pk_fp8_f32(d.z, d.w, word, true);
      *reinterpret_cast<int*>(row + p * kRowBytes + 4 * lane) = word;
      t = (t - d) * 32.f;
    }
    if ((lane & 7) == 0) scale[m * 8 + lane / 8] = static_cast<uint8_t>(byte);
  }
}

// A lane's operand of 128 columns (step s of the wave's 256) of a tile of x's rows.
struct Rows {
  i32x8 digits;
  int scale;
};
template <int TT, size_t ROOM>
__device__ __forceinline__ Rows read_rows(const uint8_t* mine, const uint8_t (&scale)[ROOM], int tt,
                                          int s) {
  static_assert(ROOM >= TT * kTokens * 8, "read for rows of no token too");
  const int lane = threadIdx.x & (kWave - 1), r = lane & 15, g = lane >> 4;
  // Row 15 of a tile holds nothing that is read again; nor do rows of no token, up to TT
  // kTokens of which are read.
  const int m_of = r < kTokens * kDigits ? r / kDigits : 0, p_of = r % kDigits;
  const uint8_t* row = mine + tt * kTileLds + r * kRowBytes + 128 * s + 16 * g;
  const u32x4 lo = *reinterpret_cast<const u32x4*>(row);
  const u32x4 hi = *reinterpret_cast<const u32x4*>(row + 64);
  return {i32x8{(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, (int)hi.z,
                (int)hi.w},
          scale[(tt * kTokens + m_of) * 8 + 4 * s + g] - 5 * p_of};
}

template <int TT, int NT>
__device__ __forceinline__ void multiply(f32x4 (&acc)[TT][NT], const Rows& a, int tt,
                                         const Operand<NT>& w, int s) {
  const int shift = 8 * ((threadIdx.x & (kWave - 1)) >> 5);
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int scale = static_cast<int>(w.scale[t] >> shift);
    const u32x4 q = w.code[t][s];
    const i32x8 b = {(int)q.x, (int)q.y, (int)q.z, (int)q.w, 0, 0, 0, 0};
    if (s == 0)
      acc[tt][t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
          a.digits, b, acc[tt][t], 0, 4, 0, a.scale, 0, scale);
    else
      acc[tt][t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
          a.digits, b, acc[tt][t], 0, 4, 0, a.scale, 2, scale);
  }
}

// A wave's sums to parts: its digits are added up first, the smallest first, through
// the wave's own part of LDS ([tile of rows][tile of columns][16 rows][16 columns],
// over the digits of x): lane (g, j) takes column j of row g of x and of every fourth after.
template <int TT, int NT>
__device__ __forceinline__ void add_digits(const f32x4 (&acc)[TT][NT], uint8_t* mine, int M,
                                           float (&parts)[NT][kMx4FewRows][16]) {
  static_assert(NT * 1024 <= kTileLds, "the sums lie over the digits");
  const int lane = threadIdx.x & (kWave - 1), j = lane & 15, g = lane >> 4;
  float* red = reinterpret_cast<float*>(mine);
  wave_lds_order();
#pragma unroll
  for (int tt = 0; tt < TT; ++tt)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) red[((tt * NT + t) * 16 + 4 * g + i) * 16 + j] = acc[tt][t][i];
  wave_lds_order();
#pragma unroll
  for (int i = 0; i < (TT * kTokens + 3) / 4; ++i) {
    const int m = 4 * i + g;
    if (m >= M) continue;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const float* at = red + (((m / kTokens) * NT + t) * 16 + (m % kTokens) * kDigits) * 16 + j;
      float d[kDigits];
#pragma unroll
      for (int p = 0; p < kDigits; ++p) d[p] = at[p * 16];
      parts[t][m][j] = (((d[4] + d[3]) + d[2]) + d[1]) + d[0];
    }
  }
  wave_lds_order();
}

template <int TT, int NT, int W>
__device__ __forceinline__ void note_squares(const Mx4Call& c, const float (&ss)[TT * kTokens],
                                             Shared<TT, NT, W>& sh, int w) {
  if (!c.norm_w) return;
#pragma unroll
  for (int m = 0; m < TT * kTokens; ++m) {
    if (m >= c.M) continue;
    const float v = sum_of_64(ss[m]);
    if ((threadIdx.x & (kWave - 1)) == 0) sh.squares[w][m] = v;
  }
}

// Adds up the waves' parts, in their order, and stores the block's columns.
template <int TT, int NT, int W, bool GATE>
__device__ __forceinline__ void store_block(const Mx4Call& c, const Shared<TT, NT, W>& sh,
                                            const float (&parts)[W][NT][kMx4FewRows][16], int seg,
                                            int64_t blk) {
  constexpr int kOut = GATE ? NT / 2 : NT;
  const int64_t N = c.N[seg];
  for (int i = threadIdx.x; i < static_cast<int>(c.M) * kOut * 16; i += W * kWave) {
    const int m = i / (kOut * 16), col = i % (kOut * 16);
    const int64_t n = blk * kOut * 16 + col;
    if (n >= N) continue;
    float v[GATE ? 2 : 1];
#pragma unroll
    for (int q = 0; q < (GATE ? 2 : 1); ++q) {
      v[q] = 0.f;
#pragma unroll
      for (int u = 0; u < W; ++u) v[q] += parts[u][q * kOut + col / 16][m][col % 16];
    }
    if (c.norm_w) {
      float sum = 0.f;
#pragma unroll
      for (int u = 0; u < W; ++u) sum += sh.squares[u][m];
      const float rstd = 1.0f / sqrtf(sum / static_cast<float>(c.K) + c.eps);
#pragma unroll
      for (int q = 0; q < (GATE ? 2 : 1); ++q) v[q] *= rstd;
    }
    float* y = c.y[seg] + m * N + n;
    if constexpr (GATE) *y = mx4_silu_mul(v[0], v[1]);
    else *y = c.res[seg] ? c.res[seg][m * N + n] + v[0] : v[0];
  }
}

// The tiles of 16 weight rows of block blk of segment seg.
template <int NT, bool GATE>
__device__ __forceinline__ void block_tiles(const Mx4Call& c, int seg, int64_t blk,
                                            Mx4Weight (&weight)[NT], int64_t (&tile)[NT]) {
  constexpr int kOut = GATE ? NT / 2 : NT;
  const int64_t last = (c.N[seg] - 1) / 16;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int64_t at = blk * kOut + t % kOut;
    tile[t] = at < last ? at : last;  // past the end: the last tile again, not stored
    weight[t] = c.W[GATE ? t / kOut : seg];
  }
}

// One block of columns a workgroup, any K.
template <int TT, int NT, int W, bool GATE>
__global__ __launch_bounds__(W* kWave) void mx4_few_kernel(Mx4Call c, Mx4Blocks bl) {
  __shared__ Shared<TT, NT, W> sh;
  const int w = threadIdx.x / kWave;
  int64_t blk = blockIdx.x;
  const int seg = GATE ? 0 : mx4_segment(bl, c.nseg, blk);
  Mx4Weight weight[NT];
  int64_t tile[NT];
  block_tiles<NT, GATE>(c, seg, blk, weight, tile);
  f32x4 acc[TT][NT] = {};
  float ss[TT * kTokens] = {};
  Columns<TT> x;
  Operand<NT> next;
  if (w < c.ks) {
    load_columns<TT>(c, w, x);
    load_weights<NT>(next, weight, tile, w, c.kb, c.ks);
  }
  for (int64_t kblk = w; kblk < c.ks; kblk += W) {
    wave_lds_order();  // over the digits of the 256 columns before
    cut_x<TT>(c, kblk, x, sh.digits[w], sh.scale[w], ss);
    const Operand<NT> cur = next;
    if (kblk + W < c.ks) {
      load_columns<TT>(c, kblk + W, x);
      load_weights<NT>(next, weight, tile, kblk + W, c.kb, c.ks);
    }
    wave_lds_order();
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int tt = 0; tt < TT; ++tt)
        multiply<TT, NT>(acc, read_rows<TT>(sh.digits[w], sh.scale[w], tt, s), tt, cur, s);
  }
  add_digits<TT, NT>(acc, sh.digits[w], static_cast<int>(c.M), sh.parts[w]);
  note_squares<TT, NT, W>(c, ss, sh, w);
  __syncthreads();
  store_block<TT, NT, W, GATE>(c, sh, sh.parts, seg, blk);
}

// Many blocks of columns a workgroup, K of at most W blocks of 256 columns: a wave cuts
// its part of x once, keeps it in registers, and asks for the next block's weights before
// it works on this one's.
template <int TT, int NT, int W>
__global__ __launch_bounds__(W* kWave) void mx4_stream_kernel(Mx4Call c, Mx4Blocks bl,
                                                              int64_t total) {
  __shared__ Shared<TT, NT, W> sh;
  __shared__ float other[W][NT][kMx4FewRows][16];  // every second block's parts
  const int w = threadIdx.x / kWave;
  const bool busy = w < c.ks;
  float ss[TT * kTokens] = {};
  Rows rows[2][TT];
  int64_t blk = blockIdx.x;
  int seg = mx4_segment(bl, c.nseg, blk);
  Mx4Weight weight[NT];
  int64_t tile[NT];
  block_tiles<NT, false>(c, seg, blk, weight, tile);
  Operand<NT> next;
  if (busy) {
    Columns<TT> x;
    load_columns<TT>(c, w, x);
    load_weights<NT>(next, weight, tile, w, c.kb, c.ks);
    cut_x<TT>(c, w, x, sh.digits[w], sh.scale[w], ss);
    wave_lds_order();
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int tt = 0; tt < TT; ++tt) rows[s][tt] = read_rows<TT>(sh.digits[w], sh.scale[w], tt, s);
  }
  note_squares<TT, NT, W>(c, ss, sh, w);
  bool odd = false;
  for (int64_t at = blockIdx.x; at < total; at += gridDim.x) {
    const Operand<NT> cur = next;
    const int this_seg = seg;
    const int64_t this_blk = blk;
    if (at + gridDim.x < total) {
      blk = at + gridDim.x;
      seg = mx4_segment(bl, c.nseg, blk);
      block_tiles<NT, false>(c, seg, blk, weight, tile);
      if (busy) load_weights<NT>(next, weight, tile, w, c.kb, c.ks);
    }
    f32x4 acc[TT][NT] = {};
    if (busy) {
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) multiply<TT, NT>(acc, rows[s][tt], tt, cur, s);
    }
    // The two places for the parts take turns, so that a wave may be a block ahead of one
    // that still stores.
    auto& parts = odd ? other : sh.parts;
    add_digits<TT, NT>(acc, sh.digits[w], static_cast<int>(c.M), parts[w]);
    __syncthreads();
    store_block<TT, NT, W, false>(c, sh, parts, this_seg, this_blk);
    odd = !odd;
  }
}

template <int TT, int NT, int W, bool GATE>
int launch(const Mx4Call& c, hipStream_t st) {
  constexpr int kOut = GATE ? NT / 2 : NT;
  Mx4Blocks bl{};
  for (int i = 0; i < c.nseg; ++i)
    bl.first[i + 1] = bl.first[i] + (c.N[i] + 16 * kOut - 1) / (16 * kOut);
  const int64_t total = bl.first[GATE ? 1 : c.nseg];
  if constexpr (!GATE && NT == 4) {
    constexpr int kSlots = 256 * (TT == 1 ? 2 : 1);
    if (c.ks <= W && total > kSlots) {
      mx4_stream_kernel<TT, NT, W><<<kSlots, W * kWave, 0, st>>>(c, bl, total);
      return launch_status();
    }
  }
  if (!mx4_launch_ok(total, W * kWave)) return EMBER_EINVAL;
  mx4_few_kernel<TT, NT, W, GATE><<<static_cast<unsigned>(total), W * kWave, 0, st>>>(c, bl);
  return launch_status();
}

template <int NT, int W, bool GATE>
int by_rows(const Mx4Call& c, hipStream_t st) {
  if (c.M <= kTokens) return launch<1, NT, W, GATE>(c, st);
  if (c.M <= 2 * kTokens) return launch<2, NT, W, GATE>(c, st);
  return launch<3, NT, W, GATE>(c, st);
}

template <int NT, bool GATE>
int by_waves(const Mx4Call& c, hipStream_t st) {
  if (c.ks <= 4) return by_rows<NT, 4, GATE>(c, st);
  return by_rows<NT, 8, GATE>(c, st);
}

}  // namespace

int ember::mx4_few_rows(const Mx4Call& c, bool gate, hipStream_t st) {
  int64_t tiles = 0;
  for (int i = 0; i < (gate ? 1 : c.nseg); ++i) tiles += (c.N[i] + 15) / 16;
  // Workgroups of one tile of columns as long as the GPU holds them all at once (two a CU
  // up to six rows, by registers and LDS), else of more: a workgroup cuts x for itself (8
  // rows of K = 2048 to 2 x 6144 columns: 16.9 us with 384 workgroups, 10.7 with 192).
  const int64_t slots = c.M <= 2 * kTokens ? 512 : 256;
  if (gate) return tiles <= slots ? by_waves<2, true>(c, st) : by_waves<4, true>(c, st);
  // Twice the waves for a long K where a CU has one workgroup at most (one row of K = 8192,
  // N = 2048 7.4 -> 6.7 us; with N = 8192 11.1, and 12.8 so).
  if (tiles <= 256 && c.ks >= 16 && c.M <= kTokens) return launch<1, 1, 16, false>(c, st);
  if (tiles <= slots) return by_waves<1, false>(c, st);
  return tiles <= 2 * slots ? by_waves<2, false>(c, st) : by_waves<4, false>(c, st);
}
