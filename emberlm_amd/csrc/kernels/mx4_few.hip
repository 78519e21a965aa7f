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
// small values beside large ones in full, lose them: the instruction drops a
// product 2^-17 of its neighbour.)  Digit p of row m is row 5 m + p of the 16
// that v_mfma_scale_f32_16x16x128_f8f6f4 takes: three rows of x an
// instruction, and every digit has a sum of its own, so that nothing small
// meets anything large before the end, where they are added from the smallest up.
//
// A wave takes 256 columns (one register of scales a lane) of 16 NT weight rows
// at a time, the waves of a workgroup every 256 columns in turn.  It asks for
// its weights first and cuts up x while they come; its part of x goes through
// its own LDS, so that no wave waits for another before the sums are joined.
// A norm's factor 1 / rms is the row's, so it waits for the end: the products
// take x times the norm's weight.
#include <algorithm>

#include "mx4_linear.h"

using namespace ember;

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kBlockCols = 256;
constexpr int kDigits = 5;
constexpr int kTokens = 3;               // rows of x in a 16-row tile
constexpr int kRowBytes = kBlockCols + 16;  // a row of digits: 16 rows at one column in 16 banks
constexpr int kTileLds = 16 * kRowBytes;
constexpr int kMaxWaves = 8;

// The largest of eight neighbouring lanes' values, in each of them.
__device__ __forceinline__ unsigned max_of_8(unsigned v) {
  v = max(v, static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0xB1, 0xf,
                                                               0xf, true)));  // lane ^ 1
  v = max(v, static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x4E, 0xf,
                                                               0xf, true)));  // lane ^ 2
  return max(v, static_cast<unsigned>(__builtin_amdgcn_update_dpp(
                    0, static_cast<int>(v), 0x141, 0xf, 0xf, true)));  // lane ^ 7
}

// LDS accesses of one wave run in order; this keeps the compiler from moving a
// lane's read over another lane's write.
__device__ __forceinline__ void wave_lds_order() { asm volatile("" ::: "memory"); }

__device__ __forceinline__ f32x4 load_x(const float* __restrict__ row, int64_t c, int64_t K,
                                        bool vec) {
  if (vec) return c < K ? *reinterpret_cast<const f32x4*>(row + c) : f32x4{0.f, 0.f, 0.f, 0.f};
  f32x4 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = c + e < K ? row[c + e] : 0.f;
  return v;
}

// One lane's operand of NT tiles of 16 weight rows by 256 columns, with the
// scales' bytes for its half of the groups in bytes 0 and 2.
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
      const int64_t k = 4 * kblk + 2 * s + (g >> 1);
      o.code[t][s] = k < kb ? *reinterpret_cast<const u32x4*>(W[t].codes +
                                                              ((nb * kb + k) * 64 + at) * 4)
                            : u32x4{0, 0, 0, 0};
    }
    o.scale[t] = W[t].scales[(nb * ks + kblk) * 64 + at] >> (8 * (g >> 1));
  }
}

template <int TT, int NT, bool GATE>
__global__ __launch_bounds__(kMaxWaves* kWave) void mx4_few_kernel(Mx4Call c, Mx4Blocks bl) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  __shared__ float sums[kMaxWaves][kMx4FewRows];  // of x^2
  constexpr int kOut = GATE ? NT / 2 : NT;        // tiles of 16 output columns
  const int lane = threadIdx.x & (kWave - 1), w = threadIdx.x / kWave;
  const int waves = blockDim.x / kWave;
  const int M = static_cast<int>(c.M);
  int64_t blk = blockIdx.x;
  const int seg = GATE ? 0 : mx4_segment(bl, c.nseg, blk);
  const int64_t N = c.N[seg], last = (N - 1) / 16;
  Mx4Weight W[NT];
  int64_t tile[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int64_t at = blk * kOut + t % kOut;
    tile[t] = at < last ? at : last;  // past the end: the last tile again, not stored
    W[t] = c.W[GATE ? t / kOut : seg];
  }
  uint8_t* mine = lds + static_cast<size_t>(w) * TT * kTileLds;
  uint8_t* scale_lds = lds + static_cast<size_t>(waves) * TT * kTileLds + w * (kMx4FewRows * 8);

  f32x4 acc[TT][NT] = {};
  float ss[TT * kTokens] = {};
  Operand<NT> next;
  if (w < c.ks) load_weights<NT>(next, W, tile, w, c.kb, c.ks);
  for (int64_t kblk = w; kblk < c.ks; kblk += waves) {
    Operand<NT> cur = next;
    const int64_t col = kblk * kBlockCols + 4 * lane;
    f32x4 xv[TT * kTokens];
#pragma unroll
    for (int m = 0; m < TT * kTokens; ++m)
      xv[m] = m < M ? load_x(c.x + m * c.K, col, c.K, c.x_vec) : f32x4{0.f, 0.f, 0.f, 0.f};
    f32x4 nw{1.f, 1.f, 1.f, 1.f};
    if (c.norm_w) nw = load_x(c.norm_w, col, c.K, c.x_vec);
    if (kblk + waves < c.ks) load_weights<NT>(next, W, tile, kblk + waves, c.kb, c.ks);
#pragma unroll
    for (int m = 0; m < TT * kTokens; ++m) {
      if (m >= M) continue;
      f32x4 t = xv[m];
      if (c.norm_w) {
        ss[m] += t.x * t.x + t.y * t.y + t.z * t.z + t.w * t.w;
        t *= nw;
      }
      unsigned top = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(t[e]) & 0x7fffffffu);
      top = max_of_8(top);
      // 255: a group that is not finite makes its row NaN; 20 and up leave room for
      // the digits' factors 2^-5 .. 2^-20
      const int byte = top >= 0x7f800000u ? 255 : max(static_cast<int>(top >> 23) - 3, 20);
#pragma unroll
      for (int e = 0; e < 4; ++e) t[e] = __builtin_ldexpf(t[e], 127 - byte);
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
      if ((lane & 7) == 0) scale_lds[m * 8 + lane / 8] = static_cast<uint8_t>(byte);
    }
    wave_lds_order();
    const int r = lane & 15, g = lane >> 4;
    // Row 15 of a tile holds nothing that is read again; nor do rows of no token.
    const int m_of = r < kTokens * kDigits ? r / kDigits : 0, p_of = r % kDigits;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int tt = 0; tt < TT; ++tt) {
        const uint8_t* row = mine + tt * kTileLds + r * kRowBytes + 128 * s + 16 * g;
        const u32x4 lo = *reinterpret_cast<const u32x4*>(row);
        const u32x4 hi = *reinterpret_cast<const u32x4*>(row + 64);
        const int sa = scale_lds[(tt * kTokens + m_of) * 8 + 4 * s + g] - 5 * p_of;
        const i32x8 a = {(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w,
                         (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const u32x4 q = cur.code[t][s];
          const i32x8 b = {(int)q.x, (int)q.y, (int)q.z, (int)q.w, 0, 0, 0, 0};
          if (s == 0)
            acc[tt][t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                a, b, acc[tt][t], 0, 4, 0, sa, 0, static_cast<int>(cur.scale[t]));
          else
            acc[tt][t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                a, b, acc[tt][t], 0, 4, 0, sa, 2, static_cast<int>(cur.scale[t]));
        }
      }
    }
    wave_lds_order();  // the next 256 columns' digits overwrite these
  }

  // Join the waves' sums: [tile of rows][tile of columns][16 rows][16 columns]
  // over the digits (a tile's 1 KB a column tile, at most 4, fits its rows).
  static_assert(NT * 1024 <= kTileLds, "the sums lie over the digits");
  float* red = reinterpret_cast<float*>(mine);
#pragma unroll
  for (int tt = 0; tt < TT; ++tt)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        red[((tt * NT + t) * 16 + 4 * (lane >> 4) + i) * 16 + (lane & 15)] = acc[tt][t][i];
  if (c.norm_w) {
#pragma unroll
    for (int m = 0; m < TT * kTokens; ++m) {
      if (m >= M) continue;
      const float v = wave_sum(ss[m]);
      if (lane == 0) sums[w][m] = v;
    }
  }
  __syncthreads();
  const float* all = reinterpret_cast<const float*>(lds);
  for (int i = threadIdx.x; i < M * kOut * 16; i += blockDim.x) {
    const int m = i / (kOut * 16), j = i % (kOut * 16);
    const int64_t n = blk * kOut * 16 + j;
    if (n >= N) continue;
    float v[GATE ? 2 : 1];
#pragma unroll
    for (int q = 0; q < (GATE ? 2 : 1); ++q) {
      const float* at = all + (((m / kTokens) * NT + q * kOut + j / 16) * 16 +
                               (m % kTokens) * kDigits) * 16 + j % 16;
      v[q] = 0.f;
#pragma unroll
      for (int p = kDigits - 1; p >= 0; --p) {
        float digit = 0.f;
        for (int u = 0; u < waves; ++u) digit += at[u * (TT * kTileLds / 4) + p * 16];
        v[q] += digit;
      }
    }
    if (c.norm_w) {
      float sum = 0.f;
      for (int u = 0; u < waves; ++u) sum += sums[u][m];
      const float rstd = 1.0f / sqrtf(sum / static_cast<float>(c.K) + c.eps);
#pragma unroll
      for (int q = 0; q < (GATE ? 2 : 1); ++q) v[q] *= rstd;
    }
    float* y = c.y[seg] + m * N + n;
    if constexpr (GATE) *y = mx4_silu_mul(v[0], v[1]);
    else *y = c.res[seg] ? c.res[seg][m * N + n] + v[0] : v[0];
  }
}

template <int TT, int NT, bool GATE>
int launch(const Mx4Call& c, hipStream_t st) {
  constexpr int kOut = GATE ? NT / 2 : NT;
  Mx4Blocks bl{};
  for (int i = 0; i < c.nseg; ++i)
    bl.first[i + 1] = bl.first[i] + (c.N[i] + 16 * kOut - 1) / (16 * kOut);
  const int64_t grid = bl.first[GATE ? 1 : c.nseg];
  const int waves = static_cast<int>(std::min<int64_t>(c.ks, kMaxWaves));
  const size_t lds = static_cast<size_t>(waves) * (TT * kTileLds + kMx4FewRows * 8);
  mx4_few_kernel<TT, NT, GATE>
      <<<static_cast<unsigned>(grid), waves * kWave, lds, st>>>(c, bl);
  return launch_status();
}

template <int NT, bool GATE>
int by_rows(const Mx4Call& c, hipStream_t st) {
  if (c.M <= kTokens) return launch<1, NT, GATE>(c, st);
  if (c.M <= 2 * kTokens) return launch<2, NT, GATE>(c, st);
  return launch<3, NT, GATE>(c, st);
}

}  // namespace

int ember::mx4_few_rows(const Mx4Call& c, bool gate, hipStream_t st) {
  if (gate) return by_rows<2, true>(c, st);
  int64_t n = 0;
  for (int i = 0; i < c.nseg; ++i) n += c.N[i];
  return n >= 32768 ? by_rows<4, false>(c, st) : by_rows<1, false>(c, st);
}
