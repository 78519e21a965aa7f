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
#include <type_traits>

#include "common.h"
#include "quant.h"

using namespace ember;

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kMaxD = 256;  // of write and read; the attention takes 64 and 128

// ------------------------------------------------------------ write, read
// src rows [B,T,Hk,D] (blockIdx.y: keys or values) -> cache rows pos + t.
// LPR lanes per row (a power of two >= D/8), eight values a lane.  I: row
// numbers, 32-bit wherever they fit (a 64-bit division costs as much as
// quantising the lane's values).
struct WriteArgs {
  const float* src[2];
  uint32_t* codes[2];
  float* params[2];
  int64_t rows, T, Hk, S, pos;
  int words;  // D / 8
};

template <int LPR, typename I>
__global__ __launch_bounds__(kThreads) void kv4_write_kernel(WriteArgs a) {
  const int z = blockIdx.y;
  const I rows = static_cast<I>(a.rows), T = static_cast<I>(a.T), Hk = static_cast<I>(a.Hk);
  const I step = static_cast<I>(gridDim.x) * (kThreads / LPR);
  const int w = threadIdx.x % LPR;
  for (I base = static_cast<I>(blockIdx.x) * (kThreads / LPR); base < rows; base += step) {
    const I r = base + threadIdx.x / LPR;
    const bool live = r < rows && w < a.words;
    float v[8] = {};
    float lo = INFINITY, hi = -INFINITY;
    bool bad = false;
    if (live) {
      const f32x4* p = reinterpret_cast<const f32x4*>(
          a.src[z] + (static_cast<int64_t>(r) * a.words + w) * 8);
      const f32x4 x = p[0], y = p[1];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = x[e];
        v[4 + e] = y[e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        lo = fminf(lo, v[e]);
        hi = fmaxf(hi, v[e]);
        bad |= not_finite(v[e]);
      }
    }
    const QuantGrid g = quant_grid<LPR, 15>(lo, hi, bad);
    unsigned c[8];
    quant_codes<15>(g, v, c);
    if (!live) continue;
    uint32_t word = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) word |= c[e] << (4 * e);
    const I bt = r / Hk, b = bt / T;
    const int64_t row = (static_cast<int64_t>(b) * Hk + (r - bt * Hk)) * a.S + a.pos + (bt - b * T);
    a.codes[z][row * a.words + w] = word;
    if (w == 0) *reinterpret_cast<float2*>(a.params[z] + 2 * row) = float2{g.lo, g.step};
  }
}

// Cache rows [0, L) -> out [B, Hk*group, L, D]; a thread reads half a word and
// writes its four values to every head of the group, 16 bytes beside its
// neighbour's.
template <typename I>
__global__ __launch_bounds__(kThreads) void kv4_read_expanded_kernel(
    const uint32_t* __restrict__ codes, const float* __restrict__ params, float* __restrict__ out,
    int64_t n, int64_t group, int64_t L, int64_t S, int words) {
  const I stride = static_cast<I>(gridDim.x) * kThreads;
  const I per = static_cast<I>(2 * words), rows = static_cast<I>(L);
  for (I i = static_cast<I>(blockIdx.x) * kThreads + threadIdx.x; i < static_cast<I>(n);
       i += stride) {
    const I rj = i / per, c = i - rj * per, bh = rj / rows, j = rj - bh * rows;
    const int64_t row = static_cast<int64_t>(bh) * S + j;
    const uint32_t w = codes[row * words + (c >> 1)] >> (16 * (c & 1));
    const float2 p = *reinterpret_cast<const float2*>(params + 2 * row);
    f32x4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = fmaf(static_cast<float>((w >> (4 * e)) & 15u), p.y, p.x);
    f32x4* o = reinterpret_cast<f32x4*>(out) +
               (static_cast<int64_t>(bh) * group * L + j) * per + c;
    for (int64_t h = 0; h < group; ++h) o[h * L * per] = x;
  }
}

// ---------------------------------------------------------------- attention
// Query rows of a KV head: r -> (t = r / G, h = hk*G + r % G), G = H / Hk.  A
// group's rows share every code they unpack.
//
// Both products run on v_mfma_f32_16x16x32_f16 and lose nothing of the codes:
// c - 8 is exact in f16, and the fp32 operand x beside it (a query, or a weight
// times a step) is two f16 pieces, hi = f16(x) and lo = f16(x - hi), 22 bits of
// it, so a product is two MFMAs into one fp32 accumulator.  Three bf16 pieces would
// hold all 24 bits for half as many MFMAs again; the sums of D or L fp32 terms
// around them round by more than the two bits.  With lo' = lo + 8 step,
//   score_j = qmul (step_j (q' . (c_j - 8)) + lo'_j sum(q'))     (log2 units)
// where q' = q 2^(15 - ex) is a query scaled by a power of two so that its
// largest element lies in [2^14, 2^15): its low pieces then stay normal f16.
// The softmax runs against a reference per query
//   ref ~ max_j (score_j + e_j - 8),  2^e_j > step of value row j, 2^-40 |lo'_j|
// instead of max score_j, so that the weights p_j = 2^(score_j - ref) times
// their steps have their largest between 2^7 and 2^15 (ref may trail the
// maximum by kMargin): the f16 range again, whatever the rows' sizes.  A weight
// 2^-10 of the largest or more keeps its 22 bits, a smaller one is off by less
// than 2^-32 of the largest.  The offset's share in e_j bounds p_j |lo'_j| by
// 2^55 where a row's step is small beside it or 0 (the codes' errors stay below
// 2^-32 of the largest p |lo'| then).  e_j is at least -80, which bounds p_j by
// 2^95, and a sum of 2^30 of them by 2^125, where rows vanish; steps of 2^-90 still
// keep 22 bits beside such a weight, and smaller ones are off by 2^-110 a row.
// Scores reach 2^22 log2 units: the roundings of score_j + e_j - 8, in ref and
// beside it, are then at most 1/8 each, so weights times steps stay below 2^15.25,
// and f16 ends at 2^16 (scores rounded before ref is taken from them would have no
// such end, for one instruction more each).
// A query's bits depend on the rows it sees only.
//
// Fragments (lane = (g = lane / 16, i = lane % 16)):
//   S^T = K Q^T: A holds key i, dims g D/4 + 8 s + {0,4,1,5,2,6,3,7} in step s (the
//     order in which a word's codes unpack into f16 pairs), so a lane reads D/32
//     consecutive words of one row; B holds query i's same dims; C holds keys
//     4 g + e of query i.
//   O^T += V^T P^T over 32 keys: B is P as it lies in the two C tiles, keys 16 kt
//     + 4 g + e; A holds the same eight keys' codes at dim (D/16) i + t of tile t:
//     the words of eight rows, paired by 16-bit halves, then unpacked as K's are;
//     C holds dims (D/16)(4 g + e) + t of query i.
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kBlockKeys = 32;  // keys of one softmax step
constexpr int kMinExp = -80, kShift = 8;
constexpr float kLoPart = 0x1p-40f;
constexpr float kMargin = 7.f;
constexpr int kMaxSplits = 512;
constexpr int64_t kMaxRows = 1 << 30;  // of a cache: row numbers are 32-bit in the kernels

struct AttnArgs {
  const float* q;  // [B, T, H, D]
  const uint32_t* kc;
  const float* kp;
  const uint32_t* vc;
  const float* vp;
  float* o;        // [B, T, H, D]
  float* part_o;   // [B*T*H, nsplit, D]: each split's unnormalised sums
  float* part_ml;  // [B*T*H, nsplit, 2]: its reference (log2 units) and weight sum
  int64_t S;
  unsigned heads;  // B * Hk
  unsigned T, H, Hk, G;
  int L, pos;
  int nsplit, row_tiles;
  float qscale;  // scale * log2(e)
};

__device__ __forceinline__ f32x4 mfma(half8_t a, half8_t b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// The eight codes of a word, less 8, in the order 0 4 1 5 2 6 3 7, by the known
// way from small integers to floats: a code or-ed into the mantissa of 1024 makes
// 1024 + c (or + 16 c, where it lies four bits up), and what was added comes off
// again exactly.  `one` is 0x64006400 (two
// f16 1024) in a register of its own: a mask and an or of two literals would be
// two instructions.
__device__ __forceinline__ uint32_t two_1024() {
  uint32_t one = 0x64006400u;
  asm("" : "+v"(one));
  return one;
}
__device__ __forceinline__ half8_t unpack8(uint32_t w, uint32_t one) {
  const half2_t k8 = {(_Float16)1032.f, (_Float16)1032.f};
  const half2_t k72 = {(_Float16)72.f, (_Float16)72.f};
  const half2_t k16 = {(_Float16)0.0625f, (_Float16)0.0625f};
  const uint32_t v = w >> 8;
  const half2_t a = __builtin_bit_cast(half2_t, (w & 0x000f000fu) | one) - k8;
  const half2_t b = __builtin_bit_cast(half2_t, (w & 0x00f000f0u) | one) * k16 - k72;
  const half2_t c = __builtin_bit_cast(half2_t, (v & 0x000f000fu) | one) - k8;
  const half2_t d = __builtin_bit_cast(half2_t, (v & 0x00f000f0u) | one) * k16 - k72;
  return half8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Low and high 16-bit halves of two words, a's below b's.
__device__ __forceinline__ uint32_t low_halves(uint32_t a, uint32_t b) {
  return __builtin_amdgcn_perm(b, a, 0x05040100u);
}
__device__ __forceinline__ uint32_t high_halves(uint32_t a, uint32_t b) {
  return __builtin_amdgcn_perm(b, a, 0x07060302u);
}

// x as two f16 pieces (pairs convert in one instruction).
typedef float float2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void split_f16(const float (&x)[8], half8_t& hi, half8_t& lo) {
  float minus = -1.f;  // a register: x - hi is then one mixed-precision fma
  asm("" : "+s"(minus));
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const half2_t h = __builtin_convertvector((float2_t{x[e], x[e + 1]}), half2_t);
    const half2_t l = __builtin_convertvector(
        (float2_t{fmaf(static_cast<float>(h[0]), minus, x[e]),
                  fmaf(static_cast<float>(h[1]), minus, x[e + 1])}),
        half2_t);
    hi[e] = h[0];
    hi[e + 1] = h[1];
    lo[e] = l[0];
    lo[e + 1] = l[1];
  }
}

// A query row's B fragments; rows that do not exist are zero.
template <int D>
struct QRow {
  half8_t hi[D / 32], lo[D / 32];
  float mul, sum;

  // The lane's D/4 values of a row.
  static __device__ __forceinline__ void load(const float* __restrict__ row, bool live, int g,
                                              float (&x)[D / 4]) {
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      const f32x4 v = live ? reinterpret_cast<const f32x4*>(row + g * (D / 4))[c]
                           : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * c + e] = v[e];
    }
  }
  __device__ __forceinline__ void set(const float (&x)[D / 4], float qscale) {
    float amax = 0.f;
#pragma unroll
    for (int c = 0; c < D / 4; ++c) amax = fmaxf(amax, fabsf(x[c]));
    amax = max_over_rows(amax);
    const int ex = amax > 0.f && !not_finite(amax) ? __builtin_amdgcn_frexp_expf(amax) : 15;
    mul = ldexpf(qscale, ex - 15);
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < D / 32; ++k) {
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        y[e] = ldexpf(x[8 * k + (e >> 1) + 4 * (e & 1)], 15 - ex);
        s += y[e];
      }
      split_f16(y, hi[k], lo[k]);
    }
    sum = sum_over_rows(s);
  }
};

// A query's running softmax; l and olo (sum p lo') are per lane until the end.
struct Softmax {
  float ref = -INFINITY, l = 0.f, olo = 0.f;
};

// References lie as far apart as e_j do, past the range of one exp2 where a row
// of size 2^98 follows rows near 1, and the weights of these count in the sum all
// the same: beyond 2^-kFar a weight sum is scaled in two factors.  Looked for
// after the ordinary scaling, that costs 0.08 us (257 keys 5.27 -> 5.35; both
// factors always, 5.65).  The outputs' sums need no such care: what 2^-126 takes
// of them is below 2^-40 of the row that came.
constexpr float kFar = 100.f;
__device__ __forceinline__ float scale_far(float l, float d) {
  return l * __builtin_amdgcn_exp2f(fmaxf(d, -kFar)) *
         __builtin_amdgcn_exp2f(fminf(d + kFar, 0.f));
}

// The parameters of a block's keys in LDS, an array of KEYS floats each.
enum { kKStep, kKLo, kVStep, kVLo, kVExp, kParams };

// A key's or value's pair as those arrays hold it; absent rows get a step and
// an offset of 0, and their scores are masked.
template <int KEYS>
__device__ __forceinline__ void stage_params(float* par, int key, bool value, float2 p, bool in) {
  const float step = in ? p.y : 0.f;
  const float lo8 = in ? fmaf(8.f, p.y, p.x) : 0.f;
  par[(value ? kVStep : kKStep) * KEYS + key] = step;
  par[(value ? kVLo : kKLo) * KEYS + key] = lo8;
  if (value) {
    const float size = fmaxf(step, fabsf(lo8) * kLoPart);
    const int ex = size > 0.f && !not_finite(size) ? __builtin_amdgcn_frexp_expf(size) : kMinExp;
    par[kVExp * KEYS + key] = static_cast<float>((ex > kMinExp ? ex : kMinExp) - kShift);
  }
}

// One block of 32 keys for NT query tiles, in two steps; the tiles go through
// them together, so that their parameters are read once and their chains of
// arithmetic overlap.  par: the block's first key in the arrays of KEYS floats.
// vis: how many keys from this lane's first (4 g) on each tile's query sees;
// MASK: some query does not see all.
//
// score: the products s[n][kt] become scores over q.mul, in place; z[n] the
// largest of a query's scores plus exponents.
template <int KEYS, bool MASK, int D, int NT>
__device__ __forceinline__ void score(f32x4 (&s)[NT][2], const float* par, int g,
                                      const int (&vis)[NT], const QRow<D> (&q)[NT],
                                      float (&z)[NT]) {
#pragma unroll
  for (int n = 0; n < NT; ++n) z[n] = -INFINITY;
#pragma unroll
  for (int kt = 0; kt < 2; ++kt) {
    const float* p = par + 16 * kt + 4 * g;
    const f32x4 step = *reinterpret_cast<const f32x4*>(p + kKStep * KEYS);
    const f32x4 lo = *reinterpret_cast<const f32x4*>(p + kKLo * KEYS);
    const f32x4 ex = *reinterpret_cast<const f32x4*>(p + kVExp * KEYS);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[n][kt][e] = fmaf(s[n][kt][e], step[e], q[n].sum * lo[e]);
        const float t = fmaf(s[n][kt][e], q[n].mul, ex[e]);
        z[n] = fmaxf(z[n], MASK && 16 * kt + e >= vis[n] ? -INFINITY : t);
      }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) z[n] = max_over_rows(z[n]);
}

// soften: scores become weights times steps, in two f16 pieces.
template <int KEYS, bool MASK, int D, int NT>
__device__ __forceinline__ void soften(const f32x4 (&s)[NT][2], const float* par, int g,
                                       const int (&vis)[NT], const QRow<D> (&q)[NT],
                                       Softmax (&st)[NT], half8_t (&hi)[NT], half8_t (&lo8)[NT]) {
  float r[NT], x[NT][8];
  // no key seen yet: any finite reference gives weights of 0
#pragma unroll
  for (int n = 0; n < NT; ++n) r[n] = st[n].ref == -INFINITY ? 0.f : st[n].ref;
#pragma unroll
  for (int kt = 0; kt < 2; ++kt) {
    const float* p = par + 16 * kt + 4 * g;
    const f32x4 step = *reinterpret_cast<const f32x4*>(p + kVStep * KEYS);
    const f32x4 lo = *reinterpret_cast<const f32x4*>(p + kVLo * KEYS);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool hidden = MASK && 16 * kt + e >= vis[n];
        const float t = __builtin_amdgcn_exp2f(fmaf(s[n][kt][e], q[n].mul, -r[n]));
        const float w = hidden ? 0.f : t;
        st[n].l += w;
        // a row that the query does not see may hold NaN
        st[n].olo = hidden ? st[n].olo : fmaf(w, lo[e], st[n].olo);
        x[n][4 * kt + e] = hidden ? 0.f : w * step[e];
      }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) split_f16(x[n], hi[n], lo8[n]);
}

// A block's weights in pieces.  A query's reference moves, and its accumulators
// are rescaled, only where its own largest score passes that reference by more
// than kMargin (until then the weights times steps fit in f16): the other queries
// of the wave keep theirs, to the bit, or a query's rounding would depend on keys
// that only its neighbours see.  The rescaling stands outside of the two forms, or
// the compiler keeps two sets of accumulators.
// The wave goes first at the vector ALU while it is here: of two waves on a SIMD
// one is then sooner back to feed the matrix core (1024 queries over 16384
// keys 278 -> 259 us; first while it multiplies, 278).
template <int KEYS, int D, int NT, int ND>
__device__ __forceinline__ void softmax_block(bool mask, f32x4 (&s)[NT][2], const float* par,
                                              int g, const int (&vis)[NT], const QRow<D> (&q)[NT],
                                              Softmax (&st)[NT], f32x4 (&acc)[NT][ND],
                                              half8_t (&hi)[NT], half8_t (&lo)[NT]) {
  __builtin_amdgcn_s_setprio(1);
  float z[NT];
  if (mask)
    score<KEYS, true>(s, par, g, vis, q, z);
  else
    score<KEYS, false>(s, par, g, vis, q, z);
  bool past = false;
#pragma unroll
  for (int n = 0; n < NT; ++n) past |= z[n] > st[n].ref + kMargin;
  if (__any(past)) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float ref = z[n] > st[n].ref + kMargin ? z[n] : st[n].ref;
      // nothing to rescale before the first
      const float d = ref == st[n].ref || st[n].ref == -INFINITY ? 0.f : st[n].ref - ref;
      const float alpha = __builtin_amdgcn_exp2f(d);
      st[n].l = d < -kFar ? scale_far(st[n].l, d) : st[n].l * alpha;
      st[n].olo *= alpha;
      st[n].ref = ref;
#pragma unroll
      for (int t = 0; t < ND; ++t) acc[n][t] *= alpha;
    }
  }
  if (mask)
    soften<KEYS, true>(s, par, g, vis, q, st, hi, lo);
  else
    soften<KEYS, false>(s, par, g, vis, q, st, hi, lo);
  __builtin_amdgcn_s_setprio(0);
}

// The weight of a partial result with reference m and weight sum l against M.
// Rows whose scores are all NaN leave m = -inf and l = NaN.
__device__ __forceinline__ float merge_weight(float m, float l, float M) {
  return m == -INFINITY ? l : __builtin_amdgcn_exp2f(m - M);
}
// l brought from m to M where some partial result lies far from M.
__device__ __forceinline__ float merge_far(float m, float l, float M) {
  return m == -INFINITY ? l : scale_far(l, m - M);
}

// Block order: heads first, so that with 8 of them (or a multiple) a head's
// blocks share one XCD's L2; then splits; row tiles last, the longest first.
struct Item {
  int bh, split, tile;
};
__device__ __forceinline__ Item attn_item(const AttnArgs& a) {
  const unsigned x = blockIdx.x, rest = x / a.heads;
  return Item{static_cast<int>(x % a.heads), static_cast<int>(rest % a.nsplit),
              a.row_tiles - 1 - static_cast<int>(rest / a.nsplit)};
}

// Row r of a KV head: its query's number t, and its element in q and o [B,T,H,D]
// (times D).
struct RowAt {
  int t;
  int64_t row;
};
__device__ __forceinline__ RowAt attn_row(const AttnArgs& a, unsigned b, unsigned hk, unsigned r) {
  const unsigned t = r / a.G;
  return RowAt{static_cast<int>(t),
               (static_cast<int64_t>(b) * a.T + t) * a.H + hk * a.G + (r - t * a.G)};
}

// Cache row j of a (batch, KV head), clamped to the last key.
__device__ __forceinline__ int64_t clamp_row(int j, int L) { return min(j, L - 1); }

// A decode step's norms, rotations and cache write (ember_attn_kv4_qkv).
constexpr int kFoldRows = 8;       // new rows per call (T)
constexpr int kFoldGroup = 32;     // query heads per KV head
constexpr int kMaxRopePairs = 64;  // D <= 128
struct Fold {
  const float* kn;    // [B, T, Hk, D] key projection
  const float* vn;    // [B, T, Hk, D] value projection
  const float* qn_w;  // [D] QK-Norm weights, or null (no norm)
  const float* kn_w;
  uint32_t* kc;  // the cache that AttnArgs reads
  float* kp;
  uint32_t* vc;
  float* vp;
  float eps;
  float freqs[kMaxRopePairs];
};

struct NoFold {};

// A query row's D/4 values per lane (dims g D/4 ..): RMSNorm, then the
// rotation of the pairs (c, c + D/2), whose second halves lie two lane groups on.
template <int D>
__device__ __forceinline__ void fold_query(float (&x)[D / 4], const Fold& f,
                                           const float (&rot)[2][D / 2], int g) {
  if (f.qn_w) {
    float ss = 0.f;
#pragma unroll
    for (int c = 0; c < D / 4; ++c) ss = fmaf(x[c], x[c], ss);
    const float rs = 1.0f / sqrtf(sum_over_rows(ss) / static_cast<float>(D) + f.eps);
#pragma unroll
    for (int c = 0; c < D / 4; c += 4) {
      const f32x4 w = *reinterpret_cast<const f32x4*>(f.qn_w + g * (D / 4) + c);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[c + e] = x[c + e] * rs * w[e];
    }
  }
  const bool first = g < 2;
  const int c0 = (g & 1) * (D / 4);
#pragma unroll
  for (int c = 0; c < D / 4; ++c) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x[c]), __float_as_uint(x[c]),
                                                    false, false);
    const float y = __uint_as_float(first ? r[1] : r[0]);
    const float cs = rot[0][c0 + c], sn = rot[1][c0 + c];
    x[c] = first ? x[c] * cs - y * sn : y * sn + x[c] * cs;
  }
}

// The new rows p = pos + t with mine(p): keys normalised and rotated, then
// both quantised into the cache.  D/8 lanes per row; 2 T <= 16 rows fit in one
// pass of the block's THREADS / (D/8) groups.
template <int D, int THREADS, typename Mine>
__device__ __forceinline__ void fold_rows(const AttnArgs& a, const Fold& f,
                                          const float (&rot)[kFoldRows][2][D / 2], unsigned b,
                                          unsigned hk, int bh, Mine mine) {
  constexpr int LPR = D / 8;
  static_assert(THREADS / LPR >= 2 * kFoldRows, "a pass holds every new row");
  const int w = threadIdx.x % LPR, item = threadIdx.x / LPR;
  const int T = static_cast<int>(a.T);
  const bool value = item >= T, live = item < 2 * T;
  const int t = live ? (value ? item - T : item) : 0;
  const float* src = (value ? f.vn : f.kn) +
                     ((static_cast<int64_t>(b) * T + t) * a.Hk + hk) * D + 8 * w;
  float x[8], y[8];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const f32x4 v = reinterpret_cast<const f32x4*>(src)[c];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[4 * c + e] = y[4 * c + e] = v[e];
  }
  if (f.kn_w) {
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(y[e], y[e], ss);
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o, kWave);
    const float rs = 1.0f / sqrtf(ss / static_cast<float>(D) + f.eps);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = y[e] * rs * f.kn_w[8 * w + e];
  }
  const bool first = w < LPR / 2;
  const int c0 = 8 * (w % (LPR / 2));
  float lo = INFINITY, hi = -INFINITY;
  bool bad = false;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float z = __shfl_xor(y[e], LPR / 2, kWave);
    const float cs = rot[t][0][c0 + e], sn = rot[t][1][c0 + e];
    const float k = first ? y[e] * cs - z * sn : z * sn + y[e] * cs;
    x[e] = value ? x[e] : k;
    lo = fminf(lo, x[e]);
    hi = fmaxf(hi, x[e]);
    bad |= not_finite(x[e]);
  }
  const QuantGrid g = quant_grid<LPR, 15>(lo, hi, bad);
  unsigned c[8];
  quant_codes<15>(g, x, c);
  if (!live || !mine(a.pos + t)) return;
  uint32_t word = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) word |= c[e] << (4 * e);
  const int64_t row = bh * a.S + a.pos + t;
  (value ? f.vc : f.kc)[row * LPR + w] = word;
  if (w == 0)
    *reinterpret_cast<float2*>((value ? f.vp : f.kp) + 2 * row) = float2{g.lo, g.step};
}

// Few query rows: a workgroup owns up to 16 NT rows of one KV head and one key
// split, whose WAVES waves take blocks of 32 keys in turn (split by split, so
// that all splits read one stretch of the cache at a time), unpack their own
// codes and are merged through LDS.  The next block's loads (five or so per
// lane: K as fragments, V as 16-byte pieces that pass through LDS for their
// transpose, one pair of parameters) are in flight during a block.  One token at
// 130001 keys, 8 KV heads of 128: 32 us, 4.7 TB/s, the vector ALU busy 55% of them.
//
// FOLD: a decode step's raw projections.  Queries are normalised and rotated as
// they are loaded, and the workgroup whose blocks hold the new rows quantises
// them into the cache before it reads any of its blocks; no other workgroup
// of that head reads them, except those of another row tile, which write the
// same bits themselves.  Sines, the new rows and two barriers before the owner's
// first load make 2 to 3 us: 257 keys 7.5 against 5.2, 4096 keys 9.2 against 6.4,
// 130001 keys 34.5 against 31.9.
template <int D, int NT, int WAVES, bool FOLD>
__global__ __launch_bounds__(kWave * WAVES, 2) void attn_kv4_narrow(
    AttnArgs a, std::conditional_t<FOLD, Fold, NoFold> f) {
  constexpr int W = D / 8, S = D / 32, ND = D / 16, ROWS = 16 * NT;
  constexpr int kThreads = kWave * WAVES, kWaves = WAVES;
  constexpr int VS = W + 4;                       // words per V row in LDS
  constexpr int VP = kBlockKeys * W / 4 / kWave;  // 16-byte pieces of V per lane
  constexpr int kStage = kBlockKeys * VS + kParams * kBlockKeys;  // per wave, words
  constexpr int OS = D + 4;
  constexpr int kMerge = kWaves * ROWS * (OS + 2);
  constexpr int kLds = kWaves * kStage > kMerge ? kWaves * kStage : kMerge;
  __shared__ __attribute__((aligned(16))) float lds[kLds];

  const int lane = threadIdx.x & (kWave - 1), g = lane >> 4, i = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const uint32_t one = two_1024();
  const Item it = attn_item(a);
  const unsigned b = static_cast<unsigned>(it.bh) / a.Hk, hk = it.bh - b * a.Hk;
  const int R = a.G * a.T, r0 = it.tile * ROWS;
  const int nr = min(R - r0, ROWS);
  // Keys [0, jend) are seen by some row, [0, jall) by every one.
  const int jend = min(a.pos + static_cast<int>((r0 + nr - 1) / a.G) + 1, a.L);
  const int jall = min(a.pos + static_cast<int>(r0 / a.G) + 1, a.L);

  uint32_t* vbuf = reinterpret_cast<uint32_t*>(lds) + w * kStage;
  float* par = lds + w * kStage + kBlockKeys * VS;
  const uint32_t* kc = a.kc + it.bh * a.S * W;
  const uint32_t* vc = a.vc + it.bh * a.S * W;
  const float2* pp = reinterpret_cast<const float2*>(lane < 32 ? a.kp : a.vp) + it.bh * a.S;

  u32x4 kw[2], vw[VP];
  float2 pw;
  auto load = [&](int j0) {  // rows past the last key read that one again
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const int64_t row = clamp_row(j0 + 16 * kt + i, a.L);
      const uint32_t* p = kc + row * W + g * S;
      if constexpr (S == 4) {
        kw[kt] = *reinterpret_cast<const u32x4*>(p);
      } else {
        const u32x2 x = *reinterpret_cast<const u32x2*>(p);
        kw[kt] = u32x4{x[0], x[1], 0u, 0u};
      }
    }
#pragma unroll
    for (int u = 0; u < VP; ++u) {
      const int c = lane + kWave * u;
      const int64_t row = clamp_row(j0 + c / (W / 4), a.L);
      vw[u] = *reinterpret_cast<const u32x4*>(vc + row * W + 4 * (c % (W / 4)));
    }
    pw = pp[clamp_row(j0 + (lane & 31), a.L)];
  };
  const int j_first = kBlockKeys * (it.split * kWaves + w);
  const int j_step = kBlockKeys * kWaves * a.nsplit;
  __shared__ float rot[FOLD ? kFoldRows : 1][2][D / 2];  // cosines and sines
  bool owner = false;  // of new rows; the same in every wave
  if constexpr (FOLD) {
    auto split_of = [&](int j) { return j / (kBlockKeys * kWaves) % a.nsplit; };
    owner = split_of(a.pos) == it.split || split_of(a.L - 1) == it.split;
  }
  if (!owner && j_first < jend) load(j_first);
  if constexpr (FOLD) {
    for (int e = threadIdx.x; e < static_cast<int>(a.T) * (D / 2); e += kThreads) {
      const int t = e / (D / 2), c = e % (D / 2);
      float sn, cs;
      sincosf(static_cast<float>(a.pos + t) * f.freqs[c], &sn, &cs);
      rot[t][0][c] = cs;
      rot[t][1][c] = sn;
    }
    __syncthreads();
    if (owner) {
      fold_rows<D, kThreads>(a, f, rot, b, hk, it.bh, [&](int p) {
        return p / (kBlockKeys * kWaves) % a.nsplit == it.split;
      });
      __syncthreads();
      if (j_first < jend) load(j_first);
    }
  }

  QRow<D> q[NT];
  int lim[NT];  // keys j < lim are seen; rows that do not exist see all
  Softmax st[NT];
  f32x4 acc[NT][ND];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = 16 * n + i;
    const bool live = r < nr;
    const RowAt at = attn_row(a, b, hk, r0 + (live ? r : 0));
    float x[D / 4];
    QRow<D>::load(a.q + at.row * D, live, g, x);
    if constexpr (FOLD) fold_query<D>(x, f, rot[at.t], g);
    q[n].set(x, a.qscale);
    lim[n] = live ? min(a.pos + at.t + 1, a.L) : 0x7fffffff;
#pragma unroll
    for (int t2 = 0; t2 < ND; ++t2) acc[n][t2] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  for (int j0 = j_first; j0 < jend; j0 += j_step) {
    half8_t kf[2][S];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int k = 0; k < S; ++k) kf[kt][k] = unpack8(kw[kt][k], one);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int u = 0; u < VP; ++u) {
      const int c = lane + kWave * u;
      *reinterpret_cast<u32x4*>(vbuf + (c / (W / 4)) * VS + 4 * (c % (W / 4))) = vw[u];
    }
    stage_params<kBlockKeys>(par, lane & 31, lane >= 32, pw, j0 + (lane & 31) < jend);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (j0 + j_step < jend) load(j0 + j_step);

    f32x4 s[NT][2];
    int vis[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      s[n][0] = s[n][1] = f32x4{0.f, 0.f, 0.f, 0.f};
      vis[n] = lim[n] - j0 - 4 * g;
    }
#pragma unroll
    for (int k = 0; k < S; ++k) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) s[n][kt] = mfma(kf[kt][k], q[n].hi[k], s[n][kt]);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) s[n][kt] = mfma(kf[kt][k], q[n].lo[k], s[n][kt]);
    }
    half8_t ph[NT], pl[NT];
    softmax_block<kBlockKeys>(j0 + kBlockKeys > jall, s, par, g, vis, q, st, acc, ph, pl);
    // V words of this lane's eight keys, then a half (D = 128: both) of each.
    uint32_t vx[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      vx[e] = vbuf[(16 * (e >> 2) + 4 * g + (e & 3)) * VS + (D == 128 ? i : i >> 1)];
#pragma unroll
    for (int half = 0; half < ND / 4; ++half) {
      half8_t u[4], vf[4];
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const uint32_t x = vx[2 * p], y = vx[2 * p + 1];
        const bool high = D == 128 ? half == 1 : (i & 1) == 1;
        u[p] = unpack8(high ? high_halves(x, y) : low_halves(x, y), one);
      }
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          vf[t][2 * p] = u[p][2 * t];
          vf[t][2 * p + 1] = u[p][2 * t + 1];
        }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[n][4 * half + t] = mfma(vf[t], ph[n], acc[n][4 * half + t]);
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[n][4 * half + t] = mfma(vf[t], pl[n], acc[n][4 * half + t]);
      }
    }
  }

  __syncthreads();  // the stages are read no more
  float* so = lds;                        // [wave][row][OS]
  float* sm = lds + kWaves * ROWS * OS;   // [wave][row][2]
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const float l = sum_over_rows(st[n].l), olo = sum_over_rows(st[n].olo);
    const int row = w * ROWS + 16 * n + i;
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int t4 = 0; t4 < ND / 4; ++t4) {
        const f32x4 v = {acc[n][4 * t4][e], acc[n][4 * t4 + 1][e], acc[n][4 * t4 + 2][e],
                         acc[n][4 * t4 + 3][e]};
        *reinterpret_cast<f32x4*>(so + row * OS + ND * (4 * g + e) + 4 * t4) = v + olo;
      }
    if (g == 0) {
      sm[2 * row] = st[n].ref;
      sm[2 * row + 1] = l;
    }
  }
  __syncthreads();
  for (int x = threadIdx.x; x < nr * (D / 4); x += kThreads) {
    const int row = x / (D / 4), c4 = x % (D / 4);
    float M = -INFINITY;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) M = fmaxf(M, sm[2 * (v * ROWS + row)]);
    float l = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    bool far = false;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) {
      const int at = v * ROWS + row;
      const float m = sm[2 * at], e = merge_weight(m, sm[2 * at + 1], M);
      far |= m < M - kFar && m != -INFINITY;
      l += sm[2 * at + 1] * e;
      o += *reinterpret_cast<const f32x4*>(so + at * OS + 4 * c4) * e;
    }
    if (far) {
      l = 0.f;
      for (int v = 0; v < kWaves; ++v)
        l += merge_far(sm[2 * (v * ROWS + row)], sm[2 * (v * ROWS + row) + 1], M);
    }
    const int64_t orow = attn_row(a, b, hk, r0 + row).row;
    if (a.nsplit == 1) {
      *reinterpret_cast<f32x4*>(a.o + orow * D + 4 * c4) = o * (1.f / l);
    } else {
      *reinterpret_cast<f32x4*>(a.part_o + (orow * a.nsplit + it.split) * D + 4 * c4) = o;
      if (c4 == 0) {
        a.part_ml[(orow * a.nsplit + it.split) * 2] = M;
        a.part_ml[(orow * a.nsplit + it.split) * 2 + 1] = l;
      }
    }
  }
}

// Many query rows: a workgroup owns 128 rows, 32 to a wave, and one key split.
// Tiles of 64 keys are unpacked once, each wave a quarter, into two LDS buffers
// that hold them as fragments, 16 bytes per lane one after another, so that
// every wave's reads are free of bank conflicts; the next tile's codes are
// loaded during a tile and unpacked after it.  1024 queries at 16384 keys, 16
// heads of 128: 243 us, and 9 for the merge: 530 TFLOP/s in all (twice that on the
// matrix cores); bound by the vector ALU and the matrix cores, which two waves of a
// SIMD keep busy at once for about half of the time.
constexpr int kWideRows = 128;
constexpr int kTileKeys = 64;
constexpr int64_t kWideKeys = 256;  // a split's keys at least

template <int D>
__global__ __launch_bounds__(kThreads, 2) void attn_kv4_wide(AttnArgs a) {
  constexpr int W = D / 8, S = D / 32, ND = D / 16, NT = 2;
  __shared__ half8_t kfrag[2][kTileKeys / 16][S][kWave];
  __shared__ half8_t vfrag[2][kTileKeys / 32][ND][kWave];
  __shared__ __attribute__((aligned(16))) float par[2][kParams * kTileKeys];

  const int lane = threadIdx.x & (kWave - 1), g = lane >> 4, i = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const uint32_t one = two_1024();
  const Item it = attn_item(a);
  const unsigned b = static_cast<unsigned>(it.bh) / a.Hk, hk = it.bh - b * a.Hk;
  const int r0 = it.tile * kWideRows, rend = min(static_cast<int>(a.G * a.T), r0 + kWideRows);
  const int ks = kTileKeys * it.split, j_step = kTileKeys * a.nsplit;
  // How many keys row r sees.
  auto seen = [&](int r) { return min(a.pos + static_cast<int>(r / a.G) + 1, a.L); };
  const int jend = seen(rend - 1);
  // This wave's rows, and the keys that some and all of them see.
  const int wr0 = r0 + 32 * w;
  const int wend = wr0 < rend ? seen(min(wr0 + 32, rend) - 1) : 0;
  const int wall = wr0 < rend ? seen(wr0) : 0;

  const uint32_t* kc = a.kc + it.bh * a.S * W;
  const uint32_t* vc = a.vc + it.bh * a.S * W;
  const float2* pp = reinterpret_cast<const float2*>(w == 0 ? a.kp : a.vp) + it.bh * a.S;
  u32x4 kw;
  uint32_t vw[4];
  float2 pw = {0.f, 0.f};
  auto load = [&](int j0) {  // rows past the last key read that one again
    const uint32_t* p = kc + clamp_row(j0 + 16 * w + i, a.L) * W + g * S;
    if constexpr (S == 4) {
      kw = *reinterpret_cast<const u32x4*>(p);
    } else {
      const u32x2 x = *reinterpret_cast<const u32x2*>(p);
      kw = u32x4{x[0], x[1], 0u, 0u};
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      vw[e] = vc[clamp_row(j0 + 16 * w + 4 * g + e, a.L) * W + (D == 128 ? i : i >> 1)];
    if (w < 2) pw = pp[clamp_row(j0 + lane, a.L)];
  };
  auto stage = [&](int buf, int j0) {
#pragma unroll
    for (int k = 0; k < S; ++k) kfrag[buf][w][k][lane] = unpack8(kw[k], one);
#pragma unroll
    for (int half = 0; half < ND / 4; ++half) {
      const bool high = D == 128 ? half == 1 : (i & 1) == 1;
      const half8_t x = unpack8(high ? high_halves(vw[0], vw[1]) : low_halves(vw[0], vw[1]), one);
      const half8_t y = unpack8(high ? high_halves(vw[2], vw[3]) : low_halves(vw[2], vw[3]), one);
#pragma unroll
      for (int t = 0; t < 4; ++t)
        reinterpret_cast<half4_t*>(&vfrag[buf][w >> 1][4 * half + t][lane])[w & 1] =
            half4_t{x[2 * t], x[2 * t + 1], y[2 * t], y[2 * t + 1]};
    }
    if (w < 2) stage_params<kTileKeys>(par[buf], lane, w == 1, pw, j0 + lane < jend);
  };

  if (ks < jend) load(ks);
  QRow<D> q[NT];
  int lim[NT];
  Softmax st[NT];
  f32x4 acc[NT][ND];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = wr0 + 16 * n + i;
    const bool live = r < rend;
    const RowAt at = attn_row(a, b, hk, live ? r : r0);
    float x[D / 4];
    QRow<D>::load(a.q + at.row * D, live, g, x);
    q[n].set(x, a.qscale);
    lim[n] = live ? min(a.pos + at.t + 1, a.L) : 0x7fffffff;
#pragma unroll
    for (int t2 = 0; t2 < ND; ++t2) acc[n][t2] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  if (ks < jend) stage(0, ks);
  __syncthreads();

  int buf = 0;
  for (int j0 = ks; j0 < jend; j0 += j_step, buf ^= 1) {
    const bool more = j0 + j_step < jend;
    if (more) load(j0 + j_step);
#pragma unroll 1
    for (int u = 0; u < kTileKeys / 32; ++u) {
      const int jb = j0 + 32 * u;
      if (jb >= wend) break;
      f32x4 s[NT][2];
      int vis[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        s[n][0] = s[n][1] = f32x4{0.f, 0.f, 0.f, 0.f};
        vis[n] = lim[n] - jb - 4 * g;
      }
#pragma unroll
      for (int k = 0; k < S; ++k)
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          const half8_t kf = kfrag[buf][2 * u + kt][k][lane];
#pragma unroll
          for (int n = 0; n < NT; ++n) s[n][kt] = mfma(kf, q[n].hi[k], s[n][kt]);
#pragma unroll
          for (int n = 0; n < NT; ++n) s[n][kt] = mfma(kf, q[n].lo[k], s[n][kt]);
        }
      half8_t ph[NT], pl[NT];
      const float* pb = par[buf] + 32 * u;
      softmax_block<kTileKeys>(jb + 32 > wall, s, pb, g, vis, q, st, acc, ph, pl);
#pragma unroll
      for (int t = 0; t < ND; ++t) {
        const half8_t vf = vfrag[buf][u][t][lane];
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[n][t] = mfma(vf, ph[n], acc[n][t]);
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[n][t] = mfma(vf, pl[n], acc[n][t]);
      }
    }
    if (more) stage(buf ^ 1, j0 + j_step);
    __syncthreads();
  }

#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const float l = sum_over_rows(st[n].l), olo = sum_over_rows(st[n].olo);
    const int r = wr0 + 16 * n + i;
    if (r >= rend) continue;
    const int64_t orow = attn_row(a, b, hk, r).row;
    const float mul = a.nsplit == 1 ? 1.f / l : 1.f;
    float* out = a.nsplit == 1 ? a.o + orow * D
                               : a.part_o + (orow * a.nsplit + it.split) * D;
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int t4 = 0; t4 < ND / 4; ++t4) {
        const f32x4 v = {acc[n][4 * t4][e], acc[n][4 * t4 + 1][e], acc[n][4 * t4 + 2][e],
                         acc[n][4 * t4 + 3][e]};
        *reinterpret_cast<f32x4*>(out + ND * (4 * g + e) + 4 * t4) = (v + olo) * mul;
      }
    if (a.nsplit > 1 && g == 0) {
      a.part_ml[(orow * a.nsplit + it.split) * 2] = st[n].ref;
      a.part_ml[(orow * a.nsplit + it.split) * 2 + 1] = l;
    }
  }
}

// Merges a row's splits in a fixed order.  PARTS groups of D/4 lanes take every
// PARTS-th split of a row each, four at a time, and are then added in order:
// a wave per row (PARTS = 256 / D) where splits are few, a block per row (1024 / D)
// where they are many (a token at 4096 keys, 32 splits: 7.9 against 9.2 us in
// all).
template <int D, int PARTS>
__global__ __launch_bounds__(kThreads) void attn_kv4_combine(const float* __restrict__ part_o,
                                                             const float* __restrict__ part_ml,
                                                             float* __restrict__ o, int rows,
                                                             int nsplit) {
  constexpr int LANES = D / 4, PER_ROW = PARTS * LANES, RPB = kThreads / PER_ROW;
  __shared__ f32x4 s_o[kThreads];
  __shared__ float s_l[kThreads];
  __shared__ float s_m[kThreads / kWave];
  const int c4 = threadIdx.x % LANES, part = threadIdx.x / LANES % PARTS;
  const int row = blockIdx.x * RPB + threadIdx.x / PER_ROW;
  const bool live = row < rows;
  const float* ml = part_ml + static_cast<int64_t>(live ? row : 0) * nsplit * 2;
  const float* po = part_o + static_cast<int64_t>(live ? row : 0) * nsplit * D + 4 * c4;
  const int own = threadIdx.x % PER_ROW;
  // The first kAhead of a group's partial rows are on their way while the
  // weights are formed.
  constexpr int kAhead = 4;
  f32x4 x[kAhead];
#pragma unroll
  for (int u = 0; u < kAhead; ++u) {
    const int s = min(part + u * PARTS, nsplit - 1);
    x[u] = *reinterpret_cast<const f32x4*>(po + static_cast<int64_t>(s) * D);
  }
  float M = -INFINITY;
  for (int s = own; s < nsplit; s += PER_ROW) M = fmaxf(M, ml[2 * s]);
  M = wave_max(M);
  if constexpr (PER_ROW > kWave) {
    if (threadIdx.x % kWave == 0) s_m[threadIdx.x / kWave] = M;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / kWave; ++w) M = fmaxf(M, s_m[w]);
  }
  float l = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  bool far = false;
  auto add = [&](int s, f32x4 v) {
    const float m = ml[2 * s], ls = ml[2 * s + 1], e = merge_weight(m, ls, M);
    far |= m < M - kFar && m != -INFINITY;
    l += ls * e;
    acc += v * e;
  };
#pragma unroll
  for (int u = 0; u < kAhead; ++u)
    if (part + u * PARTS < nsplit) add(part + u * PARTS, x[u]);
#pragma unroll 4
  for (int s = part + kAhead * PARTS; s < nsplit; s += PARTS)
    add(s, *reinterpret_cast<const f32x4*>(po + static_cast<int64_t>(s) * D));
  if (far) {
    l = 0.f;
    for (int s = part; s < nsplit; s += PARTS) l += merge_far(ml[2 * s], ml[2 * s + 1], M);
  }
  s_o[threadIdx.x] = acc;
  s_l[threadIdx.x] = l;
  __syncthreads();
  if (part == 0 && live) {
#pragma unroll
    for (int p = 1; p < PARTS; ++p) {
      acc += s_o[threadIdx.x + p * LANES];
      l += s_l[threadIdx.x + p * LANES];
    }
    *reinterpret_cast<f32x4*>(o + static_cast<int64_t>(row) * D + 4 * c4) = acc * (1.f / l);
  }
}

// How a call is laid out, R = rows of a KV head (us for 8 KV heads of D = 128 on
// an MI355X).
//  - R <= 16, a decode step: one query tile.  Up to kOneKeys keys, or where every
//    CU has a head of its own, one workgroup of eight waves per head and no second
//    launch (257 keys 6.5 against 7.1 in splits of four waves, 512 keys 7.5 and
//    7.3, 1024 keys 10.4 and 7.3; 256 heads of 4000 keys 33.6 and 36.0); else splits.
//  - beyond, two query tiles, each workgroup for itself; or the shared tiles of
//    128 rows where there is so much to do that unpacking counts for more than
//    their barriers, kWideWork rows times keys or more (512 rows: 16384 keys 102
//    against 101, 32768 keys 176 and 161; 2048 rows: 4096 keys 85 and 91, 16384
//    keys 308 and 278).
//  - Splits: a workgroup for each CU, two where that leaves kLongKeys keys or more
//    to each (130001 keys 36 against 43 with one; 4096 keys and 128 rows, where
//    the partial results weigh more, 23 against 19), and 32 keys a wave at least.
//    A prompt whose row tiles fill the GPU once, the later ones with twice the
//    mean's keys, is split in two all the same (4096 queries and keys 235 -> 194).
constexpr int64_t kCus = 256;
constexpr int64_t kOneKeys = 512;
constexpr int64_t kWideWork = int64_t{1} << 24;
constexpr int64_t kLongKeys = 1024;
constexpr int kOneWaves = 8;
// A launch holds fewer than 2^32 threads.
constexpr int64_t kMaxBlocks = (int64_t{1} << 32) / (kWave * kOneWaves) - 1;

enum Variant { kOne, kTile, kTwoTiles, kWide };

struct Plan {
  Variant variant;
  int nsplit;
  int64_t row_tiles;
};

Plan attn_plan(int64_t B, int64_t T, int64_t H, int64_t Hk, int64_t L) {
  const int64_t R = H / Hk * T, heads = B * Hk;
  if (R <= 16 && (L <= kOneKeys || heads >= kCus)) return Plan{kOne, 1, 1};
  const bool wide = R > kFoldRows * kFoldGroup && R * L >= kWideWork;  // a decode step's never
  const Variant variant = R <= 16 ? kTile : wide ? kWide : kTwoTiles;
  const int64_t rows = variant == kTile ? 16 : variant == kTwoTiles ? 32 : kWideRows;
  const int64_t unit = variant == kWide ? kWideKeys : kBlockKeys * kWaves;
  const int64_t row_tiles = (R + rows - 1) / rows, items = heads * row_tiles;
  int64_t want = (kCus + items - 1) / items;
  if (L / want >= kLongKeys) want = (2 * kCus + items - 1) / items;
  if (wide && want == 1 && items < 4 * kCus && 2 * T >= L) want = 2;
  const int64_t units = (L + unit - 1) / unit;
  if (want > units) want = units;
  if (want > kMaxSplits) want = kMaxSplits;
  return Plan{variant, static_cast<int>(want), row_tiles};
}

// Below this a 32-bit index does not wrap when a grid's stride (at most 2^28) is
// added to it.
constexpr int64_t kIndex32 = int64_t{1} << 31;

// The tensors' and the workspace's sizes in bytes are 64-bit numbers.
bool attn_sizes_fit(int64_t B, int64_t T, int64_t H, int64_t Hk, int64_t D, int64_t S) {
  return D <= kMaxRows && fits64(B, Hk, S, D, sizeof(float)) &&
         fits64(B, T, H, D + 2, kMaxSplits, sizeof(float));
}

bool aligned8(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7u) == 0; }

}  // namespace

extern "C" int ember_kv4_write(const float* k, const float* v, uint32_t* k_codes, float* k_params,
                               uint32_t* v_codes, float* v_params, int64_t B, int64_t T,
                               int64_t Hk, int64_t D, int64_t S, int64_t pos, ember_stream_t s) {
  if (B < 0 || T < 0 || Hk < 0 || pos < 0 || T > S || pos > S - T) return EMBER_EINVAL;
  if (D < 8 || D > kMaxD || D % 8) return EMBER_EINVAL;
  if (B == 0 || T == 0 || Hk == 0) return EMBER_OK;
  if (!fits64(B, Hk, S, D, sizeof(float))) return EMBER_EINVAL;
  if (!k || !v || !k_codes || !k_params || !v_codes || !v_params) return EMBER_EINVAL;
  if (!aligned16(k) || !aligned16(v) || !aligned16(k_codes) || !aligned16(v_codes) ||
      !aligned8(k_params) || !aligned8(v_params))
    return EMBER_EALIGN;
  WriteArgs a{{k, v}, {k_codes, v_codes}, {k_params, v_params}, B * T * Hk, T, Hk, S, pos,
              static_cast<int>(D / 8)};
  auto launch = [&](auto lpr) {
    constexpr int LPR = decltype(lpr)::value;
    const dim3 grid(grid_1d(a.rows, kThreads / LPR), 2);
    if (a.rows < kIndex32)
      kv4_write_kernel<LPR, uint32_t><<<grid, kThreads, 0, as_stream(s)>>>(a);
    else
      kv4_write_kernel<LPR, int64_t><<<grid, kThreads, 0, as_stream(s)>>>(a);
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
  if (B == 0 || Hk == 0 || L == 0) return EMBER_OK;
  if (!fits64(B, Hk, S, D, sizeof(float)) || !fits64(B, Hk, L, D, group, sizeof(float)))
    return EMBER_EINVAL;
  const int64_t n = B * Hk * L * (D / 4);
  if (!codes || !params || !out) return EMBER_EINVAL;
  if (!aligned16(codes) || !aligned16(out) || !aligned8(params)) return EMBER_EALIGN;
  const unsigned grid = grid_1d(n, kThreads);
  const int words = static_cast<int>(D / 8);
  if (n < kIndex32)
    kv4_read_expanded_kernel<uint32_t>
        <<<grid, kThreads, 0, as_stream(s)>>>(codes, params, out, n, group, L, S, words);
  else
    kv4_read_expanded_kernel<int64_t>
        <<<grid, kThreads, 0, as_stream(s)>>>(codes, params, out, n, group, L, S, words);
  return launch_status();
}

extern "C" size_t ember_attn_kv4_workspace_bytes(int64_t B, int64_t T, int64_t H, int64_t Hk,
                                                 int64_t D, int64_t L) {
  if (B <= 0 || T <= 0 || H <= 0 || Hk <= 0 || H % Hk || D <= 0 || L <= 0 ||
      !attn_sizes_fit(B, T, H, Hk, D, L))
    return 0;
  const Plan p = attn_plan(B, T, H, Hk, L);
  if (p.nsplit == 1) return 0;
  return static_cast<size_t>(B * T * H) * p.nsplit * (D + 2) * sizeof(float);
}

namespace {

// Shared by ember_attn_kv4 and ember_attn_kv4_qkv (fold != null).
int run_attn(const float* q, const uint32_t* kc, const float* kp, const uint32_t* vc,
             const float* vp, float* o, int64_t B, int64_t T, int64_t H, int64_t Hk, int64_t D,
             int64_t L, int64_t pos, int64_t S, float scale, void* workspace,
             size_t workspace_bytes, const Fold* fold, hipStream_t st) {
  const Plan p = attn_plan(B, T, H, Hk, L);
  const int64_t blocks = B * Hk * p.row_tiles * p.nsplit;
  const int64_t rows = B * T * H;
  if (blocks > kMaxBlocks || rows > 0x7fffffff) return EMBER_EINVAL;
  const size_t need = ember_attn_kv4_workspace_bytes(B, T, H, Hk, D, L);
  if (need && (!workspace || workspace_bytes < need)) return EMBER_EWORKSPACE;
  if (need && !aligned16(workspace)) return EMBER_EALIGN;
  AttnArgs a{};
  a.q = q;
  a.kc = kc;
  a.kp = kp;
  a.vc = vc;
  a.vp = vp;
  a.o = o;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = need ? a.part_o + rows * p.nsplit * D : nullptr;
  a.S = S;
  a.heads = static_cast<unsigned>(B * Hk);
  a.T = static_cast<unsigned>(T);
  a.H = static_cast<unsigned>(H);
  a.Hk = static_cast<unsigned>(Hk);
  a.G = static_cast<unsigned>(H / Hk);
  a.pos = static_cast<int>(pos);
  a.L = static_cast<int>(L);
  a.nsplit = p.nsplit;
  a.row_tiles = static_cast<int>(p.row_tiles);
  a.qscale = scale * 1.4426950408889634f;
  auto launch = [&](auto d, auto folded) {
    constexpr int DD = decltype(d)::value;
    constexpr bool FOLD = decltype(folded)::value;
    std::conditional_t<FOLD, Fold, NoFold> f;
    if constexpr (FOLD) f = *fold;
    const dim3 grid(static_cast<unsigned>(blocks));
    if (p.variant == kOne)
      attn_kv4_narrow<DD, 1, kOneWaves, FOLD><<<grid, kWave * kOneWaves, 0, st>>>(a, f);
    else if (p.variant == kTile)
      attn_kv4_narrow<DD, 1, kWaves, FOLD><<<grid, kThreads, 0, st>>>(a, f);
    else if (p.variant == kTwoTiles)
      attn_kv4_narrow<DD, 2, kWaves, FOLD><<<grid, kThreads, 0, st>>>(a, f);
    else
      attn_kv4_wide<DD><<<grid, kThreads, 0, st>>>(a);
    const int rc = launch_status();
    if (rc || p.nsplit == 1) return rc;
    constexpr int kWaveParts = 256 / DD, kBlockParts = 1024 / DD;
    if (p.nsplit > 2 * kWaveParts)
      attn_kv4_combine<DD, kBlockParts><<<static_cast<unsigned>(rows), kThreads, 0, st>>>(
          a.part_o, a.part_ml, o, static_cast<int>(rows), p.nsplit);
    else
      attn_kv4_combine<DD, kWaveParts>
          <<<static_cast<unsigned>((rows + kWaves - 1) / kWaves), kThreads, 0, st>>>(
              a.part_o, a.part_ml, o, static_cast<int>(rows), p.nsplit);
    return launch_status();
  };
  using D128 = std::integral_constant<int, 128>;
  using D64 = std::integral_constant<int, 64>;
  if (fold) return D == 128 ? launch(D128{}, std::true_type{}) : launch(D64{}, std::true_type{});
  return D == 128 ? launch(D128{}, std::false_type{}) : launch(D64{}, std::false_type{});
}

}  // namespace

extern "C" int ember_attn_kv4(const float* q, const uint32_t* k_codes, const float* k_params,
                              const uint32_t* v_codes, const float* v_params, float* o, int64_t B,
                              int64_t T, int64_t H, int64_t Hk, int64_t D, int64_t L, int64_t pos,
                              int64_t S, float scale, void* workspace, size_t workspace_bytes,
                              ember_stream_t s) {
  if (B < 0 || T < 0 || H <= 0 || Hk <= 0 || H % Hk != 0 || pos < 0) return EMBER_EINVAL;
  if (D != 64 && D != 128) return EMBER_EINVAL;
  if (B == 0 || T == 0) return EMBER_OK;
  if (L < 1 || L > S || S > kMaxRows || T > kMaxRows || pos > kMaxRows) return EMBER_EINVAL;
  if (!attn_sizes_fit(B, T, H, Hk, D, S)) return EMBER_EINVAL;
  if (!q || !k_codes || !k_params || !v_codes || !v_params || !o) return EMBER_EINVAL;
  if (!aligned16(q) || !aligned16(o) || !aligned16(k_codes) || !aligned16(v_codes) ||
      !aligned8(k_params) || !aligned8(v_params))
    return EMBER_EALIGN;
  return run_attn(q, k_codes, k_params, v_codes, v_params, o, B, T, H, Hk, D, L, pos, S, scale,
                  workspace, workspace_bytes, nullptr, as_stream(s));
}

extern "C" int ember_attn_kv4_qkv(const float* q, const float* k, const float* v, int64_t B,
                                  int64_t T, int64_t H, int64_t Hk, int64_t D,
                                  const float* q_norm_w, const float* k_norm_w, float eps,
                                  const float* freqs_host, int64_t pos, uint32_t* k_codes,
                                  float* k_params, uint32_t* v_codes, float* v_params, int64_t S,
                                  float scale, float* o, void* workspace, size_t workspace_bytes,
                                  ember_stream_t s) {
  if (B < 0 || T < 0 || H <= 0 || Hk <= 0 || H % Hk != 0 || pos < 0 || !freqs_host)
    return EMBER_EINVAL;
  if ((D != 64 && D != 128) || T > kFoldRows || H / Hk > kFoldGroup)
    return EMBER_EINVAL;
  if (S > kMaxRows || T > S || pos > S - T) return EMBER_EINVAL;
  if (B == 0 || T == 0) return EMBER_OK;
  if (!attn_sizes_fit(B, T, H, Hk, D, S)) return EMBER_EINVAL;
  if (!q || !k || !v || !o || !k_codes || !k_params || !v_codes || !v_params) return EMBER_EINVAL;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o) || !aligned16(k_codes) ||
      !aligned16(v_codes) || !aligned8(k_params) || !aligned8(v_params) ||
      (q_norm_w && !aligned16(q_norm_w)) || (k_norm_w && !aligned16(k_norm_w)))
    return EMBER_EALIGN;
  Fold f{};
  f.kn = k;
  f.vn = v;
  f.qn_w = q_norm_w;
  f.kn_w = k_norm_w;
  f.kc = k_codes;
  f.kp = k_params;
  f.vc = v_codes;
  f.vp = v_params;
  f.eps = eps;
  for (int64_t i = 0; i < D / 2; ++i) f.freqs[i] = freqs_host[i];
  return run_attn(q, k_codes, k_params, v_codes, v_params, o, B, T, H, Hk, D, pos + T, pos, S,
                  scale, workspace, workspace_bytes, &f, as_stream(s));
}
