// Inference-only ops: KV-cache writes/reads and attention with a position
// offset (reference src/ops/kv_cache.cu:50-108, include/ctd/nn/attention.h:43-97).
// None of these record autograd history.
#include <cmath>

#include "ctd/ops/attention.h"
#include "ctd/ops/decode.h"
#include "ctd/ops/kv_cache.h"
#include "ember_hip.h"
#include "op_util.h"

namespace ctd::ops {

using namespace detail;

void write_kv_inplace(Tensor& cache, const Tensor& src, int pos) {
  check_f32(cache, "write_kv", "cache");
  check_f32(src, "write_kv", "src");
  require(cache.dim() == 4 && src.dim() == 4, "write_kv: expected 4D inputs");
  const int64_t B = src.shape()[0], T = src.shape()[1], Hk = src.shape()[2], D = src.shape()[3];
  const int64_t max_seq = cache.shape()[2];
  require(cache.shape()[0] == B && cache.shape()[1] == Hk && cache.shape()[3] == D,
          "write_kv: cache / src dim mismatch");
  require(pos >= 0 && pos + T <= max_seq, "write_kv: write range out of cache bounds");
  CTD_CHECK(ember_kv_write(cfp(src), fp(cache), B, T, Hk, D, max_seq, pos, S()));
}

Tensor read_kv_expanded(const Tensor& cache, int valid_len, int group) {
  check_f32(cache, "read_kv_expanded", "cache");
  require(cache.dim() == 4, "read_kv_expanded: 4D cache required");
  const int64_t B = cache.shape()[0], Hk = cache.shape()[1], max_seq = cache.shape()[2],
                D = cache.shape()[3];
  require(valid_len >= 0 && valid_len <= max_seq, "read_kv_expanded: valid_len out of range");
  require(group > 0, "read_kv_expanded: group must be > 0");
  Tensor out = Tensor::empty({B, Hk * group, valid_len, D}, DType::kFloat32, cache.device());
  CTD_CHECK(
      ember_kv_read_expanded(cfp(cache), fp(out), B, Hk, group, valid_len, D, max_seq, S()));
  return out;
}

namespace {

uint32_t* codes_of(Tensor& t) { return static_cast<uint32_t*>(t.data_ptr()); }
const uint32_t* codes_of(const Tensor& t) { return static_cast<const uint32_t*>(t.data_ptr()); }

// One tensor of a 4-bit cache: codes [B, Hk, S, D/8] and params [B, Hk, S, 2].
void check_kv4(const Tensor& codes, const Tensor& params, const char* op, const char* what) {
  const std::string o = std::string(op) + ": " + what;
  require(codes.defined() && codes.dtype() == DType::kInt32 && codes.device().is_hip() &&
              codes.is_contiguous() && codes.dim() == 4,
          o + " codes must be a contiguous int32 [B,Hk,S,D/8] on the HIP device");
  check_f32(params, op, what);
  std::vector<int64_t> want = codes.shape();
  want.back() = 2;
  require(params.shape() == want, o + " params must be [B,Hk,S,2]");
}

// Both tensors of a cache; returns D.
int64_t check_kv4_pair(const Tensor& kc, const Tensor& kp, const Tensor& vc, const Tensor& vp,
                       const char* op) {
  check_kv4(kc, kp, op, "k cache");
  check_kv4(vc, vp, op, "v cache");
  require(kc.shape() == vc.shape(), std::string(op) + ": k and v caches differ");
  return kc.shape()[3] * 8;
}

}  // namespace

void write_kv4_inplace(Tensor& k_codes, Tensor& k_params, Tensor& v_codes, Tensor& v_params,
                       const Tensor& k, const Tensor& v, int pos) {
  const int64_t D = check_kv4_pair(k_codes, k_params, v_codes, v_params, "write_kv4");
  check_f32(k, "write_kv4", "k");
  check_f32(v, "write_kv4", "v");
  require(k.dim() == 4 && k.shape() == v.shape(), "write_kv4: expected k and v [B,T,Hk,D]");
  const int64_t B = k.shape()[0], T = k.shape()[1], Hk = k.shape()[2];
  const int64_t max_seq = k_codes.shape()[2];
  require(k_codes.shape()[0] == B && k_codes.shape()[1] == Hk && D == k.shape()[3],
          "write_kv4: cache / src dim mismatch");
  require(D <= 256, "write_kv4: head_dim must be a multiple of 8 up to 256");
  require(pos >= 0 && pos + T <= max_seq, "write_kv4: write range out of cache bounds");
  CTD_CHECK(ember_kv4_write(cfp(k), cfp(v), codes_of(k_codes), fp(k_params), codes_of(v_codes),
                            fp(v_params), B, T, Hk, D, max_seq, pos, S()));
}

Tensor read_kv4_expanded(const Tensor& codes, const Tensor& params, int valid_len, int group) {
  check_kv4(codes, params, "read_kv4_expanded", "cache");
  const int64_t B = codes.shape()[0], Hk = codes.shape()[1], max_seq = codes.shape()[2],
                D = codes.shape()[3] * 8;
  require(valid_len >= 0 && valid_len <= max_seq, "read_kv4_expanded: valid_len out of range");
  require(group > 0, "read_kv4_expanded: group must be > 0");
  Tensor out = Tensor::empty({B, Hk * group, valid_len, D}, DType::kFloat32, codes.device());
  CTD_CHECK(ember_kv4_read_expanded(codes_of(codes), cfp(params), fp(out), B, Hk, group, valid_len,
                                    D, max_seq, S()));
  return out;
}

Tensor cached_attention_kv4(const Tensor& q, const Tensor& k_codes, const Tensor& k_params,
                            const Tensor& v_codes, const Tensor& v_params, int64_t valid_len,
                            int position_start, float scale) {
  const char* op = "cached_attention_kv4";
  check_f32(q, op, "q");
  require(q.dim() == 4, "cached_attention_kv4: expected q [B,T,H,D]");
  const int64_t D = check_kv4_pair(k_codes, k_params, v_codes, v_params, op);
  const int64_t B = q.shape()[0], T = q.shape()[1], H = q.shape()[2];
  const int64_t Hk = k_codes.shape()[1], max_seq = k_codes.shape()[2];
  require(k_codes.shape()[0] == B && D == q.shape()[3],
          "cached_attention_kv4: q / cache shape mismatch");
  require(Hk > 0 && H % Hk == 0, "cached_attention_kv4: num_heads % num_kv_heads != 0");
  require(D == 64 || D == 128, "cached_attention_kv4: head_dim must be 64 or 128");
  require(valid_len >= 0 && valid_len <= max_seq, "cached_attention_kv4: valid_len out of range");
  require(position_start >= 0, "cached_attention_kv4: position_start must be >= 0");
  Tensor o = empty_like(q);
  if (B == 0 || T == 0) return o;
  require(valid_len >= 1, "cached_attention_kv4: no keys to attend to");
  const size_t wsb = ember_attn_kv4_workspace_bytes(B, T, H, Hk, D, valid_len);
  Tensor ws = wsb ? workspace(wsb) : Tensor{};
  CTD_CHECK(ember_attn_kv4(cfp(q), codes_of(k_codes), cfp(k_params), codes_of(v_codes),
                           cfp(v_params), fp(o), B, T, H, Hk, D, valid_len, position_start,
                           max_seq, scale, wsb ? ws.data_ptr() : nullptr, wsb, S()));
  return o;
}

namespace {

Tensor decode_attention(const Tensor& q, const Tensor& k, const Tensor& v, int64_t Hk,
                        int64_t L, int position_start, int64_t sb, int64_t sh, int64_t st,
                        float scale, const char* op) {
  const int64_t B = q.shape()[0], T = q.shape()[1], H = q.shape()[2], D = q.shape()[3];
  require(Hk > 0 && H % Hk == 0, std::string(op) + ": num_heads % num_kv_heads != 0");
  require(D == 64 || D == 128, std::string(op) + ": head_dim must be 64 or 128");
  require(position_start >= 0, std::string(op) + ": position_start must be >= 0");
  Tensor o = empty_like(q);
  if (B == 0 || T == 0) return o;
  require(L >= 1, std::string(op) + ": no keys to attend to");
  const size_t wsb = ember_attn_decode_workspace_bytes(B, T, H, Hk, D, L);
  Tensor ws = wsb ? workspace(wsb) : Tensor{};
  CTD_CHECK(ember_attn_decode(cfp(q), cfp(k), cfp(v), fp(o), B, T, H, Hk, D, L, position_start,
                              sb, sh, st, scale, wsb ? ws.data_ptr() : nullptr, wsb, S()));
  return o;
}

}  // namespace

Tensor cached_attention(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache,
                        int64_t valid_len, int position_start, float scale) {
  check_f32(q, "cached_attention", "q");
  check_f32(k_cache, "cached_attention", "k cache");
  check_f32(v_cache, "cached_attention", "v cache");
  require(q.dim() == 4 && k_cache.dim() == 4, "cached_attention: expected q [B,T,H,D] and "
                                              "cache [B,Hk,S,D]");
  require(k_cache.shape() == v_cache.shape(), "cached_attention: k and v caches differ");
  const int64_t Hk = k_cache.shape()[1], max_seq = k_cache.shape()[2], D = k_cache.shape()[3];
  require(k_cache.shape()[0] == q.shape()[0] && D == q.shape()[3],
          "cached_attention: q / cache shape mismatch");
  require(valid_len >= 0 && valid_len <= max_seq, "cached_attention: valid_len out of range");
  return decode_attention(q, k_cache, v_cache, Hk, valid_len, position_start, Hk * max_seq * D,
                          max_seq * D, D, scale, "cached_attention");
}

Tensor offset_attention(const Tensor& q, const Tensor& k, const Tensor& v, int position_start,
                        float scale) {
  check_f32(q, "offset_attention", "q");
  check_f32(k, "offset_attention", "k");
  check_f32(v, "offset_attention", "v");
  require(q.dim() == 4 && k.dim() == 4, "offset_attention: expected [B,T,H,D]");
  require(k.shape() == v.shape(), "offset_attention: k and v shapes differ");
  const int64_t T = k.shape()[1], Hk = k.shape()[2], D = k.shape()[3];
  require(k.shape()[0] == q.shape()[0] && T == q.shape()[1] && D == q.shape()[3],
          "offset_attention: q/k shape mismatch");
  return decode_attention(q, k, v, Hk, T, position_start, T * Hk * D, D, Hk * D, scale,
                          "offset_attention");
}

namespace {

int64_t rows_of(const Tensor& x, int64_t K, const char* op) {
  require(x.dim() >= 1 && x.shape().back() == K, std::string(op) + ": in_features mismatch");
  const int64_t M = x.numel() / K;
  require(M <= kDecodeMaxRows, std::string(op) + ": more than 8 token rows");
  return M;
}

std::vector<int64_t> with_last(const Tensor& x, int64_t n) {
  std::vector<int64_t> sh = x.shape();
  sh.back() = n;
  return sh;
}

}  // namespace

std::vector<Tensor> decode_linear(const Tensor& x, const Tensor& norm_w, float eps,
                                  const std::vector<Tensor>& weights,
                                  const std::vector<Tensor>& residuals) {
  check_f32(x, "decode_linear", "x");
  require(!weights.empty() && weights.size() <= 3, "decode_linear: 1 to 3 weights");
  require(residuals.empty() || residuals.size() == weights.size(),
          "decode_linear: one residual per weight");
  const int64_t K = weights[0].shape().at(1);
  const int64_t M = rows_of(x, K, "decode_linear");
  if (norm_w.defined()) {
    check_f32(norm_w, "decode_linear", "norm weight");
    require(norm_w.numel() == K, "decode_linear: norm weight size != in_features");
  }
  std::vector<Tensor> out;
  const float* W[3] = {};
  int64_t N[3] = {};
  float* y[3] = {};
  const float* res[3] = {};
  for (size_t i = 0; i < weights.size(); ++i) {
    check_f32(weights[i], "decode_linear", "weight");
    require(weights[i].dim() == 2 && weights[i].shape()[1] == K,
            "decode_linear: weights must be [N, K] with one K");
    N[i] = weights[i].shape()[0];
    out.push_back(Tensor::empty(with_last(x, N[i]), DType::kFloat32, x.device()));
    W[i] = cfp(weights[i]);
    y[i] = fp(out.back());
    if (!residuals.empty()) {
      check_f32(residuals[i], "decode_linear", "residual");
      require(residuals[i].shape() == out.back().shape(), "decode_linear: residual shape");
      res[i] = cfp(residuals[i]);
    }
  }
  CTD_CHECK(ember_decode_gemv(cfp(x), M, K, norm_w.defined() ? cfp(norm_w) : nullptr, eps,
                              static_cast<int>(weights.size()), W, N, y,
                              residuals.empty() ? nullptr : res, S()));
  return out;
}

Tensor decode_gate_up(const Tensor& x, const Tensor& norm_w, float eps, const Tensor& w_gate,
                      const Tensor& w_up) {
  check_f32(x, "decode_gate_up", "x");
  check_f32(w_gate, "decode_gate_up", "gate weight");
  check_f32(w_up, "decode_gate_up", "up weight");
  require(w_gate.dim() == 2 && w_gate.shape() == w_up.shape(),
          "decode_gate_up: gate and up weights differ");
  const int64_t I = w_gate.shape()[0], K = w_gate.shape()[1];
  const int64_t M = rows_of(x, K, "decode_gate_up");
  if (norm_w.defined()) {
    check_f32(norm_w, "decode_gate_up", "norm weight");
    require(norm_w.numel() == K, "decode_gate_up: norm weight size != in_features");
  }
  Tensor out = Tensor::empty(with_last(x, I), DType::kFloat32, x.device());
  CTD_CHECK(ember_decode_gateup(cfp(x), M, K, norm_w.defined() ? cfp(norm_w) : nullptr, eps,
                                cfp(w_gate), cfp(w_up), I, fp(out), S()));
  return out;
}

namespace {

// Checks shared by decode_qkv_post and the two decode_qkv_attention; returns the
// RoPE frequencies of head_dim under theta / scaling.  The caches' own types
// are checked by the caller; their rows hold row_len elements.
std::vector<float> check_qkv_post(const char* op, const Tensor& q, const Tensor& k,
                                  const Tensor& v, int64_t H, int64_t Hk, int64_t D,
                                  const Tensor& q_norm_w, const Tensor& k_norm_w, float theta,
                                  const RopeScaling& scaling, int position_start,
                                  const Tensor& k_cache, const Tensor& v_cache, int64_t row_len) {
  const std::string o(op);
  check_f32(q, op, "q");
  check_f32(k, op, "k");
  check_f32(v, op, "v");
  require(q.dim() == 3 && k.dim() == 3 && k.shape() == v.shape(),
          o + ": expected q [B,T,H*D], k/v [B,T,Hk*D]");
  const int64_t B = q.shape()[0], T = q.shape()[1];
  require(q.shape()[2] == H * D && k.shape()[0] == B && k.shape()[1] == T &&
              k.shape()[2] == Hk * D,
          o + ": q/k/v widths != heads * head_dim");
  require(k_cache.dim() == 4 && k_cache.shape() == v_cache.shape() && k_cache.shape()[0] == B &&
              k_cache.shape()[1] == Hk && k_cache.shape()[3] == row_len,
          o + ": cache / src dim mismatch");
  require(position_start >= 0 && position_start + T <= k_cache.shape()[2],
          "write_kv: write range out of cache bounds");
  for (const Tensor* w : {&q_norm_w, &k_norm_w})
    if (w->defined()) {
      check_f32(*w, op, "norm weight");
      require(w->numel() == D, o + ": QK-Norm weight size != head_dim");
    }
  std::vector<float> freqs(static_cast<size_t>(D / 2));
  CTD_CHECK(ember_rope_freqs_host(freqs.data(), static_cast<int>(D), theta, scaling.factor,
                                  scaling.low_freq_factor, scaling.high_freq_factor,
                                  scaling.original_max_pos));
  return freqs;
}

}  // namespace

Tensor decode_qkv_post(const Tensor& q, const Tensor& k, const Tensor& v, int num_heads,
                       int num_kv_heads, int head_dim, const Tensor& q_norm_w,
                       const Tensor& k_norm_w, float eps, float theta, const RopeScaling& scaling,
                       int position_start, Tensor& k_cache, Tensor& v_cache) {
  const int64_t H = num_heads, Hk = num_kv_heads, D = head_dim;
  check_f32(k_cache, "decode_qkv_post", "k cache");
  check_f32(v_cache, "decode_qkv_post", "v cache");
  const std::vector<float> freqs =
      check_qkv_post("decode_qkv_post", q, k, v, H, Hk, D, q_norm_w, k_norm_w, theta, scaling,
                     position_start, k_cache, v_cache, D);
  const int64_t B = q.shape()[0], T = q.shape()[1], max_seq = k_cache.shape()[2];
  Tensor qo = Tensor::empty({B, T, H, D}, DType::kFloat32, q.device());
  CTD_CHECK(ember_decode_qkv_post(cfp(q), cfp(k), cfp(v), B, T, H, Hk, D,
                                  q_norm_w.defined() ? cfp(q_norm_w) : nullptr,
                                  k_norm_w.defined() ? cfp(k_norm_w) : nullptr, eps, freqs.data(),
                                  position_start, fp(qo), fp(k_cache), fp(v_cache), max_seq, S()));
  return qo;
}

Tensor decode_qkv_attention(const Tensor& q, const Tensor& k, const Tensor& v, int num_heads,
                            int num_kv_heads, int head_dim, const Tensor& q_norm_w,
                            const Tensor& k_norm_w, float eps, float theta,
                            const RopeScaling& scaling, int position_start, Tensor& k_cache,
                            Tensor& v_cache, float scale) {
  const int64_t H = num_heads, Hk = num_kv_heads, D = head_dim;
  check_f32(k_cache, "decode_qkv_attention", "k cache");
  check_f32(v_cache, "decode_qkv_attention", "v cache");
  const std::vector<float> freqs =
      check_qkv_post("decode_qkv_attention", q, k, v, H, Hk, D, q_norm_w, k_norm_w, theta,
                     scaling, position_start, k_cache, v_cache, D);
  require(Hk > 0 && H % Hk == 0, "decode_qkv_attention: num_heads % num_kv_heads != 0");
  require(D == 64 || D == 128, "decode_qkv_attention: head_dim must be 64 or 128");
  const int64_t B = q.shape()[0], T = q.shape()[1], max_seq = k_cache.shape()[2];
  require(T <= kDecodeMaxRows, "decode_qkv_attention: more than 8 new rows per call");
  Tensor o = Tensor::empty({B, T, H, D}, DType::kFloat32, q.device());
  if (B == 0 || T == 0) return o;
  const size_t wsb = ember_attn_decode_workspace_bytes(B, T, H, Hk, D, position_start + T);
  Tensor ws = wsb ? workspace(wsb) : Tensor{};
  CTD_CHECK(ember_attn_decode_qkv(cfp(q), cfp(k), cfp(v), B, T, H, Hk, D,
                                  q_norm_w.defined() ? cfp(q_norm_w) : nullptr,
                                  k_norm_w.defined() ? cfp(k_norm_w) : nullptr, eps, freqs.data(),
                                  position_start, fp(k_cache), fp(v_cache), max_seq, scale, fp(o),
                                  wsb ? ws.data_ptr() : nullptr, wsb, S()));
  return o;
}

Tensor decode_qkv_attention_kv4(const Tensor& q, const Tensor& k, const Tensor& v, int num_heads,
                                int num_kv_heads, int head_dim, const Tensor& q_norm_w,
                                const Tensor& k_norm_w, float eps, float theta,
                                const RopeScaling& scaling, int position_start, Tensor& k_codes,
                                Tensor& k_params, Tensor& v_codes, Tensor& v_params, float scale) {
  const char* op = "decode_qkv_attention_kv4";
  const int64_t H = num_heads, Hk = num_kv_heads, D = head_dim;
  require(D == 64 || D == 128, "decode_qkv_attention_kv4: head_dim must be 64 or 128");
  check_kv4_pair(k_codes, k_params, v_codes, v_params, op);
  const std::vector<float> freqs =
      check_qkv_post(op, q, k, v, H, Hk, D, q_norm_w, k_norm_w, theta, scaling, position_start,
                     k_codes, v_codes, D / 8);
  require(Hk > 0 && H % Hk == 0, "decode_qkv_attention_kv4: num_heads % num_kv_heads != 0");
  require(H / Hk <= kDecodeKv4MaxGroup, "decode_qkv_attention_kv4: more than 32 heads per KV head");
  const int64_t B = q.shape()[0], T = q.shape()[1], max_seq = k_codes.shape()[2];
  require(T <= kDecodeMaxRows, "decode_qkv_attention_kv4: more than 8 new rows per call");
  Tensor o = Tensor::empty({B, T, H, D}, DType::kFloat32, q.device());
  if (B == 0 || T == 0) return o;
  const size_t wsb = ember_attn_kv4_workspace_bytes(B, T, H, Hk, D, position_start + T);
  Tensor ws = wsb ? workspace(wsb) : Tensor{};
  CTD_CHECK(ember_attn_kv4_qkv(cfp(q), cfp(k), cfp(v), B, T, H, Hk, D,
                               q_norm_w.defined() ? cfp(q_norm_w) : nullptr,
                               k_norm_w.defined() ? cfp(k_norm_w) : nullptr, eps, freqs.data(),
                               position_start, codes_of(k_codes), fp(k_params), codes_of(v_codes),
                               fp(v_params), max_seq, scale, fp(o), wsb ? ws.data_ptr() : nullptr,
                               wsb, S()));
  return o;
}

}  // namespace ctd::ops
