// Rows held in 8 bits, weights held in 4.  None of these record autograd history.
#include "ctd/ops/quant.h"

#include "ember_hip.h"
#include "op_util.h"

namespace ctd::ops {

using namespace detail;

namespace {

struct Rows {
  int64_t rows, H;
};

Rows rows_of(const std::vector<int64_t>& shape) {
  int64_t rows = 1;
  for (size_t i = 0; i + 1 < shape.size(); ++i) rows *= shape[i];
  return {rows, shape.back()};
}

Rows check_q8(const Q8Rows& q, const char* op) {
  const std::string o(op);
  require(!q.shape.empty(), o + ": rows must have at least one axis");
  const Rows r = rows_of(q.shape);
  require(q.codes.defined() && q.codes.dtype() == DType::kInt32 && q.codes.device().is_hip() &&
              q.codes.is_contiguous() && q.codes.nbytes() == ember_q8_code_bytes(r.rows, r.H),
          o + ": codes do not belong to the shape");
  check_f32(q.params, op, "params");
  require(q.params.nbytes() == ember_q8_param_bytes(r.rows, r.H),
          o + ": params do not belong to the shape");
  return r;
}

}  // namespace

Q8Rows quantize_q8(const Tensor& x) {
  check_f32(x, "quantize_q8", "x");
  require(x.dim() >= 1, "quantize_q8: x must have >= 1 dim");
  const Rows r = rows_of(x.shape());
  Q8Rows q;
  q.shape = x.shape();
  q.codes = Tensor::empty({static_cast<int64_t>(ember_q8_code_bytes(r.rows, r.H) / 4)},
                          DType::kInt32, x.device());
  q.params = Tensor::empty({static_cast<int64_t>(ember_q8_param_bytes(r.rows, r.H) / 4)},
                           DType::kFloat32, x.device());
  CTD_CHECK(ember_q8_quantize(cfp(x), q.codes.data_ptr(), fp(q.params), r.rows, r.H, S()));
  return q;
}

Tensor dequantize_q8(const Q8Rows& q) {
  const Rows r = check_q8(q, "dequantize_q8");
  Tensor x = Tensor::empty(q.shape, DType::kFloat32, q.params.device());
  CTD_CHECK(ember_q8_dequantize(q.codes.data_ptr(), cfp(q.params), fp(x), r.rows, r.H, S()));
  return x;
}

std::pair<Tensor, NormValues> dequantize_q8_rms_norm(const Q8Rows& q, const Tensor& weight,
                                                     float eps) {
  const Rows r = check_q8(q, "dequantize_q8_rms_norm");
  check_f32(weight, "dequantize_q8_rms_norm", "weight");
  require(weight.dim() == 1 && weight.numel() == r.H,
          "dequantize_q8_rms_norm: weight shape mismatch");
  Tensor x = Tensor::empty(q.shape, DType::kFloat32, q.params.device());
  NormValues v{empty_like(x), Tensor::empty({r.rows}, DType::kFloat32, x.device())};
  CTD_CHECK(ember_q8_dequantize_rmsnorm(q.codes.data_ptr(), cfp(q.params), cfp(weight), fp(x),
                                        fp(v.y), fp(v.rstd), r.rows, r.H, eps, S()));
  return {x, v};
}

namespace {

void check_mx4(const Mx4Weight& w, const char* op) {
  const std::string o(op);
  require(w.defined(), o + ": the weight is undefined");
  auto buffer = [](const Tensor& t, size_t bytes) {
    return t.defined() && t.dtype() == DType::kInt32 && t.device().is_hip() && t.is_contiguous() &&
           t.nbytes() == bytes;
  };
  require(buffer(w.codes, ember_mx4_code_bytes(w.N, w.K)), o + ": codes do not belong to [N, K]");
  require(buffer(w.scales, ember_mx4_scale_bytes(w.N, w.K)), o + ": scales do not belong to [N, K]");
}

// x's rows, with the checks that both products make; M rows of K values.
int64_t check_product(const Tensor& x, const Tensor& norm_w,
                      const std::vector<const Mx4Weight*>& weights, const char* op) {
  const std::string o(op);
  check_f32(x, op, "x");
  require(!autograd::any_requires_grad({x}), o + ": x requires grad, and weights in 4 bits give none");
  for (const Mx4Weight* w : weights) {
    require(w != nullptr, o + ": null weight");
    check_mx4(*w, op);
    require(w->K == weights[0]->K, o + ": weights must be [N, K] with one K");
  }
  const int64_t K = weights[0]->K;
  require(x.dim() >= 1 && x.shape().back() == K, o + ": in_features mismatch");
  if (norm_w.defined()) {
    check_f32(norm_w, op, "norm weight");
    require(norm_w.numel() == K, o + ": norm weight size != in_features");
    require(!autograd::any_requires_grad({norm_w}), o + ": the norm's weight requires grad");
  }
  return x.numel() / K;
}

Tensor with_last(const Tensor& x, int64_t n) {
  std::vector<int64_t> sh = x.shape();
  sh.back() = n;
  return Tensor::empty(sh, DType::kFloat32, x.device());
}

Tensor int_words(size_t bytes) {
  return Tensor::empty({static_cast<int64_t>(bytes / 4)}, DType::kInt32, kHIP0);
}

}  // namespace

Mx4Weight quantize_mx4(const Tensor& w) {
  check_f32(w, "quantize_mx4", "weight");
  require(w.dim() == 2 && w.shape()[0] >= 1 && w.shape()[1] >= 1,
          "quantize_mx4: the weight must be [N, K]");
  Mx4Weight q;
  q.N = w.shape()[0];
  q.K = w.shape()[1];
  q.codes = int_words(ember_mx4_code_bytes(q.N, q.K));
  q.scales = int_words(ember_mx4_scale_bytes(q.N, q.K));
  CTD_CHECK(ember_mx4_quantize(cfp(w), q.codes.data_ptr(), q.scales.data_ptr(), q.N, q.K, S()));
  return q;
}

Tensor dequantize_mx4(const Mx4Weight& q) {
  check_mx4(q, "dequantize_mx4");
  Tensor w = Tensor::empty({q.N, q.K}, DType::kFloat32, q.codes.device());
  CTD_CHECK(ember_mx4_dequantize(q.codes.data_ptr(), q.scales.data_ptr(), fp(w), q.N, q.K, S()));
  return w;
}

Tensor embedding_mx4(const Tensor& ids, const Mx4Weight& table) {
  check_mx4(table, "embedding_mx4");
  require(ids.defined() && ids.dtype() == DType::kInt64 && ids.device().is_hip() &&
              ids.is_contiguous(),
          "embedding_mx4: ids must be contiguous int64 on the HIP device");
  std::vector<int64_t> shape = ids.shape();
  shape.push_back(table.K);
  Tensor out = Tensor::empty(shape, DType::kFloat32, ids.device());
  CTD_CHECK(ember_mx4_embedding(static_cast<const int64_t*>(ids.data_ptr()),
                                table.codes.data_ptr(), table.scales.data_ptr(), fp(out),
                                ids.numel(), table.K, table.N, S()));
  return out;
}

std::vector<Tensor> linear_mx4(const Tensor& x, const Tensor& norm_w, float eps,
                               const std::vector<const Mx4Weight*>& weights,
                               const std::vector<Tensor>& residuals) {
  require(!weights.empty() && weights.size() <= 3, "linear_mx4: 1 to 3 weights");
  require(residuals.empty() || residuals.size() == weights.size(),
          "linear_mx4: one residual per weight");
  const int64_t M = check_product(x, norm_w, weights, "linear_mx4"), K = weights[0]->K;
  std::vector<Tensor> out;
  const void* codes[3] = {};
  const void* scales[3] = {};
  int64_t N[3] = {}, rows = 0;
  float* y[3] = {};
  const float* res[3] = {};
  for (size_t i = 0; i < weights.size(); ++i) {
    const Mx4Weight& w = *weights[i];
    N[i] = w.N;
    rows += w.N;
    codes[i] = w.codes.data_ptr();
    scales[i] = w.scales.data_ptr();
    out.push_back(with_last(x, w.N));
    y[i] = fp(out.back());
    if (!residuals.empty() && residuals[i].defined()) {
      check_f32(residuals[i], "linear_mx4", "residual");
      require(!autograd::any_requires_grad({residuals[i]}), "linear_mx4: a residual requires grad");
      require(residuals[i].shape() == out.back().shape(), "linear_mx4: residual shape");
      res[i] = cfp(residuals[i]);
    }
  }
  const size_t wsb = ember_mx4_workspace_bytes(M, K, rows);
  Tensor ws = wsb ? workspace(wsb) : Tensor{};
  CTD_CHECK(ember_mx4_linear(cfp(x), M, K, norm_w.defined() ? cfp(norm_w) : nullptr, eps,
                             static_cast<int>(weights.size()), codes, scales, N, y, res,
                             wsb ? ws.data_ptr() : nullptr, wsb, S()));
  return out;
}

Tensor gate_up_mx4(const Tensor& x, const Tensor& norm_w, float eps, const Mx4Weight& gate,
                   const Mx4Weight& up) {
  const int64_t M = check_product(x, norm_w, {&gate, &up}, "gate_up_mx4"), K = gate.K;
  require(gate.N == up.N, "gate_up_mx4: gate and up weights differ");
  Tensor out = with_last(x, gate.N);
  const size_t wsb = ember_mx4_workspace_bytes(M, K, 2 * gate.N);
  Tensor ws = wsb ? workspace(wsb) : Tensor{};
  CTD_CHECK(ember_mx4_gateup(cfp(x), M, K, norm_w.defined() ? cfp(norm_w) : nullptr, eps,
                             gate.codes.data_ptr(), gate.scales.data_ptr(), up.codes.data_ptr(),
                             up.scales.data_ptr(), gate.N, fp(out), wsb ? ws.data_ptr() : nullptr,
                             wsb, S()));
  return out;
}

}  // namespace ctd::ops
