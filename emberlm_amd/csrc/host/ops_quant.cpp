// Rows held in 8 bits.  None of these record autograd history.
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

}  // namespace ctd::ops
