#pragma once
// RMSNorm with learned scale, no bias (mirrors nn/rms_norm.h of the reference).
#include "ctd/ops/norm.h"
#include "ctd/tensor.h"

namespace ctd::nn {

struct RMSNorm {
  Tensor weight;  // [hidden]
  float eps = 1e-5f;

  Tensor forward(const Tensor& x) const { return ops::rms_norm(x, weight, eps); }
  // forward(x), its values given (ops::rms_norm_from).
  Tensor forward_from(const Tensor& x, const ops::NormValues& values) const {
    return ops::rms_norm_from(x, weight, eps, values);
  }
};

}  // namespace ctd::nn
