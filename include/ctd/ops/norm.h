#pragma once
// RMSNorm (mirrors ops/norm.h of the reference).
#include <utility>

#include "ctd/tensor.h"

namespace ctd::ops {

// y = x * rsqrt(mean(x^2, -1) + eps) * weight; backward gives grads for x and weight.
Tensor rms_norm(const Tensor& x, const Tensor& weight, float eps);
Tensor rms_norm_impl(const Tensor& x, const Tensor& weight, float eps);
std::pair<Tensor, Tensor> rms_norm_backward_impl(const Tensor& dy, const Tensor& x,
                                                 const Tensor& w, float eps);

// What a forward RMSNorm of some x gave, for rms_norm_from.
struct NormValues {
  Tensor y;     // x's shape
  Tensor rstd;  // [rows]
};
// rms_norm(x, weight, eps) where its values are known already: the node
// rms_norm records, over `values.y`.  Added in this build.
Tensor rms_norm_from(const Tensor& x, const Tensor& weight, float eps, const NormValues& values);

}  // namespace ctd::ops
