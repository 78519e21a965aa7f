#pragma once
// Values held in few bits (added in this build): rows in 8 bits, what
// autograd::checkpoint_q8 keeps of a block's input, and weights in 4 bits, what
// nn::Model::quantize_weights makes of a model's (ember_q8_quantize and
// ember_mx4_quantize in ember_hip.h give the rules).
#include <utility>
#include <vector>

#include "ctd/ops/norm.h"
#include "ctd/tensor.h"

namespace ctd::ops {

// x [..., H] fp32 as 8-bit codes (int32 words, rows of round_up(H, 16) bytes) and
// {offset, step} per group of 128 values along the last axis.
struct Q8Rows {
  std::vector<int64_t> shape;
  Tensor codes;
  Tensor params;
};

Q8Rows quantize_q8(const Tensor& x);
Tensor dequantize_q8(const Q8Rows& q);
// dequantize_q8(q) and the values of its RMSNorm, in one pass.
std::pair<Tensor, NormValues> dequantize_q8_rms_norm(const Q8Rows& q, const Tensor& weight,
                                                     float eps);

// A weight [N, K] in microscaled 4-bit floating point: groups of 32 values along
// a row with a power of two each, 17/32 bytes a value, in the tiles that the
// products read (int32 words).
struct Mx4Weight {
  int64_t N = 0, K = 0;
  Tensor codes;
  Tensor scales;
  bool defined() const { return codes.defined(); }
};

Mx4Weight quantize_mx4(const Tensor& w);
Tensor dequantize_mx4(const Mx4Weight& w);
// Rows of the table: ids int64 [...] -> fp32 [..., K] (zeros for ids outside it).
Tensor embedding_mx4(const Tensor& ids, const Mx4Weight& table);
// Products with such weights, for x [..., K] of any number of rows; none of them
// records autograd history, and an x, norm weight or residual that requires grad is
// refused.
// linear_mx4: for each of 1 to 3 weights, xn W_i^T (+ residuals[i] where given and
// defined, same shape) -> [..., N_i], xn = RMSNorm(x; norm_w, eps) when norm_w is
// defined, else x.  gate_up_mx4: silu(xn Wg^T) * (xn Wu^T), the MLP's input half.
std::vector<Tensor> linear_mx4(const Tensor& x, const Tensor& norm_w, float eps,
                               const std::vector<const Mx4Weight*>& weights,
                               const std::vector<Tensor>& residuals = {});
Tensor gate_up_mx4(const Tensor& x, const Tensor& norm_w, float eps, const Mx4Weight& gate,
                   const Mx4Weight& up);

}  // namespace ctd::ops
