#pragma once
// Rows held in 8 bits (added in this build; ember_q8_quantize in ember_hip.h
// gives the rule): what autograd::checkpoint_q8 keeps of a block's input.
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

}  // namespace ctd::ops
