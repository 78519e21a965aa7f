#pragma once
// Token embedding lookup (mirrors nn/embedding.h of the reference).
#include "ctd/ops/embedding.h"
#include "ctd/ops/quant.h"
#include "ctd/tensor.h"

namespace ctd::nn {

struct Embedding {
  Tensor weight;  // [vocab, hidden]
  // Instead of weight: the table in 4 bits (nn::Model::quantize_weights).
  ops::Mx4Weight mx4{};
  Tensor forward(const Tensor& ids) const {
    return mx4.defined() ? ops::embedding_mx4(ids, mx4) : ops::embedding(ids, weight);
  }
};

}  // namespace ctd::nn
