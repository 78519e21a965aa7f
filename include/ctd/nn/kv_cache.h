#pragma once
// KV cache for autoregressive decoding (mirrors nn/kv_cache.h of the reference).
#include <cstdint>
#include <stdexcept>
#include <vector>

#include "ctd/tensor.h"

namespace ctd::nn {

// One layer's cache, k and v each fp32 [B, H_kv, max_seq_len, D]; in 4 bits
// (added in this build) k and v are the codes, int32 [B, H_kv, max_seq_len, D/8],
// and k_params / v_params [B, H_kv, max_seq_len, 2] their rows' offsets and
// steps (ops/kv_cache.h).
struct KVLayer {
  Tensor k;
  Tensor v;
  Tensor k_params{};
  Tensor v_params{};
  bool kv4() const { return k_params.defined(); }
};

struct KVCache {
  std::vector<KVLayer> layers;
  int64_t current_len = 0;
  int64_t max_seq_len = 0;
  int64_t batch = 0;

  // Zero-filled cache for num_layers layers: 2 * num_layers * batch * H_kv *
  // max_seq rows of 4 D bytes, or of D / 2 + 8 with bits = 4 (head_dim a
  // multiple of 8 up to 256).
  static KVCache allocate(int num_layers, int num_kv_heads, int head_dim, int64_t batch,
                          int64_t max_seq, Device device, int bits = 32) {
    if (bits != 32 && bits != 4) throw std::runtime_error("KVCache: bits must be 32 or 4");
    if (bits == 4 && (head_dim < 8 || head_dim > 256 || head_dim % 8 != 0))
      throw std::runtime_error("KVCache: 4 bits need a head_dim that is a multiple of 8 up to 256");
    KVCache c;
    c.batch = batch;
    c.max_seq_len = max_seq;
    c.layers.reserve(num_layers);
    for (int i = 0; i < num_layers; ++i) {
      if (bits == 4) {
        auto codes = [&] {
          return Tensor::zeros({batch, num_kv_heads, max_seq, head_dim / 8}, DType::kInt32, device);
        };
        auto params = [&] {
          return Tensor::zeros({batch, num_kv_heads, max_seq, 2}, DType::kFloat32, device);
        };
        c.layers.push_back({codes(), codes(), params(), params()});
        continue;
      }
      c.layers.push_back({Tensor::zeros({batch, num_kv_heads, max_seq, head_dim},
                                        DType::kFloat32, device),
                          Tensor::zeros({batch, num_kv_heads, max_seq, head_dim},
                                        DType::kFloat32, device)});
    }
    return c;
  }

  void reset() { current_len = 0; }
};

}  // namespace ctd::nn
