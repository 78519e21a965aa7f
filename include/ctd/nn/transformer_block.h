#pragma once
// Llama-style decoder block: h = x + attn(norm(x)); y = h + mlp(norm(h))
// (mirrors nn/transformer_block.h of the reference).
#include "ctd/nn/attention.h"
#include "ctd/nn/mlp.h"
#include "ctd/nn/rms_norm.h"
#include "ctd/ops/decode.h"
#include "ctd/ops/elementwise.h"
#include "ctd/tensor.h"

namespace ctd::nn {

struct TransformerBlock {
  RMSNorm input_layernorm;
  RMSNorm post_attention_layernorm;
  Attention self_attn;
  MLP mlp;

  // Inference forward.  With a KV cache and at most ops::kDecodeMaxRows token
  // rows (a decode step), the fused decode kernels run the same functions in
  // five launches (six when long contexts split the keys); otherwise the
  // module ops run one by one.
  Tensor forward(const Tensor& x, KVLayer* kv = nullptr, int position_start = 0) const {
    autograd::NoGradGuard ng;
    if (mx4()) return forward_mx4(x, kv, position_start);
    if (fused_decode(x, kv)) return decode_step(x, *kv, position_start);
    Tensor h1 = input_layernorm.forward(x);
    Tensor h = self_attn.o_proj.forward_add(self_attn.forward_context(h1, kv, position_start), x);
    Tensor h2 = post_attention_layernorm.forward(h);
    return mlp.forward_add(h2, h);
  }

  // Whether the projections are held in 4 bits (nn::Model::quantize_weights: all
  // of them or none).
  bool mx4() const { return self_attn.q_proj.mx4.defined(); }

  // forward() with projections in 4 bits, from one token to a long prompt: Q, K
  // and V from one call that takes the norm along, the MLP's input half from
  // another, the residuals added in the products' stores.  A decode step's
  // attention is the fused kernels' (decode_step).
  Tensor forward_mx4(const Tensor& x, KVLayer* kv, int position_start) const {
    autograd::NoGradGuard ng;
    if (x.dim() != 3) throw std::runtime_error("TransformerBlock: x must be [B, T, hidden]");
    const int64_t B = x.shape()[0], T = x.shape()[1];
    const Attention& at = self_attn;
    const int64_t H = at.num_heads, Hk = at.num_kv_heads, D = at.head_dim;
    auto qkv = ops::linear_mx4(x, input_layernorm.weight, input_layernorm.eps,
                               {&at.q_proj.mx4, &at.k_proj.mx4, &at.v_proj.mx4});
    Tensor a = fused_decode(x, kv)
                   ? decode_attention(qkv, *kv, position_start)
                   : at.context_of(qkv[0].reshape({B, T, H, D}), qkv[1].reshape({B, T, Hk, D}),
                                   qkv[2].reshape({B, T, Hk, D}), kv, position_start);
    Tensor h =
        ops::linear_mx4(a.reshape({B, T, H * D}), Tensor{}, 0.0f, {&at.o_proj.mx4}, {x})[0];
    Tensor m = ops::gate_up_mx4(h, post_attention_layernorm.weight, post_attention_layernorm.eps,
                                mlp.gate_proj.mx4, mlp.up_proj.mx4);
    return ops::linear_mx4(m, Tensor{}, 0.0f, {&mlp.down_proj.mx4}, {h})[0];
  }

  // Whether a call is a decode step of the fused kernels.
  bool fused_decode(const Tensor& x, const KVLayer* kv) const {
    return kv != nullptr && x.dim() == 3 &&
           x.shape()[0] * x.shape()[1] <= ops::kDecodeMaxRows &&
           Attention::fused_head_dim(self_attn.head_dim) &&
           (!kv->kv4() || self_attn.group() <= ops::kDecodeKv4MaxGroup);
  }

  // A decode step's attention from its raw projections: norms, rotation, cache
  // write and attention in one launch (plus the split merge).
  Tensor decode_attention(const std::vector<Tensor>& qkv, KVLayer& kv, int position_start) const {
    const Attention& at = self_attn;
    const int H = at.num_heads, Hk = at.num_kv_heads, D = at.head_dim;
    const float scale = 1.0f / std::sqrt(static_cast<float>(D));
    return kv.kv4()
               ? ops::decode_qkv_attention_kv4(qkv[0], qkv[1], qkv[2], H, Hk, D, at.q_norm.weight,
                                               at.k_norm.weight, at.q_norm.eps, at.rope_theta,
                                               at.rope_scaling, position_start, kv.k, kv.k_params,
                                               kv.v, kv.v_params, scale)
               : ops::decode_qkv_attention(qkv[0], qkv[1], qkv[2], H, Hk, D, at.q_norm.weight,
                                           at.k_norm.weight, at.q_norm.eps, at.rope_theta,
                                           at.rope_scaling, position_start, kv.k, kv.v, scale);
  }

  Tensor decode_step(const Tensor& x, KVLayer& kv, int position_start) const {
    const int64_t B = x.shape()[0], T = x.shape()[1];
    const Attention& at = self_attn;
    const int H = at.num_heads, D = at.head_dim;
    auto qkv = ops::decode_linear(x, input_layernorm.weight, input_layernorm.eps,
                                  {at.q_proj.weight, at.k_proj.weight, at.v_proj.weight});
    Tensor a = decode_attention(qkv, kv, position_start);
    Tensor h = ops::decode_linear(a.reshape({B, T, static_cast<int64_t>(H) * D}), Tensor{}, 0.0f,
                                  {at.o_proj.weight}, {x})[0];
    Tensor m = ops::decode_gate_up(h, post_attention_layernorm.weight,
                                   post_attention_layernorm.eps, mlp.gate_proj.weight,
                                   mlp.up_proj.weight);
    return ops::decode_linear(m, Tensor{}, 0.0f, {mlp.down_proj.weight}, {h})[0];
  }

  // The residual adds run inside the o_proj and down_proj GEMMs (bitwise the
  // same as ops::add after the product, same autograd graph).
  Tensor forward_train(const Tensor& x) const {
    Tensor h1 = input_layernorm.forward(x);
    Tensor h = self_attn.o_proj.forward_add(self_attn.forward_train_context(h1), x);
    Tensor h2 = post_attention_layernorm.forward(h);
    return mlp.forward_add(h2, h);
  }

  // forward_train(x) for a checkpoint's recompute, whose backward reads only
  // the graph of the block's output: down_proj and the last residual add are
  // recorded but not run, so the returned tensor has forward_train(x)'s
  // grad_fn but no values of its own (a placeholder: data_ptr() and
  // copy_to_host() throw).  Its gradients are forward_train's, kernel for
  // kernel.  The checkpointed forward already computed the real output: it is
  // the next block's saved input.
  // normed: input_layernorm's values at x where they are known
  // (autograd::checkpoint_q8 restores them with x).
  Tensor forward_train_for_backward(const Tensor& x,
                                    const ops::NormValues* normed = nullptr) const {
    Tensor h1 = normed ? input_layernorm.forward_from(x, *normed) : input_layernorm.forward(x);
    Tensor h = self_attn.o_proj.forward_add(self_attn.forward_train_context(h1), x);
    Tensor h2 = post_attention_layernorm.forward(h);
    Tensor m = mlp.down_proj.forward_graph_only(mlp.activation(h2), h);
    return ops::add_graph_only(h, m.reshape(h.shape()), h).mark_placeholder();
  }
};

}  // namespace ctd::nn
