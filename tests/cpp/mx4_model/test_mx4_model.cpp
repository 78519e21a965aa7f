// C++-API tests of what nn::Model::quantize_weights leaves to others: models that share its tensors,
// gradients, memory.  Run on a GPU by tests/test_gpu_mx4_owners.py; exit status = number of failed checks.
#include <cmath>
#include <cstdio>
#include <random>
#include <string>
#include <vector>

#include "ctd/allocator.h"
#include "ctd/autograd.h"
#include "ctd/nn/model.h"
#include "ctd/runtime.h"
#include "ctd/tensor.h"

using namespace ctd;

namespace {

int g_failed = 0;

void check(bool ok, const std::string& what) {
  if (!ok) {
    ++g_failed;
    std::printf("  FAILED: %s\n", what.c_str());
  }
}

std::vector<float> host(const Tensor& t) {
  std::vector<float> h(static_cast<size_t>(t.numel()));
  t.copy_to_host(h.data());
  return h;
}

nn::Model small_model() {
  nn::LlamaConfig c{};
  c.vocab_size = 50;
  c.hidden_size = 96;
  c.intermediate_size = 160;
  c.num_hidden_layers = 2;
  c.num_attention_heads = 2;
  c.num_key_value_heads = 1;
  c.head_dim = 64;
  c.rms_norm_eps = 1e-5f;
  c.rope_theta = 1e4f;
  c.tie_word_embeddings = true;
  c.qk_norm = true;
  TensorDict w;
  std::mt19937 rng(7);
  auto put = [&](const std::string& name, const std::vector<int64_t>& shape) {
    std::normal_distribution<float> nd(0.0f, shape.size() == 1 ? 1.0f : 0.1f);
    int64_t n = 1;
    for (int64_t d : shape) n *= d;
    std::vector<float> h(static_cast<size_t>(n));
    for (float& v : h) v = nd(rng);
    w.emplace(name, Tensor::from_host(h.data(), shape, DType::kFloat32, kHIP0));
  };
  put("model.embed_tokens.weight", {50, 96});
  put("model.norm.weight", {96});
  for (int l = 0; l < 2; ++l) {
    const std::string p = "model.layers." + std::to_string(l) + ".";
    put(p + "input_layernorm.weight", {96});
    put(p + "post_attention_layernorm.weight", {96});
    put(p + "self_attn.q_proj.weight", {128, 96});
    put(p + "self_attn.k_proj.weight", {64, 96});
    put(p + "self_attn.v_proj.weight", {64, 96});
    put(p + "self_attn.o_proj.weight", {96, 128});
    put(p + "self_attn.q_norm.weight", {64});
    put(p + "self_attn.k_norm.weight", {64});
    put(p + "mlp.gate_proj.weight", {160, 96});
    put(p + "mlp.up_proj.weight", {160, 96});
    put(p + "mlp.down_proj.weight", {96, 160});
  }
  return nn::build_model(w, c);
}

Tensor some_ids() {
  const std::vector<int64_t> ids{3, 49, 0, 7, 7, 21, 30, 2, 11, 12, 13, 14};
  return Tensor::from_host(ids.data(), {1, 12}, DType::kInt64, kHIP0);
}

// Gradients of every parameter, cleared behind.
std::vector<std::vector<float>> gradients(const nn::Model& m, nn::Model::NamedParameters& named) {
  m.forward_train(some_ids(), some_ids()).backward();
  std::vector<std::vector<float>> out;
  for (auto& [name, p] : named.all) {
    check(p.grad().defined(), "a gradient for " + name);
    out.push_back(p.grad().defined() ? host(p.grad()) : std::vector<float>{});
    p.zero_grad_();
  }
  return out;
}

// A copy of a model shares its tensors; bringing the copy into 4 bits changes nothing of the other.
void the_model_it_was_copied_from() {
  for (bool table : {false, true}) {
    nn::Model m = small_model();
    auto named = m.collect_parameters();
    const auto before = gradients(m, named);
    nn::Model held = m;
    held.quantize_weights(table);
    for (auto& [name, p] : named.all) check(p.requires_grad(), name + " still requires grad");
    check(gradients(m, named) == before, "the same gradients as before");
    check(!held.forward_train(some_ids(), some_ids()).requires_grad(), "no graph over the copy");
    check(!held.norm.weight.requires_grad() && !held.layers[1].self_attn.k_norm.weight.requires_grad(),
          "the copy's norms");
    check(table || !held.embed_tokens.weight.requires_grad(), "the copy's table");
    check(!m.weights_quantized() && std::isfinite(host(held.forward(some_ids()))[0]), "both run");
  }
}

// Live bytes of a model in 4 bits that had gradients before, or had none.
size_t held_bytes(bool trained, bool table) {
  runtime::synchronize();
  const size_t base = device_memory_stats().allocated_bytes;
  nn::Model m = small_model();
  if (trained) {
    auto named = m.collect_parameters();
    m.forward_train(some_ids(), some_ids()).backward();
  }
  m.quantize_weights(table);
  runtime::synchronize();
  return device_memory_stats().allocated_bytes - base;
}

void gradients_go_too() {
  for (bool table : {false, true})
    check(held_bytes(true, table) == held_bytes(false, table), "no gradient is kept");
}

}  // namespace

int main() {
  the_model_it_was_copied_from();
  gradients_go_too();
  runtime::synchronize();
  std::printf("%d failure(s)\n", g_failed);
  return g_failed;
}
