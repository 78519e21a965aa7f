// C++-API tests of weights held in 4 bits, through include/ctd/.  Run on a GPU
// by tests/test_gpu_mx4_model.py; exit status = number of failed checks.
#include <cmath>
#include <cstdio>
#include <random>
#include <stdexcept>
#include <string>
#include <vector>

#include "ctd/autograd.h"
#include "ctd/nn/linear.h"
#include "ctd/nn/mlp.h"
#include "ctd/nn/model.h"
#include "ctd/ops/embedding.h"
#include "ctd/ops/matmul.h"
#include "ctd/ops/norm.h"
#include "ctd/ops/quant.h"
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

template <typename F>
void refuses(F f, const std::string& text) {
  std::string got = "(nothing)";
  try {
    f();
  } catch (const std::runtime_error& e) {
    got = e.what();
  }
  check(got.find(text) != std::string::npos, "expected an error with '" + text + "', got " + got);
}

std::vector<float> host(const Tensor& t) {
  std::vector<float> h(static_cast<size_t>(t.numel()));
  t.copy_to_host(h.data());
  return h;
}

Tensor randn(const std::vector<int64_t>& shape, unsigned seed, float scale = 1.0f) {
  std::mt19937 rng(seed);
  std::normal_distribution<float> nd(0.0f, scale);
  int64_t n = 1;
  for (int64_t d : shape) n *= d;
  std::vector<float> h(static_cast<size_t>(n));
  for (float& v : h) v = nd(rng);
  return Tensor::from_host(h.data(), shape, DType::kFloat32, kHIP0);
}

// Two fp32 sums of the same products in other orders: 3e-6 in the 2-norm is some
// tens of half-steps (2^-24), and a term left out at K = 100 shows as 1e-1.
bool near(const Tensor& a, const Tensor& b, double rtol = 3e-6) {
  const auto x = host(a), y = host(b);
  double err = 0, norm = 0;
  for (size_t i = 0; i < x.size() && i < y.size(); ++i) {
    err += (double(x[i]) - y[i]) * (double(x[i]) - y[i]);
    norm += double(y[i]) * y[i];
  }
  return a.shape() == b.shape() && std::sqrt(err) <= rtol * std::sqrt(norm);
}

void products() {
  const Tensor wf[3] = {randn({70, 100}, 1, 0.1f), randn({33, 100}, 2, 0.1f),
                        randn({64, 100}, 3, 0.1f)};
  const Tensor nw = randn({100}, 4, 0.3f);
  ops::Mx4Weight w[3];
  Tensor back[3];
  for (int i = 0; i < 3; ++i) {
    w[i] = ops::quantize_mx4(wf[i]);
    back[i] = ops::dequantize_mx4(w[i]);
    check(back[i].shape() == wf[i].shape(), "dequantize_mx4's shape");
    check(near(back[i], wf[i], 0.2) && !near(back[i], wf[i], 0.01), "four bits of the weight");
  }
  for (const std::vector<int64_t>& lead :
       {std::vector<int64_t>{1}, {2, 3}, {1, 9}, {4, 50}, {0}, {2, 1, 5}}) {
    std::vector<int64_t> shape = lead;
    shape.push_back(100);
    const Tensor x = randn(shape, 5);
    const int64_t M = x.numel() / 100;
    const Tensor x2 = x.reshape({M, 100});
    const Tensor xn = M ? ops::rms_norm(x2, nw, 1e-5f) : x2;
    std::vector<int64_t> last = lead;
    last.push_back(33);
    const Tensor res = randn(last, 6);
    const auto y = ops::linear_mx4(x, nw, 1e-5f, {&w[0], &w[1], &w[2]}, {Tensor{}, res, Tensor{}});
    check(y.size() == 3, "three products");
    if (M == 0) {
      check(y[1].numel() == 0 && ops::gate_up_mx4(x, nw, 1e-5f, w[0], w[0]).numel() == 0,
            "no rows, no products");
      continue;
    }
    for (int i = 0; i < 3; ++i) {
      Tensor want = ops::matmul(xn, back[i], false, true);
      if (i == 1) want = ops::add(want, res.reshape({M, 33}));
      check(near(y[size_t(i)].reshape(want.shape()), want), "linear_mx4 under a norm");
      check(y[size_t(i)].shape().back() == w[i].N && y[size_t(i)].dim() == x.dim(), "its shape");
    }
    const Tensor plain = ops::linear_mx4(x, Tensor{}, 0.0f, {&w[0]})[0];
    check(near(plain.reshape({M, 70}), ops::matmul(x2, back[0], false, true)), "linear_mx4");
    nn::MLP mlp;
    mlp.gate_proj.weight = back[0];
    mlp.up_proj.weight = ops::dequantize_mx4(ops::quantize_mx4(randn({70, 100}, 7, 0.1f)));
    autograd::NoGradGuard ng;
    const ops::Mx4Weight up = ops::quantize_mx4(randn({70, 100}, 7, 0.1f));
    check(near(ops::gate_up_mx4(x, nw, 1e-5f, w[0], up).reshape({M, 70}), mlp.activation(xn)),
          "gate_up_mx4");
  }
  const std::vector<int64_t> idh{0, 69, 5, 5, -1, 70};
  const Tensor ids = Tensor::from_host(idh.data(), {2, 3}, DType::kInt64, kHIP0);
  check(host(ops::embedding_mx4(ids, w[0])) == host(ops::embedding(ids, back[0])),
        "embedding_mx4 is the table's read back");
}

void modules() {
  const Tensor wf = randn({48, 96}, 1, 0.1f);
  nn::Linear held, plain;
  held.mx4 = ops::quantize_mx4(wf);
  plain.weight = ops::dequantize_mx4(held.mx4);
  const Tensor x = randn({2, 7, 96}, 2), r = randn({2, 7, 48}, 3);
  check(near(held.forward(x), plain.forward(x)), "Linear::forward");
  check(near(held.forward_add(x, r), plain.forward_add(x, r)), "Linear::forward_add");
  refuses([&] { held.forward(randn({2, 95}, 4)); }, "in_features mismatch");
  refuses([&] { held.forward_add(x, randn({2, 7, 47}, 4)); }, "residual shape");
  refuses([&] { held.forward_graph_only(x, r); }, "no backward");
  Tensor g = randn({3, 96}, 5);
  g.requires_grad_(true);
  refuses([&] { held.forward(g); }, "x requires grad");
  autograd::NoGradGuard ng;
  check(near(held.forward(g), plain.forward(g)), "under no-grad it does not matter");
}

void refusals() {
  const Tensor w = randn({8, 64}, 1);
  const ops::Mx4Weight q = ops::quantize_mx4(w);
  refuses([&] { ops::quantize_mx4(randn({64}, 1)); }, "must be [N, K]");
  refuses([&] { ops::quantize_mx4(Tensor{}); }, "undefined");
  refuses([&] { ops::dequantize_mx4({}); }, "undefined");
  ops::Mx4Weight bad = q;
  bad.K = 65;
  refuses([&] { ops::dequantize_mx4(bad); }, "codes do not belong");
  bad = q;
  bad.scales = q.codes;
  refuses([&] { ops::dequantize_mx4(bad); }, "scales do not belong");
  const Tensor x = randn({2, 64}, 2);
  refuses([&] { ops::linear_mx4(x, Tensor{}, 0.0f, {}); }, "1 to 3 weights");
  refuses([&] { ops::linear_mx4(x, Tensor{}, 0.0f, {&q, &q, &q, &q}); }, "1 to 3 weights");
  refuses([&] { ops::linear_mx4(x, Tensor{}, 0.0f, {nullptr}); }, "null weight");
  refuses([&] { ops::linear_mx4(x, randn({63}, 1), 0.0f, {&q}); }, "norm weight size");
  refuses([&] { ops::linear_mx4(x, Tensor{}, 0.0f, {&q}, {x, x}); }, "one residual per weight");
  refuses([&] { ops::linear_mx4(x, Tensor{}, 0.0f, {&q}, {x}); }, "residual shape");
  const ops::Mx4Weight other = ops::quantize_mx4(randn({8, 65}, 3));
  refuses([&] { ops::linear_mx4(x, Tensor{}, 0.0f, {&q, &other}); }, "one K");
  refuses([&] { ops::gate_up_mx4(x, Tensor{}, 0.0f, q, other); }, "one K");
  const ops::Mx4Weight taller = ops::quantize_mx4(randn({9, 64}, 3));
  refuses([&] { ops::gate_up_mx4(x, Tensor{}, 0.0f, q, taller); }, "differ");
  refuses([&] { ops::embedding_mx4(x, q); }, "int64");
  Tensor r = randn({2, 8}, 4);
  r.requires_grad_(true);
  refuses([&] { ops::linear_mx4(x, Tensor{}, 0.0f, {&q}, {r}); }, "residual requires grad");
  Tensor nw = randn({64}, 5);
  nw.requires_grad_(true);
  refuses([&] { ops::linear_mx4(x, nw, 1e-5f, {&q}); }, "norm's weight requires grad");
  refuses([&] { ops::gate_up_mx4(x, nw, 1e-5f, q, q); }, "norm's weight requires grad");
}

nn::Model small_model(bool qk_norm) {
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
  c.qk_norm = qk_norm;
  TensorDict w;
  unsigned seed = 1;
  auto put = [&](const std::string& k, std::vector<int64_t> s, float scale) {
    w.emplace(k, randn(s, seed++, scale));
  };
  put("model.embed_tokens.weight", {50, 96}, 0.5f);
  put("model.norm.weight", {96}, 1.0f);
  for (int l = 0; l < 2; ++l) {
    const std::string p = "model.layers." + std::to_string(l) + ".";
    put(p + "input_layernorm.weight", {96}, 1.0f);
    put(p + "post_attention_layernorm.weight", {96}, 1.0f);
    put(p + "self_attn.q_proj.weight", {128, 96}, 0.1f);
    put(p + "self_attn.k_proj.weight", {64, 96}, 0.1f);
    put(p + "self_attn.v_proj.weight", {64, 96}, 0.1f);
    put(p + "self_attn.o_proj.weight", {96, 128}, 0.1f);
    if (qk_norm) {
      put(p + "self_attn.q_norm.weight", {64}, 1.0f);
      put(p + "self_attn.k_norm.weight", {64}, 1.0f);
    }
    put(p + "mlp.gate_proj.weight", {160, 96}, 0.1f);
    put(p + "mlp.up_proj.weight", {160, 96}, 0.1f);
    put(p + "mlp.down_proj.weight", {96, 160}, 0.1f);
  }
  return nn::build_model(w, c);
}

void models() {
  for (bool qk : {false, true}) {
    nn::Model m = small_model(qk);
    m.collect_parameters();  // everything requires grad, as after training
    check(!m.weights_quantized(), "fp32 to begin with");
    m.quantize_weights();
    check(m.weights_quantized() && !m.layers[1].mlp.up_proj.weight.defined() &&
              m.embed_tokens.weight.defined() && !m.norm.weight.requires_grad(),
          "the projections only");
    refuses([&] { m.collect_parameters(); }, "no parameters");
    const std::vector<int64_t> idh{3, 49, 0, 7, 7, 21, 30, 2, 11, 12, 13, 14};
    const Tensor ids = Tensor::from_host(idh.data(), {1, 12}, DType::kInt64, kHIP0);
    const Tensor all = m.forward(ids);
    Tensor logits = m.forward_train_logits(ids);
    check(!logits.requires_grad(), "no graph");
    check(near(logits, all), "the training forward is the same function");
    const Tensor loss = m.forward_train(ids, ids);
    m.gradient_checkpointing = true;
    check(host(m.forward_train(ids, ids)) == host(loss), "checkpointing changes nothing");
    m.quantize_weights(true);
    check(!m.embed_tokens.weight.defined(), "and now the table");
    m.quantize_weights(true);
    const Tensor again = m.forward(ids);
    check(!near(again, all, 1e-3) && near(again, m.forward_train_logits(ids)), "a 4-bit head");
    check(std::isfinite(host(m.forward_train(ids, ids))[0]), "a loss over it");
  }
}

}  // namespace

int main() {
  products();
  modules();
  refusals();
  models();
  runtime::synchronize();
  std::printf("%d failure(s)\n", g_failed);
  return g_failed;
}
