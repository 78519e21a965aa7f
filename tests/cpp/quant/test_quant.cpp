// C++-API tests of the few-bit stores: checkpoints in 8 bits and the 4-bit KV
// cache, through include/ctd/.  Run on a GPU by tests/test_gpu_quant_model.py;
// exit status = number of failed checks.
#include <cmath>
#include <cstdio>
#include <functional>
#include <random>
#include <stdexcept>
#include <string>
#include <vector>

#include "ctd/autograd.h"
#include "ctd/nn/kv_cache.h"
#include "ctd/nn/transformer_block.h"
#include "ctd/ops/attention.h"
#include "ctd/ops/decode.h"
#include "ctd/ops/elementwise.h"
#include "ctd/ops/kv_cache.h"
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

// fn(x) = silu(RMSNorm(x) W): what the checkpoints below wrap.
struct Layer {
  Tensor nw = randn({96}, 1, 0.2f), w = randn({96, 40}, 2, 0.1f);
  float eps = 1e-5f;
  Layer() {
    nw.requires_grad_(true);
    w.requires_grad_(true);
  }
  Tensor operator()(const Tensor& x, const ops::NormValues* normed = nullptr) const {
    Tensor h = normed ? ops::rms_norm_from(x, nw, eps, *normed) : ops::rms_norm(x, nw, eps);
    return ops::silu(ops::matmul(h, w));
  }
  void zero() {
    nw.zero_grad_();
    w.zero_grad_();
  }
};

bool near(const std::vector<float>& a, const std::vector<float>& b, double rtol) {
  double err = 0, norm = 0;
  for (size_t i = 0; i < a.size(); ++i) {
    err += (double(a[i]) - b[i]) * (double(a[i]) - b[i]);
    norm += double(b[i]) * b[i];
  }
  return a.size() == b.size() && std::sqrt(err) <= rtol * std::sqrt(norm);
}

// The forward is fn's; the gradients are fn's at the restored input, also with
// a norm given, under a retained graph twice over, and for an input that other
// nodes use too.
void checkpoint_gradients(bool norm) {
  Layer f;
  const Tensor x0 = randn({3, 70, 96}, 3), dy = randn({210, 40}, 4);
  const Tensor held = ops::dequantize_q8(ops::quantize_q8(x0));
  auto flat = [](const Tensor& x) { return x.reshape({210, 96}); };
  auto run = [&](Tensor x) {
    if (norm)
      return autograd::checkpoint_q8(
          [&](const Tensor& v, const ops::NormValues* n) { return f(v, n); }, flat(x), f.nw, f.eps);
    return autograd::checkpoint_q8([&](const Tensor& v) { return f(v); }, flat(x));
  };
  Tensor at = held.detach();
  at.requires_grad_(true);
  f(flat(at)).backward(dy);
  const auto gx = host(at.grad()), gw = host(f.w.grad()), gn = host(f.nw.grad());
  f.zero();

  std::vector<float> want;
  {
    autograd::NoGradGuard ng;
    want = host(f(flat(x0)));
  }
  Tensor x = x0.detach();
  x.requires_grad_(true);
  Tensor y = run(x);
  check(host(y) == want, "the forward pass runs on the input itself");
  y.backward(dy, /*retain_graph=*/true);
  // rms_norm's own sums against those of the restoring pass: roundings only
  check(near(host(x.grad()), gx, 1e-5), "input gradient at the restored input");
  check(near(host(f.w.grad()), gw, 1e-5), "weight gradient at the restored input");
  check(near(host(f.nw.grad()), gn, 1e-5), "norm weight gradient at the restored input");
  const auto once = host(x.grad());
  y.backward(dy);
  auto twice = host(x.grad());
  for (float& v : twice) v *= 0.5f;
  check(near(twice, once, 1e-6), "a second pass through the retained graph");
  f.zero();

  // the input's other use adds its gradient: here dy2 itself
  Tensor z = x0.detach();
  z.requires_grad_(true);
  Tensor s = ops::mul(z, z);  // not a leaf
  Tensor p = run(s);
  p.backward(dy);
  check(z.grad().defined() && z.grad().shape() == z.shape(), "gradient through a non-leaf input");
  f.zero();

  autograd::NoGradGuard ng;
  Tensor plain = run(x0);
  check(!plain.requires_grad() && host(plain) == want, "without a graph it is fn");
}

void refusals() {
  Layer f;
  const Tensor x = randn({4, 96}, 5);
  const Tensor ids = Tensor::zeros({4, 96}, DType::kInt64, kHIP0);
  auto fn = [&](const Tensor& v) { return f(v); };
  refuses([&] { autograd::checkpoint_q8(fn, ids); }, "must be float32");
  refuses([&] {
    autograd::checkpoint_q8([&](const Tensor& v, const ops::NormValues*) { return f(v); }, x,
                            randn({95}, 6), 1e-5f);
  }, "norm weight does not belong");
  ops::Q8Rows q = ops::quantize_q8(x);
  refuses([&] { ops::dequantize_q8_rms_norm(q, randn({95}, 6), 1e-5f); }, "weight shape");
  q.shape = {5, 96};
  refuses([&] { ops::dequantize_q8(q); }, "do not belong to the shape");
  refuses([&] { ops::rms_norm_from(x, f.nw, 1e-5f, {randn({4, 95}, 1), randn({4}, 1)}); },
          "another shape");

  refuses([&] { nn::KVCache::allocate(1, 2, 64, 1, 8, kHIP0, 5); }, "bits must be 32 or 4");
  refuses([&] { nn::KVCache::allocate(1, 2, 60, 1, 8, kHIP0, 4); }, "multiple of 8");
  nn::KVCache c = nn::KVCache::allocate(1, 2, 64, 1, 8, kHIP0, 4);
  nn::KVLayer& l = c.layers[0];
  const Tensor k = randn({1, 3, 2, 64}, 7), q4 = randn({1, 3, 4, 64}, 8);
  auto write = [&](const Tensor& a, int pos) {
    ops::write_kv4_inplace(l.k, l.k_params, l.v, l.v_params, a, a, pos);
  };
  refuses([&] { write(k, 6); }, "out of cache bounds");
  refuses([&] { write(k, -1); }, "out of cache bounds");
  refuses([&] { write(randn({1, 3, 3, 64}, 7), 0); }, "dim mismatch");
  refuses([&] { write(randn({1, 3, 2, 128}, 7), 0); }, "dim mismatch");
  refuses([&] { ops::write_kv4_inplace(l.k_params, l.k, l.v, l.v_params, k, k, 0); }, "int32");
  refuses([&] { ops::read_kv4_expanded(l.k, l.k_params, 9, 1); }, "valid_len");
  refuses([&] { ops::read_kv4_expanded(l.k, l.k_params, 3, 0); }, "group");
  auto attend = [&](const Tensor& x4, int64_t len, int pos) {
    ops::cached_attention_kv4(x4, l.k, l.k_params, l.v, l.v_params, len, pos, 0.1f);
  };
  refuses([&] { attend(q4, 0, 0); }, "no keys");
  refuses([&] { attend(q4, 9, 0); }, "valid_len");
  refuses([&] { attend(q4, 3, -1); }, "position_start");
  refuses([&] { attend(randn({1, 3, 3, 64}, 7), 3, 0); }, "num_heads % num_kv_heads");
  refuses([&] { attend(randn({2, 3, 4, 64}, 7), 3, 0); }, "shape mismatch");
  refuses([&] { attend(randn({1, 3, 4, 128}, 7), 3, 0); }, "shape mismatch");
  auto step = [&](int64_t T, int H, int pos) {
    const Tensor none;
    ops::decode_qkv_attention_kv4(randn({1, T, H * 64}, 1), randn({1, T, 128}, 2),
                                  randn({1, T, 128}, 3), H, 2, 64, none, none, 1e-6f, 1e4f, {}, pos,
                                  l.k, l.k_params, l.v, l.v_params, 0.1f);
  };
  refuses([&] { step(9, 4, 0); }, "out of cache bounds");
  refuses([&] { step(1, 4, 8); }, "out of cache bounds");
  refuses([&] { step(1, 3, 0); }, "num_heads % num_kv_heads");
  refuses([&] { step(1, 66, 0); }, "more than 32 heads");
  // an fp32 layer's tensors are not a 4-bit cache, and the other way round
  nn::KVLayer wide = nn::KVCache::allocate(1, 2, 64, 1, 8, kHIP0).layers[0];
  check(!wide.kv4() && l.kv4(), "kv4() tells the two apart");
  refuses([&] { ops::cached_attention(q4, l.k, l.v, 3, 0, 0.1f); }, "must be float32");
  refuses([&] { ops::cached_attention_kv4(q4, wide.k, l.k_params, wide.v, l.v_params, 3, 0, 0.1f); },
          "int32");
}

}  // namespace

int main() {
  auto run = [](const char* name, const std::function<void()>& f) {
    std::printf("%s\n", name);
    std::fflush(stdout);
    try {
      f();
    } catch (const std::exception& e) {
      check(false, std::string("unexpected exception: ") + e.what());
    }
  };
  run("Checkpoint8.Gradients", [] { checkpoint_gradients(false); });
  run("Checkpoint8.GradientsWithNorm", [] { checkpoint_gradients(true); });
  run("Quant.Refusals", [] { refusals(); });
  std::printf("%d failure(s)\n", g_failed);
  return g_failed;
}
