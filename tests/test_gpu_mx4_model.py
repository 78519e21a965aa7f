"""Weights in 4 bits as a model uses them: prompts, cached decode steps, losses, generation and
ctd_generate, against the fp32 model that holds the same values."""
import json
import os
import subprocess

import numpy as np
import pytest

from oracle import mx4 as OM

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from emberlm_amd import trainer as TR  # noqa: E402
from tests.test_gpu_infer import host_params, infer_cfg  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.cuda.init()


def rng(s=0):
    return np.random.default_rng(s)


def far(a, b):
    return np.linalg.norm(a.astype(np.float64) - b) / np.linalg.norm(b)


def read_back(a):
    return OM.values(*OM.quantise(a)).astype(np.float32)


def pair(c, seed, table, std=0.2):
    """A model with weights in 4 bits, and the fp32 model whose weights are what those read back as."""
    held, params = host_params(c, seed, std)
    plain, _ = host_params(c, seed, std)
    for i, (name, a) in enumerate(zip(plain.names, params)):
        if name.endswith("proj.weight") or (table and name == "model.embed_tokens.weight"):
            plain.set_param(i, read_back(a))
    held.quantize_weights(table)
    return held, plain


# Logits of two fp32 forwards that sum in other orders agree to 1e-4 of their norm (the bound that the
# framework's model tests have for them); 4-bit weights alone change them by 10% and more.
RTOL = 1e-4


@pytest.mark.parametrize("variant", ["smollm2", "qwen3", "llama3", "d32"])
@pytest.mark.parametrize("table", [False, True])
def test_forward_and_cached_steps(variant, table):
    c = infer_cfg(variant)
    held, plain = pair(c, 41, table)
    first, _ = host_params(c, 41)
    B, T = 2, 48
    ids = rng(42).integers(0, c.vocab_size, (B, T))
    want = plain.forward(ids)
    assert far(first.forward(ids), want) > 0.02
    assert far(held.forward(ids), want) <= RTOL
    assert far(held.forward(ids, last_only=True), want[:, -1:]) <= RTOL
    for cuts in ([30, 1, 1, 1, 4, 10, 1], [1] * 12 + [3] + [33], [11, 37]):
        cache, pos = held.kv_cache(B, T), 0
        for n in cuts:
            out = held.forward(ids[:, pos:pos + n], cache, pos)
            assert far(out, want[:, pos:pos + n]) <= RTOL, (cuts, pos)
            pos += n
    for t in (held, plain, first):
        t.close()


@pytest.mark.parametrize("variant", ["qwen3", "d32"])
def test_over_a_4_bit_cache(variant):
    """Both few-bit stores at once.  A cached value near a border between two codes may take the other
    one where its fp32 form differs by a rounding: 2e-3, as for the cache alone."""
    c = infer_cfg(variant)
    held, plain = pair(c, 43, True)
    ids = rng(44).integers(0, c.vocab_size, (2, 40))
    a, b = held.kv_cache(2, 40, bits=4), plain.kv_cache(2, 40, bits=4)
    pos = 0
    for n in (29, 1, 1, 7, 2):
        x = ids[:, pos:pos + n]
        assert far(held.forward(x, a, pos), plain.forward(x, b, pos)) <= 2e-3, pos
        pos += n
    held.close(), plain.close()


@pytest.mark.parametrize("B", [1, 8, 9])
def test_batches_of_last_logits(B):
    c = infer_cfg("llama3")
    held, plain = pair(c, 45, True)
    ids = rng(B).integers(0, c.vocab_size, (B, 5))
    assert far(held.forward(ids, last_only=True), plain.forward(ids, last_only=True)) <= RTOL
    held.close(), plain.close()


@pytest.mark.parametrize("table", [False, True])
def test_losses(table):
    c = infer_cfg("qwen3")
    held, plain = pair(c, 46, table)
    r = rng(47)
    ids, tgt = (r.integers(0, c.vocab_size, (2, 33)) for _ in range(2))
    mask = (r.random((2, 33)) < 0.7).astype(np.float32)
    for t in (held, plain):
        t.set_batch(ids, tgt, mask)
    a, b = held.forward_backward(False), plain.forward_backward(False)
    assert abs(a - b) <= RTOL * abs(b)
    held.set_checkpointing(True)
    assert held.forward_backward(False) == a
    with pytest.raises(TR.CtdError):
        held.forward_backward(True)
    held.close(), plain.close()


def test_what_needs_parameters_is_refused(tmp_path):
    c = infer_cfg("qwen3")
    tr, _ = host_params(c, 48)
    ids = rng(1).integers(0, c.vocab_size, (1, 9))
    tr.set_batch(ids, ids)
    tr.make_optimizer(offload=True)
    tr.set_checkpointing(True)
    tr.train_step()
    tr.quantize_weights()
    x = np.zeros((1, 2, c.hidden_size), np.float32)
    for call in (lambda: tr.make_optimizer(), lambda: tr.save(tmp_path / "m"), lambda: tr.opt_step(),
                 lambda: tr.load(tmp_path / "m"), lambda: tr.train_step(),
                 lambda: tr.block_step(0, x, x)):
        with pytest.raises(TR.CtdError):
            call()
    assert not os.path.exists(tmp_path / "m")
    assert np.isfinite(tr.forward(ids)).all()
    tr.close()


def test_memory():
    c = TR.make_config(vocab_size=512, hidden_size=512, intermediate_size=1024, num_layers=4,
                       num_heads=4, num_kv_heads=2, head_dim=128, rms_norm_eps=1e-5, rope_theta=1e4)
    tr = TR.Trainer(c, seed=0)
    proj = 4 * (512 * (512 + 256 + 256 + 512) + 3 * 512 * 1024)
    before = TR.memory().allocated
    tr.quantize_weights()
    mid = TR.memory().allocated
    assert before - mid == proj * 4 - proj * 17 // 32
    tr.quantize_weights(table=True)
    assert mid - TR.memory().allocated == 512 * 512 * 4 - 512 * 512 * 17 // 32
    tr.close()


@pytest.mark.parametrize("table,kv", [(False, 32), (True, 32), (True, 4)])
def test_generation_and_the_tool(tmp_path, table, kv):
    """ctd_generate's loop is greedy decoding on the 4-bit weights; the tool gives its tokens."""
    c = infer_cfg("qwen3")
    tr, _ = host_params(c, 49, std=0.3)
    model = os.path.join(tmp_path, "m.safetensors")
    tr.save(model)
    tr.quantize_weights(table)
    prompt = rng(4).integers(0, c.vocab_size, 23)
    n = 40
    toks, _, _ = tr.generate(prompt, n, kv_bits=kv)
    cache = tr.kv_cache(1, 23 + n, bits=kv)
    logits = tr.forward(prompt[None], cache, 0, last_only=True)[0, -1]
    for i in range(n):
        assert toks[i] == logits.argmax(), i
        logits = tr.forward(np.array([[toks[i]]]), cache, 23 + i, last_only=True)[0, -1]
    tr.close()
    cfg = os.path.join(tmp_path, "model.json")
    with open(cfg, "w") as f:
        json.dump(dict(vocab_size=c.vocab_size, hidden_size=c.hidden_size,
                       intermediate_size=c.intermediate_size, num_hidden_layers=c.num_layers,
                       num_attention_heads=c.num_heads, num_key_value_heads=c.num_kv_heads,
                       head_dim=c.head_dim, rms_norm_eps=float(c.rms_norm_eps),
                       rope_theta=float(c.rope_theta), qk_norm=True), f)
    exe = os.path.join(os.path.dirname(TR.LIB_PATH), "ctd_generate")
    req = dict(input_ids=[int(x) for x in prompt], max_new_tokens=n, temperature=0.0,
               max_seq_len=23 + n, kv_bits=kv, weight_bits=4, embedding_bits=4 if table else 32)
    r = subprocess.run([exe, "--model", model, "--config", cfg], input=json.dumps(req),
                       capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr
    got = [json.loads(x).get("token") for x in r.stdout.splitlines()][:-1]
    assert got == [int(x) for x in toks]


def test_cpp_api_tests():
    exe = os.path.join(os.path.dirname(TR.LIB_PATH), "ctd_mx4_tests")
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    print(r.stdout)
    assert r.returncode == 0 and "0 failure(s)" in r.stdout, r.stdout + r.stderr
