"""The few-bit stores as a model uses them: decode steps and prompts over a 4-bit KV cache
(attention op, model, generation, ctd_generate), and training with checkpoints in 8 bits."""
import ctypes as C
import json
import os
import subprocess

import numpy as np
import pytest

import oracle as O
from oracle import quant as OQ
from tests.helpers import assert_close, call, dev, empty, host, p

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from emberlm_amd import capi  # noqa: E402
from emberlm_amd import trainer as TR  # noqa: E402
from tests.test_gpu_infer import host_params, infer_cfg  # noqa: E402
from tests.test_gpu_model import layer_params, oracle_cfg, shapes  # noqa: E402
from tests.test_gpu_quant import attention_bounds, held_cache, same, words  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.cuda.init()


def rng(s=0):
    return np.random.default_rng(s)


def test_cpp_api_tests():
    exe = os.path.join(os.path.dirname(TR.LIB_PATH), "ctd_quant_tests")
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    print(r.stdout)
    assert r.returncode == 0 and "0 failure(s)" in r.stdout, r.stdout + r.stderr


# ----------------------------------------------------- decode step over a 4-bit cache
@pytest.mark.parametrize("B,T,H,Hk,D,pos,S,qk,factor", [
    (1, 1, 16, 8, 128, 4095, 4096, True, 0.0),   # split keys
    (1, 1, 16, 8, 128, 300, 512, True, 0.0),     # one workgroup per head
    (2, 3, 8, 2, 64, 17, 24, False, 32.0),       # llama3 frequencies
    (1, 2, 9, 3, 64, 0, 4, False, 0.0),          # the cache's first rows
    (1, 1, 3, 1, 64, 0, 1, True, 0.0),           # one row in all
    (1, 7, 4, 2, 128, 1018, 1030, True, 0.0),    # new rows in two blocks of one split
    (1, 8, 4, 2, 128, 1020, 1030, False, 0.0),   # new rows in two splits
    (1, 8, 8, 1, 64, 700, 710, True, 0.0),       # 64 rows a KV head: two row tiles write them
    (2, 4, 32, 1, 128, 130, 134, False, 0.0),    # group 32: four row tiles
    (1, 8, 32, 1, 64, 65600, 65608, False, 0.0), # the largest group over a long cache
    (300, 1, 4, 1, 64, 40, 41, False, 0.0),      # as many heads as fill the GPU
])
def test_decode_attention_kv4_fold(B, T, H, Hk, D, pos, S, qk, factor):
    r = rng(H * D + pos)
    theta, eps = 5e5, 1e-6
    q = r.standard_normal((B, T, H, D)).astype(np.float32)
    k, v = (r.standard_normal((B, T, Hk, D)).astype(np.float32) for _ in range(2))
    qn, kn = ((1 + 0.1 * r.standard_normal(D)).astype(np.float32) for _ in range(2))
    cache = held_cache(r, B, Hk, S, D)
    for _, par, _ in cache:
        par[:, :, pos:] = np.nan                    # rows that nothing may read as they are
    buf = [words(cache[0][0]), dev(cache[0][1]), words(cache[1][0]), dev(cache[1][1])]
    freqs = (C.c_float * (D // 2))()
    capi.check(capi.lib().ember_rope_freqs_host(freqs, D, theta, factor, 1.0, 4.0, 64))
    t = [dev(x) for x in (q, k, v, qn, kn)]
    scale = D ** -0.5
    need = capi.lib().ember_attn_kv4_workspace_bytes(B, T, H, Hk, D, pos + T)
    outs = []
    for _ in range(2):                              # the second call rewrites the same rows
        o = empty((B, T, H, D))
        ws = torch.full((max(4, need // 4),), float("nan"), device="cuda")
        call("ember_attn_kv4_qkv", *[p(x) for x in t[:3]], B, T, H, Hk, D,
             p(t[3]) if qk else None, p(t[4]) if qk else None, eps, freqs, pos,
             *[p(x) for x in buf], S, scale, p(o), p(ws) if need else None, need, None)
        outs.append(host(o))
    assert same(outs[0], outs[1])
    rope = dict(theta=theta, pos0=pos, factor=factor, low=1.0, high=4.0, orig=64)
    qr = O.rope(O.rmsnorm_fwd(q, qn, eps) if qk else q, **rope)
    kr = O.rope(O.rmsnorm_fwd(k, kn, eps) if qk else k, **rope).transpose(0, 2, 1, 3)
    new = slice(pos, pos + T)
    got = [(host(buf[0]).view(np.uint32), host(buf[1])), (host(buf[2]).view(np.uint32), host(buf[3]))]
    # values are quantised as they are: the rule's own bits
    codes, params = OQ.quantise(v.transpose(0, 2, 1, 3), 15)
    assert same(got[1][1][:, :, new], params)
    assert same(got[1][0][:, :, new], OQ.pack4(codes))
    # keys: within half a step of the 64-bit norm and rotation, whose fp32 form is off by its
    # roundings (1e-5 of the largest value: some tens of half-ulps)
    step = got[0][1][:, :, new, 1:].astype(np.float64)
    held = [OQ.values(OQ.unpack4(w), par) for w, par in got]
    assert (np.abs(held[0][:, :, new] - kr) <= 0.5 * step + 1e-5 * np.abs(kr).max()).all()
    lo = got[0][1][:, :, new, 0]
    assert (np.abs(lo - kr.min(-1)) <= 1e-5 * np.abs(kr).max()).all()
    for (w, par, _), (gw, gp) in zip(cache, got):   # the other rows as they were
        keep = np.ones(S, bool)
        keep[new] = False
        assert same(gp[:, :, keep], par[:, :, keep]) and same(gw[:, :, keep], w[:, :, keep])
    ref = OQ.attention(qr, held[0], held[1], pos, scale, pos + T)
    after = [(gw, gp, h) for (gw, gp), h in zip(got, held)]
    worst, _ = attention_bounds(qr, after, scale, pos + T)
    # the query's own roundings (1e-5 of it) move a score by at most that much of A
    vmax = np.abs(held[1][:, :, :pos + T]).max()
    a = scale * np.abs(qr).sum(-1).max() * (15 * got[0][1][:, :, :pos + T, 1] +
                                            np.abs(got[0][1][:, :, :pos + T, 0])).max()
    assert np.abs(outs[0] - ref).max() <= worst + vmax * np.expm1(2e-5 * a)


# --------------------------------------------------------------- a model over a 4-bit cache
def model_kv4(c, params, ids, quantised=True):
    """Logits of every position, in 64 bits, each query seeing the held form of its keys and values."""
    it = iter(params)
    emb = next(it).astype(np.float64)
    D, H, Hk, eps = c.head_dim, c.num_heads, c.num_kv_heads, c.rms_norm_eps
    B, T = ids.shape
    h = emb[ids]
    norm = lambda x, w: x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w  # noqa: E731
    rope = dict(theta=c.rope_theta, pos0=0, factor=c.rope_factor, low=c.rope_low_freq_factor,
                high=c.rope_high_freq_factor, orig=c.rope_original_max_pos)
    for _ in range(c.num_layers):
        n1, wq, wk, wv, wo = (next(it).astype(np.float64) for _ in range(5))
        qn, kn = (next(it), next(it)) if c.qk_norm else (None, None)
        n2, wg, wu, wd = (next(it).astype(np.float64) for _ in range(4))
        x = norm(h, n1)
        q, k, v = ((x @ w.T).reshape(B, T, -1, D) for w in (wq, wk, wv))
        if c.qk_norm:
            q, k = norm(q, qn), norm(k, kn)
        q, k = O.rope(q, **rope), O.rope(k, **rope)
        k, v = k.transpose(0, 2, 1, 3), v.transpose(0, 2, 1, 3)
        if quantised:
            k, v = (OQ.values(*OQ.quantise(y.astype(np.float32), 15)) for y in (k, v))
        a = OQ.attention(q, k, v, 0, D ** -0.5).reshape(B, T, H * D)
        h = h + a @ wo.T
        x = norm(h, n2)
        g = x @ wg.T
        h = h + (g / (1 + np.exp(-g)) * (x @ wu.T)) @ wd.T
    return norm(h, next(it)) @ emb.T


@pytest.mark.parametrize("variant", ["smollm2", "qwen3", "llama3", "d32"])
def test_model_over_kv4_cache(variant):
    """Prompt, chunks and single tokens over a 4-bit cache.  A key or value whose fp32 form lies on
    a border between two codes may take the other one (a step is 1/15 of a row's range, 4% of a row
    of 64 or more values, and one row among tens): 2e-3 of the logits' norm holds that, and what
    the 4 bits themselves change is over ten times more."""
    c = infer_cfg(variant)
    tr, params = host_params(c, 21)
    B, T = 2, 48
    ids = rng(22).integers(0, c.vocab_size, (B, T))
    ref = model_kv4(c, params, ids)
    exact = model_kv4(c, params, ids, quantised=False)
    assert np.linalg.norm(ref - exact) > 2e-2 * np.linalg.norm(exact)
    far = lambda a, b: np.linalg.norm(a - b) / np.linalg.norm(b)  # noqa: E731
    assert far(tr.forward(ids, tr.kv_cache(B, T, bits=4), 0), ref) <= 2e-3
    for cuts in ([30, 1, 1, 1, 4, 10, 1], [1] * 12 + [3] + [33], [11, 37]):
        cache, pos = tr.kv_cache(B, T + 3, bits=4), 0
        for n in cuts:
            out = tr.forward(ids[:, pos:pos + n], cache, pos)
            assert far(out, ref[:, pos:pos + n]) <= 2e-3, (cuts, pos)
            pos += n
            assert cache.current_len == pos
    with pytest.raises(TR.CtdError, match="out of cache bounds"):
        tr.forward(ids, tr.kv_cache(B, T - 1, bits=4), 0)
    tr.close()


def test_kv4_cache_memory_and_refusals():
    c = infer_cfg("qwen3")
    tr, _ = host_params(c, 3)
    before = TR.memory().allocated
    wide = tr.kv_cache(2, 4096)
    mid = TR.memory().allocated
    narrow = tr.kv_cache(2, 4096, bits=4)
    after = TR.memory().allocated
    rows = 2 * c.num_layers * 2 * c.num_kv_heads * 4096
    assert mid - before == rows * 4 * c.head_dim
    assert after - mid == rows * (c.head_dim // 2 + 8)
    wide.close(), narrow.close()
    for bits in (0, 3, 8, 16):
        with pytest.raises(TR.CtdError, match="bits"):
            tr.kv_cache(1, 8, bits=bits)
    with pytest.raises(TR.CtdError, match="bits"):
        tr.generate([1, 2], 3, kv_bits=8)
    tr.close()


def test_generation_over_kv4(tmp_path):
    """ctd_generate's loop with "kv_bits": 4 is greedy decoding over a 4-bit cache."""
    c = infer_cfg("qwen3")
    tr, params = host_params(c, 31, std=0.3)
    prompt = rng(4).integers(0, c.vocab_size, 23)
    n = 40
    toks, _, _ = tr.generate(prompt, n, kv_bits=4)
    cache = tr.kv_cache(1, 23 + n, bits=4)
    logits = tr.forward(prompt[None], cache, 0, last_only=True)[0, -1]
    for i in range(n):
        assert toks[i] == logits.argmax(), i
        logits = tr.forward(np.array([[toks[i]]]), cache, 23 + i, last_only=True)[0, -1]
    model = os.path.join(tmp_path, "m.safetensors")
    tr.save(model)
    tr.close()
    cfg = os.path.join(tmp_path, "model.json")
    with open(cfg, "w") as f:
        json.dump(dict(vocab_size=c.vocab_size, hidden_size=c.hidden_size,
                       intermediate_size=c.intermediate_size, num_hidden_layers=c.num_layers,
                       num_attention_heads=c.num_heads, num_key_value_heads=c.num_kv_heads,
                       head_dim=c.head_dim, rms_norm_eps=float(c.rms_norm_eps),
                       rope_theta=float(c.rope_theta), qk_norm=True), f)
    exe = os.path.join(os.path.dirname(TR.LIB_PATH), "ctd_generate")
    for temperature in (0.0, 0.7):
        req = dict(input_ids=[int(x) for x in prompt], max_new_tokens=n, temperature=temperature,
                   seed=5, max_seq_len=23 + n, kv_bits=4)
        r = subprocess.run([exe, "--model", model, "--config", cfg], input=json.dumps(req),
                           capture_output=True, text=True, timeout=60)
        assert r.returncode == 0, r.stderr
        got = [json.loads(x).get("token") for x in r.stdout.splitlines()][:-1]
        assert len(got) == n
        if temperature == 0.0:
            assert got == [int(x) for x in toks]


# --------------------------------------------------------------- checkpoints in 8 bits
def block_setup(qk_norm, seed):
    c = TR.make_config(vocab_size=64, hidden_size=192, intermediate_size=320, num_layers=1,
                       num_heads=4, num_kv_heads=2, head_dim=64, qk_norm=qk_norm,
                       rms_norm_eps=1e-5, rope_theta=1e4)
    tr = TR.Trainer(c, seed=seed, init_std=0.08, norm_value=1.0)
    r = rng(seed)
    B, T = 2, 50
    x = (r.standard_normal((B, T, 192)) * np.exp(r.standard_normal(192))).astype(np.float32)
    dy = r.standard_normal((B, T, 192)).astype(np.float32)
    codes, params = OQ.quantise_rows8(x.reshape(-1, 192))
    held = OQ.values_rows8(codes, params, 192).astype(np.float32).reshape(x.shape)
    return c, tr, x, dy, held


@pytest.mark.parametrize("qk_norm", [0, 1])
def test_block_gradients_at_the_restored_input(qk_norm):
    c, tr, x, dy, held = block_setup(qk_norm, 5)
    y, _ = tr.block_step(0, x, dy, checkpoint=True)
    tr.zero_grad()
    tr.set_checkpoint_bits(8)
    y8, dx8 = tr.block_step(0, x, dy, checkpoint=True)
    assert np.array_equal(y, y8)                    # the forward does not see the store
    lp = layer_params(tr, c, 0)
    g8 = {k: tr.get_grad(i) for k, (i, _) in lp.items()}
    tr.zero_grad()
    tr.set_checkpoint_bits(32)
    _, dx = tr.block_step(0, held, dy, checkpoint=True)
    assert_close(dx8, dx, rtol=1e-5, name="dx")     # the norm's sums round in another order
    for k, (i, _) in lp.items():
        assert_close(g8[k], tr.get_grad(i), rtol=1e-5, name=k)
    # the formula, in 64 bits
    w = {k: prm for k, (_, prm) in lp.items()}
    oc = oracle_cfg(c)
    rdx, rg = O.block_bwd(oc, w, held, dy)
    assert_close(dx8, rdx, name="dx vs oracle")
    for k in lp:
        assert_close(g8[k].reshape(np.asarray(rg[k]).shape), rg[k], name=k + " vs oracle")
    # and differences of the 64-bit forward along a direction: h^2 of its third derivative
    d = rng(9).standard_normal(x.shape)
    h = 1e-4
    f = lambda z: float((O.block_fwd(oc, w, z) * dy).sum())  # noqa: E731
    diff = (f(held + h * d) - f(held - h * d)) / (2 * h)
    assert abs(float((dx8 * d).sum()) - diff) <= 1e-4 * np.linalg.norm(dx8) * np.linalg.norm(d)
    tr.close()


def test_model_training_with_8_bit_checkpoints():
    """Same loss; gradients at the restored inputs.  A value is off by up to 1/510 of its group's
    range: with a range of six standard deviations 0.7% of one in the mean.  A gradient passes four
    blocks, each of which a relative error may enter two or three times over: 5% holds it."""
    c = TR.make_config(vocab_size=512, hidden_size=192, intermediate_size=320, num_layers=4,
                       num_heads=4, num_kv_heads=2, head_dim=64, qk_norm=1, rms_norm_eps=1e-5,
                       rope_theta=1e4)
    tr = TR.Trainer(c, seed=3, init_std=0.08, norm_value=1.0)
    tr.synthetic_batch(2, 257, seed=4)
    tr.set_checkpointing(True)
    loss = tr.forward_backward(True)
    g = [tr.get_grad(i) for i in range(tr.num_params())]
    tr.zero_grad()
    tr.set_checkpoint_bits(8)
    assert tr.forward_backward(True) == loss
    for i, ref in enumerate(g):
        rel = np.linalg.norm(tr.get_grad(i) - ref) / np.linalg.norm(ref)
        assert 0 < rel < 0.05 or i >= len(g) - 1, (tr.names[i], rel)
    again = [tr.get_grad(i) for i in range(tr.num_params())]
    tr.zero_grad()
    tr.forward_backward(True)
    assert all(np.array_equal(tr.get_grad(i), a) for i, a in enumerate(again))  # reproducible
    tr.set_checkpointing(False)                     # the bits are the checkpoints' alone
    tr.zero_grad()
    assert tr.forward_backward(True) == loss
    assert all(np.array_equal(tr.get_grad(i), a) for i, a in enumerate(g))
    with pytest.raises(TR.CtdError, match="32 or 8"):
        tr.set_checkpoint_bits(4)
    tr.close()


def test_8_bit_checkpoints_hold_less():
    c = TR.make_config(vocab_size=256, hidden_size=512, intermediate_size=512, num_layers=12,
                       num_heads=8, num_kv_heads=8, head_dim=64, rms_norm_eps=1e-5, rope_theta=1e4)
    tr = TR.Trainer(c, seed=3, init_std=0.05, norm_value=1.0)
    tr.synthetic_batch(2, 1024, seed=4)
    tr.set_checkpointing(True)
    peaks = {}
    for bits in (32, 8):
        tr.set_checkpoint_bits(bits)
        tr.forward_backward(False)
        TR.reset_peak_memory()
        tr.forward_backward(False)                  # the graph of the whole forward is recorded
        peaks[bits] = TR.memory().peak_allocated    # (a backward's peak is that of its gradients)
    saved = 4 * 2048 * 512                          # one block's input
    held = 2048 * (512 + 4 * 8)                     # the same in 8 bits
    # when the last block runs the inputs of at least 11 of the 12 are held
    assert peaks[32] - peaks[8] >= 10 * (saved - held), peaks
    tr.close()


def test_train_driver_with_8_bit_checkpoints(tmp_path):
    """ctd_train with "checkpoint_bits": 8: the first step's loss is the fp32 checkpoints' (the
    forward pass is the same), the later ones follow other gradients, and a resumed run ends with
    the same bits as one that was not stopped."""
    from tests.test_gpu_driver import make_run, read_st, tr_cfg
    tr = TR.Trainer(tr_cfg(), seed=3, init_std=0.05)
    init = tmp_path / "init.safetensors"
    tr.save(init)
    tr.close()
    r = rng(5)
    data = tmp_path / "data"
    data.mkdir()
    doc = r.integers(0, 1000, 49).astype(np.int32)  # every document, so that every batch is the same
    np.tile(doc, 6).tofile(data / "train.bin")
    np.ones(6 * 49, np.int8).tofile(data / "train_mask.bin")
    np.tile(doc, 2).tofile(data / "val.bin")
    np.ones(2 * 49, np.int8).tofile(data / "val_mask.bin")
    losses = {}
    for bits in (32, 8):
        run = make_run(tmp_path, f"bits{bits}", init, data, 4, checkpoint_bits=bits)
        TR.train_run(run / "config.json")
        lines = [json.loads(x) for x in (run / "loss.jsonl").read_text().splitlines()]
        losses[bits] = [x["loss"] for x in lines if "loss" in x]
        assert len(losses[bits]) >= 4 and np.isfinite(losses[bits]).all()
    assert losses[8][0] == losses[32][0] and losses[8] != losses[32]
    half = make_run(tmp_path, "resumed", init, data, 4, checkpoint_bits=8,
                    resume=tmp_path / "bits8" / "ckpt_step_2.safetensors")
    TR.train_run(half / "config.json")
    a, b = (read_st(tmp_path / n / "final.safetensors") for n in ("bits8", "resumed"))
    assert a.keys() == b.keys() and all(np.array_equal(a[k], b[k]) for k in a)


# ------------------------------------------------------------ captured, and at once
def step_buffers(r, B, H, Hk, D, S):
    cache = held_cache(r, B, Hk, S, D)
    return [words(cache[0][0]), dev(cache[0][1]), words(cache[1][0]), dev(cache[1][1])]


def test_captured_steps_replay_and_two_streams_at_once():
    """A captured run of the operators as a step uses them (a chunk written and attended to, a
    decode step on top, a checkpoint stored and restored), replayed between eager work, and the
    same eager calls on two streams at once, each with buffers of its own."""
    r = rng(12)
    B, T, H, Hk, D, S, pos = 1, 40, 8, 4, 128, 900, 700
    freqs = (C.c_float * (D // 2))()
    capi.check(capi.lib().ember_rope_freqs_host(freqs, D, 1e4, 0.0, 1.0, 4.0, 64))
    ins = [dev(r.standard_normal(s).astype(np.float32))
           for s in ((B, T, H, D), (B, T, Hk, D), (B, T, Hk, D), (B, 1, H, D), (B, 1, Hk, D),
                     (B, 1, Hk, D), (300, 640), (640,))]
    start = step_buffers(r, B, H, Hk, D, S)

    class Set:
        def __init__(self):
            self.cache = [t.clone() for t in start]
            self.o, self.o1 = empty((B, T, H, D)), empty((B, 1, H, D))
            n = [capi.lib().ember_attn_kv4_workspace_bytes(B, t, H, Hk, D, p)
                 for t, p in ((T, pos + T), (1, pos + T + 1))]
            assert n[0] and n[1]
            self.ws = [torch.full((x // 4,), float("nan"), device="cuda") for x in n]
            self.codes = torch.empty(capi.lib().ember_q8_code_bytes(300, 640), device="cuda",
                                     dtype=torch.uint8)
            self.params = empty((300, 5, 2))
            self.x, self.y, self.rstd = empty((300, 640)), empty((300, 640)), empty((300,))

        def run(self):
            st = C.c_void_p(torch.cuda.current_stream().cuda_stream)
            c = [p(t) for t in self.cache]
            capi.call("ember_kv4_write", p(ins[1]), p(ins[2]), *c, B, T, Hk, D, S, pos, st)
            capi.call("ember_attn_kv4", p(ins[0]), *c, p(self.o), B, T, H, Hk, D, pos + T, pos, S,
                      0.09, p(self.ws[0]), self.ws[0].numel() * 4, st)
            capi.call("ember_attn_kv4_qkv", p(ins[3]), p(ins[4]), p(ins[5]), B, 1, H, Hk, D, None,
                      None, 1e-6, freqs, pos + T, *c, S, 0.09, p(self.o1), p(self.ws[1]),
                      self.ws[1].numel() * 4, st)
            capi.call("ember_q8_quantize", p(ins[6]), p(self.codes), p(self.params), 300, 640, st)
            capi.call("ember_q8_dequantize_rmsnorm", p(self.codes), p(self.params), p(ins[7]),
                      p(self.x), p(self.y), p(self.rstd), 300, 640, 1e-5, st)

        def out(self):
            return [host(t) for t in (*self.cache, self.o, self.o1, self.codes, self.x, self.y,
                                      self.rstd)]

    def wipe(s):
        for t in (s.o, s.o1, s.x, s.y, s.rstd, *s.ws):
            t.zero_()
        for t, f in zip(s.cache, start):
            t.copy_(f)

    first = Set()
    first.run()
    want = first.out()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        first.run()
    other = Set()
    for _ in range(3):
        wipe(first)
        graph.replay()
        assert all(same(a, b) for a, b in zip(first.out(), want))
        wipe(other)
        other.run()
        assert all(same(a, b) for a, b in zip(other.out(), want))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    wipe(first), wipe(other)
    torch.cuda.synchronize()
    for _ in range(5):
        for s, stream in zip((first, other), streams):
            with torch.cuda.stream(stream):
                s.run()
    for s in (first, other):
        assert all(same(a, b) for a, b in zip(s.out(), want))
