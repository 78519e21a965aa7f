"""CPU checks of the few-bit stores: the oracle's own rule, and the refusals of the entry points
(no GPU compute is launched: every call here is rejected, or has nothing to do)."""
import ctypes as C
import json
import os
import subprocess

import numpy as np
import pytest

from emberlm_amd import capi
from emberlm_amd import trainer as TR
from oracle import quant as OQ

P = C.c_void_p(4096)      # never dereferenced
ODD = C.c_void_p(4096 + 4)  # not 8-byte aligned
HALF = C.c_void_p(4096 + 8)  # 8-byte but not 16-byte aligned


@pytest.mark.parametrize("top", [15, 255])
def test_oracle_reads_back_within_half_a_step(top):
    r = np.random.default_rng(top)
    x = (r.standard_normal((200, 128)) * np.exp(3 * r.standard_normal((200, 1)))).astype(np.float32)
    codes, params = OQ.quantise(x, top)
    assert codes.max() == top and codes.min() == 0
    err = np.abs(OQ.values(codes, params) - x)
    # half a step, and the rounding of step (2^-24 of it) times a code of up to `top`
    step = params[:, 1:].astype(np.float64)
    assert (err <= step * (0.5 + top * 2.0 ** -24)).all()


def test_oracle_of_equal_and_not_finite_groups():
    x = np.full((3, 16), 1.25, np.float32)
    x[1, 3], x[2, 0] = np.inf, np.nan
    codes, params = OQ.quantise(x, 15)
    assert not codes.any() and tuple(params[0]) == (1.25, 0.0) and np.isnan(params[1:]).all()


def test_oracle_packs_the_first_code_lowest():
    c = np.arange(16, dtype=np.uint32)
    assert [hex(w) for w in OQ.pack4(c)] == ["0x76543210", "0xfedcba98"]
    assert np.array_equal(OQ.unpack4(OQ.pack4(c)), c)


def kv4_write(B=1, T=2, Hk=2, D=64, S=8, pos=0, k=P, v=P, kc=P, kp=P, vc=P, vp=P):
    return capi.lib().ember_kv4_write(k, v, kc, kp, vc, vp, B, T, Hk, D, S, pos, None)


def test_write_refusals():
    assert kv4_write(pos=7) == -1 and kv4_write(pos=-1) == -1 and kv4_write(T=9) == -1
    assert kv4_write(B=-1) == -1 and kv4_write(T=-1) == -1 and kv4_write(Hk=-1) == -1
    for D in (0, 4, 12, 60, 264, -8):
        assert kv4_write(D=D) == -1, D
    assert kv4_write(pos=2 ** 62, T=2 ** 62) == -1
    for name in ("k", "v", "kc", "kp", "vc", "vp"):
        assert kv4_write(**{name: None}) == -1, name
        assert kv4_write(**{name: ODD}) == -3, name
    for name in ("k", "v", "kc", "vc"):
        assert kv4_write(**{name: HALF}) == -3, name
    assert kv4_write(B=0) == 0 and kv4_write(T=0, pos=8) == 0


def kv4_read(B=1, Hk=2, group=2, L=4, D=64, S=8, c=P, p=P, o=P):
    return capi.lib().ember_kv4_read_expanded(c, p, o, B, Hk, group, L, D, S, None)


def test_read_refusals():
    assert kv4_read(L=9) == -1 and kv4_read(L=-1) == -1 and kv4_read(group=0) == -1
    assert kv4_read(B=-1) == -1 and kv4_read(D=68) == -1 and kv4_read(D=512) == -1
    assert kv4_read(c=None) == -1 and kv4_read(p=None) == -1 and kv4_read(o=None) == -1
    assert kv4_read(c=HALF) == -3 and kv4_read(o=HALF) == -3 and kv4_read(p=ODD) == -3
    assert kv4_read(L=0) == 0 and kv4_read(B=0) == 0


def attn(B=1, T=1, H=4, Hk=2, D=64, L=4, pos=3, S=8, q=P, kc=P, kp=P, vc=P, vp=P, o=P, ws=None,
         wsb=0):
    return capi.lib().ember_attn_kv4(q, kc, kp, vc, vp, o, B, T, H, Hk, D, L, pos, S, 1.0, ws,
                                     wsb, None)


def test_attention_refusals():
    assert attn(D=96) == -1 and attn(H=3) == -1 and attn(Hk=0) == -1 and attn(pos=-1) == -1
    assert attn(L=0) == -1 and attn(L=9) == -1 and attn(S=2 ** 30 + 1, L=4) == -1
    assert attn(pos=2 ** 30 + 1) == -1 and attn(pos=2 ** 63 - 1) == -1
    assert attn(B=-1) == -1 and attn(T=-1) == -1 and attn(T=2 ** 30 + 1) == -1
    assert attn(B=2 ** 20, T=2 ** 10, H=4) == -1  # 2^32 query rows
    for name in ("q", "kc", "kp", "vc", "vp", "o"):
        assert attn(**{name: None}) == -1, name
        assert attn(**{name: ODD}) == -3, name
    assert attn(B=0) == 0 and attn(T=0) == 0
    # a long key range is split, and needs the workspace it asks for
    need = capi.lib().ember_attn_kv4_workspace_bytes(1, 1, 4, 2, 64, 4096)
    assert need > 0 and need % 16 == 0
    assert attn(L=4096, pos=4095, S=4096) == -2
    assert attn(L=4096, pos=4095, S=4096, ws=P, wsb=need - 1) == -2
    assert attn(L=4096, pos=4095, S=4096, ws=ODD, wsb=need) == -3
    assert capi.lib().ember_attn_kv4_workspace_bytes(1, 1, 4, 2, 64, 32) == 0
    assert capi.lib().ember_attn_kv4_workspace_bytes(1, 1, 4, 3, 64, 4096) == 0


def test_attention_of_more_workgroups_than_a_launch_holds():
    assert attn(B=2 ** 23, H=1, Hk=1, pos=0) == -1  # eight waves per head, 2^32 threads
    assert attn(B=2 ** 23, H=32, Hk=1, pos=0) == -1  # two tiles of 16 rows per workgroup


def test_decode_step_refusals():
    f = (C.c_float * 64)()

    def step(T=1, H=4, Hk=2, D=64, pos=0, S=8, B=1, freqs=f, **ptr):
        a = {n: ptr.get(n, P) for n in ("q", "k", "v", "qn", "kn", "kc", "kp", "vc", "vp", "o")}
        return capi.lib().ember_attn_kv4_qkv(
            a["q"], a["k"], a["v"], B, T, H, Hk, D, a["qn"], a["kn"], 1e-6, freqs, pos, a["kc"],
            a["kp"], a["vc"], a["vp"], S, 1.0, a["o"], None, 0, None)

    assert step(T=2, pos=7) == -1 and step(T=9, S=16) == -1 and step(pos=-1) == -1
    assert step(D=96) == -1 and step(H=3) == -1 and step(H=66) == -1 and step(freqs=None) == -1
    assert step(S=2 ** 30 + 1) == -1 and step(B=-1) == -1 and step(pos=2 ** 63 - 1) == -1
    for name in ("q", "k", "v", "kc", "kp", "vc", "vp", "o"):
        assert step(**{name: None}) == -1, name
        assert step(**{name: ODD}) == -3, name
    assert step(qn=HALF) == -3 and step(kn=HALF) == -3
    assert step(B=0) == 0 and step(T=0) == 0
    assert step(pos=4000, S=4096) == -2  # split keys, no workspace


@pytest.mark.parametrize("req,msg", [('"kv_bits": 8', "kv_bits must be 32 or 4"),
                                     ('"kv_bits": "4"', "kv_bits must be an integer")])
def test_generate_request_with_other_bits(req, msg):
    exe = os.path.join(os.path.dirname(TR.LIB_PATH), "ctd_generate")
    r = subprocess.run([exe, "--model", "/nonexistent.safetensors"],
                       input='{"input_ids": [1], %s}' % req, capture_output=True, text=True,
                       timeout=60)
    assert r.returncode == 1 and msg in json.loads(r.stdout)["error"]


@pytest.mark.parametrize("extra", ['"checkpoint_bits": 4, "gradient_checkpointing": true',
                                   '"checkpoint_bits": 8'])
def test_train_config_with_other_bits(tmp_path, extra):
    cfg = tmp_path / "config.json"
    cfg.write_text('{"init_weights": "w", "data_dir": "d", %s}' % extra)
    with pytest.raises(TR.CtdError, match="checkpoint_bits"):
        TR.train_run(cfg)


def test_rows8_refusals_and_sizes():
    lib = capi.lib()
    assert lib.ember_q8_code_bytes(3, 1001) == 3 * 1008 and lib.ember_q8_code_bytes(3, 0) == 0
    assert lib.ember_q8_param_bytes(3, 1001) == 3 * 8 * 8 and lib.ember_q8_param_bytes(3, 128) == 24
    q = lambda x, c, p, rows, H: lib.ember_q8_quantize(x, c, p, rows, H, None)  # noqa: E731
    d = lambda c, p, x, rows, H: lib.ember_q8_dequantize(c, p, x, rows, H, None)  # noqa: E731
    n = lambda c=P, p=P, w=P, x=P, y=P, r=P, rows=2, H=64: (  # noqa: E731
        lib.ember_q8_dequantize_rmsnorm(c, p, w, x, y, r, rows, H, 1e-6, None))
    assert q(P, P, P, -1, 4) == -1 and d(P, P, P, 4, -1) == -1 and n(rows=-1) == -1
    assert q(None, P, P, 1, 4) == -1 and q(P, None, P, 1, 4) == -1 and q(P, P, None, 1, 4) == -1
    assert d(None, P, P, 1, 4) == -1 and d(P, None, P, 1, 4) == -1 and d(P, P, None, 1, 4) == -1
    for name in ("c", "p", "w", "x", "y"):
        assert n(**{name: None}) == -1, name
    assert q(P, HALF, P, 1, 4) == -3 and q(P, P, ODD, 1, 4) == -3
    assert d(HALF, P, P, 1, 4) == -3 and n(c=HALF) == -3 and n(p=ODD) == -3
    assert q(None, None, None, 0, 4) == 0 and d(None, None, None, 4, 0) == 0 and n(rows=0) == 0
    assert n(rows=2 ** 31) == -1 and d(P, P, P, 2 ** 31, 4) == -1
