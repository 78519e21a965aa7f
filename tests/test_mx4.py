"""CPU checks of the 4-bit weights: the rule in 64 bits and the refusals of the entry points."""
import ctypes as C
import json
import os
import subprocess

import numpy as np
import pytest

from emberlm_amd import capi
from emberlm_amd import trainer as TR
from oracle import mx4 as OM

P = C.c_void_p(4096)  # never dereferenced
ODD = C.c_void_p(4100)


def test_rule_by_distances():
    """Every value lies nearest to its own code, and no smaller scale would reach."""
    r = np.random.default_rng(0)
    w = (r.standard_normal((50, 70)) * np.exp(2 * r.standard_normal((50, 1)))).astype(np.float32)
    codes, scales = OM.quantise(w)
    v = OM.values(codes, scales)
    s = np.repeat(np.ldexp(1.0, scales.astype(int) - 127), 32, 1)[:, :70]
    all_values = np.concatenate([OM.SIZES, -OM.SIZES])
    best = np.abs(w[..., None].astype(np.float64) - s[..., None] * all_values).min(-1)
    assert np.array_equal(np.abs(w - v), best)
    # half a step everywhere: 1/4 below 2, 1/2 below 4, 1 up to 7
    q = np.abs(w) / s
    assert (np.abs(w - v) <= s * np.where(q < 2, 0.25, np.where(q < 4, 0.5, 1.0))).all()
    for a in range(0, 70, 32):
        assert (np.abs(w[:, a:a + 32]).max(1) > 7 * s[:, a] / 2).all()


@pytest.mark.parametrize("x,code", [(0.25, 0), (0.2500001, 1), (0.75, 2), (1.25, 2), (1.75, 4),
                                    (2.5, 4), (2.5000002, 5), (3.5, 6), (5.0, 6), (5.000001, 7),
                                    (6.5, 7), (7.0, 7), (-0.25, 8), (-5.0, 14)])
def test_borders_go_to_the_even_code(x, code):
    codes, scales = OM.quantise(np.array([[x, 7.0]], np.float32))
    assert scales[0, 0] == 127 and codes[0, 0] == code


@pytest.mark.parametrize("top,byte", [(7.0, 127), (7.000001, 128), (3.5, 126), (3.6, 127),
                                      (0.0, 0), (2.0 ** -149, 0), (7 * 2.0 ** -127, 0),
                                      (7.1 * 2.0 ** -127, 1), (1.7e38, 252), (np.inf, 255),
                                      (np.nan, 255)])
def test_scale_byte(top, byte):
    assert OM.quantise(np.array([[top, 0.0]], np.float32))[1][0, 0] == byte


def test_form_in_memory():
    codes = np.arange(33 * 100, dtype=np.uint32).reshape(33, 100).astype(np.uint8) % 16
    scales = np.arange(33 * 4, dtype=np.uint8).reshape(33, 4)
    c, s = OM.pack(codes, scales)
    lib = capi.lib()
    assert c.size == lib.ember_mx4_code_bytes(33, 100) == 2 * 2 * 1024
    assert s.size == lib.ember_mx4_scale_bytes(33, 100) == 2 * 256
    for n, k in ((0, 0), (31, 63), (32, 64), (5, 37), (32, 99)):
        tile, h, i = (n // 32) * 2 + k // 64, k // 32 % 2, k % 32
        byte = c[tile * 1024 + 16 * (32 * h + n % 32) + i // 2]
        assert (byte >> 4 * (i % 2) & 15) == codes[n, k]
        assert s[(n // 32) * 256 + 4 * (32 * h + n % 32) + k // 64] == scales[n, k // 32]


def _linear(M=1, K=64, N=(8,), x=P, codes=P, scales=P, y=P, res=None, norm=None, ws=P, need=None,
            nseg=None):
    lib, n = capi.lib(), len(N)
    ptrs = lambda v: (C.c_void_p * n)(*[v.value if v else None] * n)  # noqa: E731
    room = lib.ember_mx4_workspace_bytes(M, K, sum(N)) if need is None else need
    return lib.ember_mx4_linear(x, M, K, norm, 1e-5, n if nseg is None else nseg, ptrs(codes),
                                ptrs(scales), (C.c_int64 * n)(*N), ptrs(y), res, ws, room, None)


def _gateup(M=1, K=64, N=8, x=P, codes=P, scales=P, out=P, ws=P, need=None):
    lib = capi.lib()
    room = lib.ember_mx4_workspace_bytes(M, K, 2 * N) if need is None else need
    return lib.ember_mx4_gateup(x, M, K, None, 1e-5, codes, scales, codes, scales, N, out, ws, room,
                                None)


def test_sizes_are_refused():
    lib = capi.lib()
    for N, K in ((-1, 64), (2 ** 31, 64), (8, 0), (8, -64), (8, 2 ** 30 + 1), (8, 2 ** 62),
                 (2 ** 62, 2 ** 62)):
        assert lib.ember_mx4_code_bytes(N, K) == 0 and lib.ember_mx4_scale_bytes(N, K) == 0
        assert lib.ember_mx4_quantize(P, P, P, N, K, None) == -1
        assert lib.ember_mx4_dequantize(P, P, P, N, K, None) == -1
        assert lib.ember_mx4_embedding(P, P, P, P, 4, K, N, None) == -1
        assert _linear(K=K, N=(N,), need=0) == -1 and _linear(K=K, N=(8, N), need=0) == -1
        assert _gateup(K=K, N=N, need=0) == -1
    for M in (-1, 2 ** 31, 2 ** 62):
        assert _linear(M=M, need=2 ** 62) == -1 and _gateup(M=M, need=2 ** 62) == -1
        assert lib.ember_mx4_embedding(P, P, P, P, M, 64, 8, None) == -1
        assert lib.ember_mx4_workspace_bytes(M, 64, 64) == 0
    assert _linear(N=(0,)) == -1 and _gateup(N=0) == -1
    # more threads than a launch holds
    assert _gateup(M=0, N=2 ** 27) == 0 and _gateup(M=0, N=2 ** 27 + 1) == -1
    assert _linear(M=1, K=2049, N=(2 ** 31 - 1,)) == -1
    for n in (0, 4, -1):
        assert _linear(nseg=n) == -1
    assert lib.ember_mx4_code_bytes(2 ** 31 - 1, 2 ** 30) == 2 ** 26 * 2 ** 24 * 1024


def test_nothing_to_do_is_done():
    lib = capi.lib()
    assert lib.ember_mx4_quantize(None, None, None, 0, 64, None) == 0
    assert lib.ember_mx4_dequantize(None, None, None, 0, 64, None) == 0
    assert lib.ember_mx4_embedding(None, None, None, None, 0, 64, 8, None) == 0
    assert _linear(M=0, x=None, codes=None, scales=None, y=None, ws=None) == 0
    assert _gateup(M=0, x=None, codes=None, scales=None, out=None, ws=None) == 0


def test_pointers_are_refused():
    lib = capi.lib()
    for bad in (dict(x=None), dict(codes=None), dict(scales=None), dict(y=None)):
        assert _linear(**bad) == -1
    for bad in (dict(x=None), dict(codes=None), dict(scales=None), dict(out=None)):
        assert _gateup(**bad) == -1
    assert _linear(codes=ODD) == -3 and _linear(scales=ODD) == -3
    assert _gateup(codes=ODD) == -3 and _gateup(scales=ODD) == -3
    for a, b in ((None, P), (P, None)):
        assert lib.ember_mx4_quantize(P, a, b, 8, 64, None) == -1
        assert lib.ember_mx4_embedding(P, a, b, P, 4, 64, 8, None) == -1
    for a, b in ((ODD, P), (P, ODD)):
        assert lib.ember_mx4_quantize(P, a, b, 8, 64, None) == -3
        assert lib.ember_mx4_dequantize(a, b, P, 8, 64, None) == -3
        assert lib.ember_mx4_embedding(P, a, b, P, 4, 64, 8, None) == -3
    assert lib.ember_mx4_quantize(None, P, P, 8, 64, None) == -1
    assert lib.ember_mx4_dequantize(P, P, None, 8, 64, None) == -1
    assert lib.ember_mx4_embedding(None, P, P, P, 4, 64, 8, None) == -1
    assert lib.ember_mx4_embedding(P, P, P, None, 4, 64, 8, None) == -1


@pytest.mark.parametrize("M", [1, 8, 9, 100, 4096])
def test_workspace_is_asked_for(M):
    need = capi.lib().ember_mx4_workspace_bytes(M, 2048, 64)
    if need:
        assert _linear(M=M, K=2048, N=(64,), need=need - 1) == -2
        assert _linear(M=M, K=2048, N=(64,), ws=None) == -2
        assert _linear(M=M, K=2048, N=(64,), ws=ODD) == -3
        assert _gateup(M=M, K=2048, N=32, need=need - 1) == -2
        assert _gateup(M=M, K=2048, N=32, ws=None) == -2
        assert _gateup(M=M, K=2048, N=32, ws=ODD) == -3


def _generate(request):
    exe = os.path.join(os.path.dirname(TR.LIB_PATH), "ctd_generate")
    r = subprocess.run([exe, "--model", "/nonexistent.safetensors"],
                       input='{"input_ids": [1], %s}' % request, capture_output=True, text=True,
                       timeout=60)
    assert r.returncode == 1
    return json.loads(r.stdout)["error"]


@pytest.mark.parametrize("bits", ["4.5", "32.25", str(2 ** 32 + 4), "-4", "0", "8", "16"])
@pytest.mark.parametrize("key", ["weight_bits", "embedding_bits"])
def test_bits_of_a_request_are_32_or_4(key, bits):
    assert key + " must be 32 or 4" in _generate('"%s": %s' % (key, bits))


def test_bits_of_a_request_that_are_taken():
    """The request passes; what fails then is the model file."""
    for request in ('"weight_bits": 4', '"weight_bits": 32, "embedding_bits": 32',
                    '"weight_bits": 4.0, "embedding_bits": 4', '"weight_bits": 4, "kv_bits": 4'):
        assert "bits" not in _generate(request)
    assert "needs weight_bits 4" in _generate('"embedding_bits": 4')
