"""CPU checks of what the few-bit stores' entry points refuse: sizes that one of a pair of calls
would take and the other not, that pass 64 bits, and bits that are not whole numbers."""
import ctypes as C
import json
import os
import subprocess

import pytest

from emberlm_amd import capi
from emberlm_amd import trainer as TR

P = C.c_void_p(4096)  # never dereferenced


def test_rows_that_could_not_be_restored_are_not_quantised():
    lib = capi.lib()
    for rows in (2 ** 31, 2 ** 40):
        assert lib.ember_q8_quantize(P, P, P, rows, 4, None) == -1
        assert lib.ember_q8_dequantize(P, P, P, rows, 4, None) == -1
        assert lib.ember_q8_dequantize_rmsnorm(P, P, P, P, P, P, rows, 4, 1e-6, None) == -1


def test_sizes_that_pass_64_bits():
    """Their products would wrap round, some of them to 0 or to a size that looks right."""
    lib = capi.lib()
    big = 2 ** 32

    def write(B, T, Hk, S, D=64):
        return lib.ember_kv4_write(P, P, P, P, P, P, B, T, Hk, D, S, 0, None)

    def read(B, Hk, group, L, S, D=64):
        return lib.ember_kv4_read_expanded(P, P, P, B, Hk, group, L, D, S, None)

    def attn(B, T, H, Hk, L, S):
        return lib.ember_attn_kv4(P, P, P, P, P, P, B, T, H, Hk, 64, L, 0, S, 1.0, P, 2 ** 62, None)

    def step(B, T, H, Hk, S):
        f = (C.c_float * 64)()
        return lib.ember_attn_kv4_qkv(P, P, P, B, T, H, Hk, 64, None, None, 1e-6, f, 0, P, P, P, P,
                                      S, 1.0, P, P, 2 ** 62, None)

    assert write(big, big, 1, big) == -1 and write(2 ** 61, 1, 8, 1) == -1
    assert write(2, 1, 1, 2 ** 62) == -1
    assert read(big, big, 1, 1, 1) == -1 and read(1, 1, 2 ** 62, 4, 4) == -1
    assert read(2, 1, 1, 1, 2 ** 62) == -1
    for n in (2 ** 62, 2 ** 61 + 1, 2 ** 60, 2 ** 57):
        assert attn(n, 1, 8, 8, 4, 4) == -1 and attn(1, 4, n, n, 4, 4) == -1, n
        assert attn(1, 4, n, 1, 4, 4) == -1 and step(n, 1, 8, 8, 4) == -1, n
        assert lib.ember_attn_kv4_workspace_bytes(n, 4, 8, 8, 64, 4096) == 0
        assert lib.ember_attn_kv4_workspace_bytes(1, 4, 8, 8, n, 2 ** 20) == 0
    for H in (2 ** 63 - 1, 2 ** 62, 2 ** 61):
        assert lib.ember_q8_quantize(P, P, P, 2, H, None) == -1, H
        assert lib.ember_q8_dequantize(P, P, P, 2, H, None) == -1, H
        assert lib.ember_q8_dequantize_rmsnorm(P, P, P, P, P, P, 2, H, 1e-6, None) == -1, H
        assert lib.ember_q8_code_bytes(2, H) == 0 and lib.ember_q8_param_bytes(2, H) == 0, H
    # nothing to do is still nothing to do, whatever the other sizes
    assert write(0, 1, 8, 2 ** 62) == 0 and read(0, 1, 1, 1, 2 ** 62) == 0
    assert lib.ember_q8_quantize(P, P, P, 0, 2 ** 63 - 1, None) == 0


@pytest.mark.parametrize("bits", ["4.5", "32.25", str(2 ** 32 + 4), "-4", "0"])
def test_kv_bits_are_32_or_4_and_nothing_that_rounds_to_them(bits):
    exe = os.path.join(os.path.dirname(TR.LIB_PATH), "ctd_generate")
    r = subprocess.run([exe, "--model", "/nonexistent.safetensors"],
                       input='{"input_ids": [1], "kv_bits": %s}' % bits, capture_output=True,
                       text=True, timeout=60)
    assert r.returncode == 1 and "kv_bits must be 32 or 4" in json.loads(r.stdout)["error"]


@pytest.mark.parametrize("bits", ["8.5", "32.25", str(2 ** 32 + 8), "-8", '"8"'])
def test_checkpoint_bits_are_32_or_8_and_nothing_that_rounds_to_them(tmp_path, bits):
    cfg = tmp_path / "config.json"
    cfg.write_text('{"init_weights": "w", "data_dir": "d", "gradient_checkpointing": true, '
                   '"checkpoint_bits": %s}' % bits)
    with pytest.raises(TR.CtdError, match="checkpoint_bits must be 32, or 8"):
        TR.train_run(cfg)


@pytest.mark.parametrize("bits", ["32", "4", "4.0", "3.2e1"])
def test_kv_bits_that_are_taken(bits):
    """The request passes; what fails then is the model file."""
    exe = os.path.join(os.path.dirname(TR.LIB_PATH), "ctd_generate")
    r = subprocess.run([exe, "--model", "/nonexistent.safetensors"],
                       input='{"input_ids": [1], "kv_bits": %s}' % bits, capture_output=True,
                       text=True, timeout=60)
    assert r.returncode == 1 and "kv_bits" not in json.loads(r.stdout)["error"]
