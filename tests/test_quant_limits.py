"""CPU checks of what the few-bit stores' entry points refuse: sizes that one of a pair of calls
would take and the other not, that pass 64 bits, and bits that are not whole numbers."""
import ctypes as C

from emberlm_amd import capi

P = C.c_void_p(4096)  # never dereferenced


def test_rows_that_could_not_be_restored_are_not_quantised():
    lib = capi.lib()
    for rows in (2 ** 31, 2 ** 40):
        assert lib.ember_q8_quantize(P, P, P, rows, 4, None) == -1
        assert lib.ember_q8_dequantize(P, P, P, rows, 4, None) == -1
        assert lib.ember_q8_dequantize_rmsnorm(P, P, P, P, P, P, rows, 4, 1e-6, None) == -1
