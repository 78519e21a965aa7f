"""What the bounds of oracle/mx4.py tell apart: x in five base-32 digits passes, x in four does not."""
import numpy as np
import pytest

from oracle import mx4 as OM


def inputs(K, seed):
    r = np.random.default_rng(seed)
    x = (r.standard_normal((24, K)) * np.exp(r.standard_normal(K))).astype(np.float32)
    w = 0.03 * r.standard_normal((2, 48, K)) * np.exp(0.4 * r.standard_normal(K))
    return x.astype(np.float64), [OM.values(*OM.quantise(v)) for v in w.astype(np.float32)]


def unlike(K, k):
    """One group in four 2^k times as large."""
    return np.where(np.arange(K) // 32 % 4 == 1, 2.0 ** k, 1.0)


SIZES = [64, 300, 576, 1001, 2048, 4100, 8192]


def ratio(err, bound):
    return np.linalg.norm(err) / np.linalg.norm(bound)


@pytest.mark.parametrize("K", SIZES)
@pytest.mark.parametrize("k", [0, 6, 16])
def test_four_digits_of_x_are_refused(K, k):
    x, (g, u) = inputs(K, K + k)
    x = x * unlike(K, k)
    y = x @ g.T
    for digits, passes in ((5, True), (4, False)):
        cut = OM.in_digits(x, digits)
        assert (ratio(cut @ g.T - y, OM.rms_bound(x, g, y)) <= 1) == passes, digits
        s = 1 / np.sqrt((y * y).mean())  # gates of ordinary size
        got = OM.silu(s * (cut @ g.T)) * (cut @ u.T)
        want = OM.silu(s * y) * (x @ u.T)
        assert (ratio(got - want, OM.gateup_rms_bound(x, s * g, u)) <= 1) == passes, digits


@pytest.mark.parametrize("K", SIZES)
def test_products_dropped_beside_others_are_refused(K):
    """What sums that keep 2^-17 of their largest term would give."""
    x, (g, _) = inputs(K, K)
    x = x * unlike(K, 8)
    y = x @ g.T
    got = np.zeros_like(y)
    for a in range(0, K, 128):
        t = x[:, None, a:a + 128] * g[None, :, a:a + 128]
        unit = np.ldexp(1.0, np.frexp(np.abs(t).max(2, keepdims=True))[1] - 17)
        got += (np.trunc(t / unit) * unit).sum(2)
    assert ratio(got - y, OM.rms_bound(x, g, y)) > 1


@pytest.mark.parametrize("K", SIZES)
def test_fp32_sums_pass(K):
    """x in five digits, products of 64 columns exact, their sums rounded to fp32 one by one."""
    x, (g, _) = inputs(K, 2 * K)
    y = x @ g.T
    cut, got = OM.in_digits(x, 5), np.zeros(y.shape, np.float32)
    for a in range(0, K, 64):
        got = (got + cut[:, a:a + 64] @ g[:, a:a + 64].T).astype(np.float32)
    assert ratio(got - y, OM.rms_bound(x, g, y)) <= 1
