"""Products with weights in 4 bits over every kernel: errors in the 2-norm (oracle.mx4.rms_bound, which a
lost digit of x is three times past), groups of unlike sizes in a row, values that are not finite,
one-sided sums, calls at once, and what lies behind a workspace."""
import ctypes as C

import numpy as np
import pytest

from oracle import mx4 as OM
from tests.helpers import dev, empty, host, p
from tests.test_gpu_mx4 import (EPS, activations, gateup, held_by_kernel, linear, ptrs, quantize,
                                rng, weight, workspace)

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from emberlm_amd import capi  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.cuda.init()


# (M, K, N), by the kernel and the workgroups that they make: one, two and three tiles of x's digits
# and one to four column tiles a workgroup; streams; sixteen waves; 32 x 32 tiles, and those that share
# a K; 64 x 128; 128 x 256 in one round and in several
LINEAR = [
    (1, 576, 192), (2, 1024, 9000), (3, 300, 130), (5, 960, 500), (6, 2048, 6000), (8, 1001, 513),
    (3, 1030, 33000), (1, 1000, 20000), (5, 250, 17000), (8, 2048, 16500),
    (1, 8192, 70), (3, 4100, 100),
    (9, 577, 130), (33, 1001, 577), (100, 2048, 300),
    (8, 8192, 48), (20, 8200, 70), (40, 4100, 33),
    (640, 256, 4000), (700, 1001, 4100), (600, 2050, 4100),
    (2000, 900, 4096), (1921, 1600, 3900), (2048, 2048, 8192),
]
GATEUP = [
    (1, 576, 320), (3, 700, 8300), (6, 1100, 8200), (8, 300, 4200), (8, 2048, 500),
    (33, 577, 130), (64, 2048, 129), (33, 4200, 50),
    (700, 300, 4100), (900, 1001, 2100),
    (2048, 576, 2040), (2048, 2048, 2040),
]


def some(n, of):
    """n of the first `of` indices, each place in a tile among them, and the last ones."""
    return np.unique(np.r_[np.arange(0, of, 1 + of // n | 1), max(0, of - 33):of])


def within(got, want, bound):
    """The 2-norm of the error, and no element more than 8 times its root mean square (a Gaussian's
    10^-15; these are sums of hundreds of roundings)."""
    err = got.astype(np.float64) - want
    assert np.linalg.norm(err) <= np.linalg.norm(bound), np.linalg.norm(err) / np.linalg.norm(bound)
    assert (np.abs(err) <= 8 * bound).all(), np.abs(err / bound).max()


class Inputs:
    """x [M, K], weights [N, K] and a norm's weight as a model has them, made on the GPU."""

    def __init__(self, M, K, N, weights=1):
        gen = torch.Generator(device="cuda")
        gen.manual_seed(M + K + N)
        rand = lambda *shape: torch.randn(shape, generator=gen, device="cuda")  # noqa: E731
        self.M, self.K, self.N = M, K, N
        self.x = rand(M, K) * torch.exp(rand(K))
        self.w = [0.03 * rand(N, K) * torch.exp(0.4 * rand(K)) for _ in range(weights)]
        self.nw = 1 + 0.1 * rand(K)
        self.rows, self.cols = some(160, M), some(320, N)

    def x64(self, x, norm):
        x = host(x[dev(self.rows)])
        return OM.rms_norm(x, host(self.nw), EPS) if norm else x.astype(np.float64)

    def part(self, y):
        return host(y[dev(self.rows)][:, dev(self.cols)])

    def held(self, w):
        """The two buffers, and the values of some rows in 64 bits."""
        c, s = quantize(w, self.N, self.K)
        back = empty((self.N, self.K))
        torch.cuda.synchronize()
        capi.call("ember_mx4_dequantize", p(c), p(s), p(back), self.N, self.K, None)
        torch.cuda.synchronize()
        return c, s, host(back[dev(self.cols)]).astype(np.float64)


def unlike(K, where, k):
    """Factors of the columns: one group in four 2^k times as large (or as small)."""
    return dev(np.where(np.arange(K) // 32 % 4 == where, 2.0 ** k, 1.0).astype(np.float32))


# which side has the unlike groups, where in each 128 columns, how much larger; with the norm or not
SIDES = [(None, 0, 0, False), ("x", 1, 6, False), ("x", 0, 10, False), ("x", 3, 16, False),
         ("w", 2, 10, False), ("w", 1, 16, False), ("x", 2, -16, False), (None, 0, 0, True),
         ("x", 2, 10, True)]


@pytest.mark.parametrize("M,K,N", LINEAR)
def test_linear(M, K, N):
    s = Inputs(M, K, N)
    for side, where, k, norm in SIDES:
        f = unlike(K, where, k)
        x = s.x * f if side == "x" else s.x
        w = s.held(s.w[0] * f if side == "w" else s.w[0])
        got = s.part(linear(x, M, K, [w], (N,), s.nw if norm else None)[0])
        xn = s.x64(x, norm)
        y = xn @ w[2].T
        within(got, y, OM.rms_bound(xn, w[2], y))


@pytest.mark.parametrize("M,K,I", GATEUP)
def test_gateup(M, K, I):
    s = Inputs(M, K, I, 2)
    for side, where, k, norm in SIDES:
        f = unlike(K, where, k)
        x = s.x * f if side == "x" else s.x
        xn = s.x64(x, norm)
        w = [v * f if side == "w" else v for v in s.w]
        # gates of ordinary size: a power of two leaves codes and digits as they are
        size = 2.0 ** -np.rint(0.5 * np.log2(((xn ** 2) @ (host(w[0][:40]).T.astype(np.float64) ** 2)).mean()))
        g, u = [s.held(v * size) for v in w]
        got = s.part(gateup(x, M, K, g, u, I, s.nw if norm else None))
        want = OM.silu(xn @ g[2].T) * (xn @ u[2].T)
        within(got, want, OM.gateup_rms_bound(xn, g[2], u[2]))


# one case of each kernel
KERNELS = [(1, 640, 300), (8, 640, 300), (3, 640, 33000), (8, 8192, 48), (40, 640, 300), (20, 8200, 70),
           (640, 640, 4000), (2048, 640, 4096)]


@pytest.mark.parametrize("M,K,N", KERNELS)
@pytest.mark.parametrize("k", [8, 20, 60])
def test_a_large_group_that_cancels(M, K, N, k):
    """Pairs of equal large values times weights of opposite signs, beside ordinary groups."""
    s = Inputs(M, K, N)
    for a in range(32, K - 31, 128):
        s.x[:, a:a + 32] = 0
        s.x[:, a + 5] = s.x[:, a + 20] = 2.0 ** k
        s.w[0][:, a + 20] = -s.w[0][:, a + 5]
    w, x64 = s.held(s.w[0]), s.x64(s.x, False)
    y = x64 @ w[2].T
    within(s.part(linear(s.x, M, K, [w], (N,))[0]), y, OM.rms_bound(x64, w[2], y))


@pytest.mark.parametrize("M,K,N", KERNELS)
@pytest.mark.parametrize("k", [7, 20, 100])
def test_a_huge_column_whose_weights_are_zero(M, K, N, k):
    """It costs the 32 columns of its own group bits, by the rule, and no others any."""
    s = Inputs(M, K, N)
    s.x[:, 40] = 2.0 ** k
    s.w[0][:, 40] = 0
    s.w[0][:N // 2, 32:64] = 0  # of these weights' products nothing is lost
    w, x64 = s.held(s.w[0]), s.x64(s.x, False)
    got = s.part(linear(s.x, M, K, [w], (N,))[0])
    for part in (s.cols < N // 2, s.cols >= N // 2):
        y = x64 @ w[2][part].T
        within(got[:, part], y, OM.rms_bound(x64, w[2][part], y))


@pytest.mark.parametrize("M,K,N", KERNELS)
def test_sums_of_one_sign(M, K, N):
    s = Inputs(M, K, N)
    x, w = s.x.abs(), s.held(s.w[0].abs())
    y = s.x64(x, False) @ w[2].T
    got = s.part(linear(x, M, K, [w], (N,))[0]).astype(np.float64)
    assert (np.abs(got - y) <= 2.0 ** -24 * (24 + 2 * K / 64) * y).all()
    # dropped parts are an eighth of a half step at most for each of two sums' K / 64 steps; roundings
    # do not have a side
    assert abs(((got - y) / y).mean()) <= 2.0 ** -24 * (1 + 2 * K / 64 / 8)


@pytest.mark.parametrize("M,K,N", KERNELS)
def test_values_that_are_not_finite(M, K, N):
    """Rows of x and of the weight: their own rows and columns of y, and nothing else's bits."""
    r = rng(N)
    x, w = activations(r, M, K), weight(r, N, K)
    x *= np.exp2(r.integers(-60, 60, (M, 1))).astype(np.float32)  # rows do not meet either
    res = r.standard_normal((M, N)).astype(np.float32)
    call = lambda x, w: host(linear(dev(x), M, K, [quantize(dev(w), N, K)], (N,), None,  # noqa: E731
                                    [dev(res)])[0])
    want = call(x, w)
    bad_m = sorted({M // 2, M - 1}) if M > 2 else []
    bad_n = [3, N // 2, N - 1]
    for i, m in enumerate(bad_m):
        x[m, (5, K - 1)[i]] = (np.inf, np.nan)[i]
    for i, n in enumerate(bad_n):
        w[n, (7, K // 2, 0)[i]] = (np.nan, -np.inf, np.inf)[i]
    got = call(x, w)
    assert not np.isfinite(got[bad_m]).any() and np.isnan(got[:, bad_n]).all()
    m, n = np.setdiff1d(np.arange(M), bad_m), np.setdiff1d(np.arange(N), bad_n)
    assert np.array_equal(got[np.ix_(m, n)], want[np.ix_(m, n)])


@pytest.mark.parametrize("M,K,N", KERNELS)
def test_residual_in_place(M, K, N):
    r = rng(K)
    x, w = dev(activations(r, M, K)), held_by_kernel(r, N, K)
    res = r.standard_normal((M, N)).astype(np.float32)
    want = host(linear(x, M, K, [w], (N,), None, [dev(res)])[0])
    ws, need = workspace(M, K, N)
    y = dev(res)
    torch.cuda.synchronize()
    capi.call("ember_mx4_linear", p(x), M, K, None, EPS, 1, ptrs([w[0]]), ptrs([w[1]]),
              (C.c_int64 * 1)(N), ptrs([y]), ptrs([y]), p(ws), need, None)
    assert np.array_equal(host(y), want)


GUARD = 4096  # bytes


def guarded_workspace(M, K, N):
    need = capi.lib().ember_mx4_workspace_bytes(M, K, N)
    t = torch.full((need + 2 * GUARD,), 0x5A, device="cuda", dtype=torch.uint8)
    return t, C.c_void_p(t.data_ptr() + GUARD) if need else None, need


def intact(t):
    return bool((t[:GUARD] == 0x5A).all()) and bool((t[-GUARD:] == 0x5A).all())


@pytest.mark.parametrize("M,K,N", KERNELS + [(9, 1, 33), (64, 8193, 1), (65, 577, 4100), (4000, 33, 4100),
                                             (9, 8200, 300), (129, 8192, 129)])
def test_nothing_is_written_beside_a_workspace(M, K, N):
    r = rng(M + N)
    x, w = dev(activations(r, M, K)), held_by_kernel(r, N, K)
    nw = dev((1 + 0.1 * r.standard_normal(K)).astype(np.float32))
    h = gateup(x, M, K, w, w, N, nw)
    y = linear(x, M, K, [w], (N,), nw)[0]
    t1, ws1, need1 = guarded_workspace(M, K, N)
    t2, ws2, need2 = guarded_workspace(M, K, 2 * N)
    y2, h2 = empty((M, N)), empty((M, N))
    torch.cuda.synchronize()
    capi.call("ember_mx4_linear", p(x), M, K, p(nw), EPS, 1, ptrs([w[0]]), ptrs([w[1]]),
              (C.c_int64 * 1)(N), ptrs([y2]), None, ws1, need1, None)
    capi.call("ember_mx4_gateup", p(x), M, K, p(nw), EPS, p(w[0]), p(w[1]), p(w[0]), p(w[1]), N, p(h2),
              ws2, need2, None)
    assert np.array_equal(host(y2), host(y)) and np.array_equal(host(h2), host(h))
    assert intact(t1) and intact(t2)


def test_calls_at_once():
    """Both streams are full from the first call to the last: nothing waits in between."""
    r = rng(1)
    I = 2000
    jobs = []
    for M, K in ((600, 2048), (20, 8200), (8, 2048), (640, 1024), (40, 8192), (2000, 1024), (3, 8192),
                 (600, 2048), (33, 8200), (512, 4096)):
        g, u = held_by_kernel(r, I, K), held_by_kernel(r, 200, K)
        x = dev(activations(r, M, K))
        jobs.append((x, M, K, g, u, host(gateup(x, M, K, g, g, I)), host(linear(x, M, K, [u], (200,))[0])))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    rounds = 6
    out = [[(empty((M, I)), empty((M, 200)), workspace(M, K, 2 * I), workspace(M, K, 200))
            for _, M, K, *_ in jobs] for _ in range(rounds)]
    torch.cuda.synchronize()
    for i in range(rounds):
        for j, (x, M, K, g, u, _, _) in enumerate(jobs):
            h, y, (ws1, need1), (ws2, need2) = out[i][j]
            # the stream of a job changes with the rounds; its two calls run on one each
            a, b = [C.c_void_p(streams[(i + j + k) % 2].cuda_stream) for k in (0, 1)]
            capi.call("ember_mx4_gateup", p(x), M, K, None, EPS, p(g[0]), p(g[1]), p(g[0]), p(g[1]), I,
                      p(h), p(ws1), need1, a)
            capi.call("ember_mx4_linear", p(x), M, K, None, EPS, 1, ptrs([u[0]]), ptrs([u[1]]),
                      (C.c_int64 * 1)(200), ptrs([y]), None, p(ws2), need2, b)
    torch.cuda.synchronize()
    for i in range(rounds):
        for j, job in enumerate(jobs):
            assert np.array_equal(host(out[i][j][0]), job[5]), (i, j)
            assert np.array_equal(host(out[i][j][1]), job[6]), (i, j)
