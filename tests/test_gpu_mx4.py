"""GPU parity of the weights in 4 bits: the store bit for bit against the 64-bit rule (oracle/mx4.py),
the products against 64 bits over the values held, within oracle.mx4.product_bound."""
import ctypes as C

import numpy as np
import pytest

from oracle import mx4 as OM
from tests.helpers import call, dev, empty, host, p

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from emberlm_amd import capi  # noqa: E402

EPS = 1e-5


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.cuda.init()


def rng(s=0):
    return np.random.default_rng(s)


def at(a, off):
    """a on the GPU, `off` floats past an aligned address."""
    t = torch.empty(a.size + off, device="cuda")
    t[off:] = dev(a).reshape(-1)
    return t[off:].view(a.shape)


def weight(r, N, K):
    return (0.03 * r.standard_normal((N, K)) * np.exp(0.4 * r.standard_normal(K))).astype(
        np.float32)


def activations(r, M, K):
    return (r.standard_normal((M, K)) * np.exp(r.standard_normal(K))).astype(np.float32)


def raw(n):
    return torch.full((n,), 0xA5, device="cuda", dtype=torch.uint8)


def quantize(w, N, K):
    lib = capi.lib()
    codes, scales = raw(lib.ember_mx4_code_bytes(N, K)), raw(lib.ember_mx4_scale_bytes(N, K))
    call("ember_mx4_quantize", p(w), p(codes), p(scales), N, K, None)
    return codes, scales


def odd_values(w, r):
    """Groups that a quantiser can get wrong, over some rows of w."""
    N, K = w.shape
    k = np.arange(K)
    put = [np.zeros(K), k % 8 * 0.25 * 2.0 ** -3, (k % 29) * 0.25, -(k % 15) * 0.5,
           2.0 ** -149 * (k % 40), 2.0 ** -127 * r.standard_normal(K), 7 * 2.0 ** (k // 32 % 9 - 4.),
           np.nextafter(np.float32(7), np.float32(8)) * np.ones(K), 1.6e38 * np.cos(k),
           np.where(k == K // 2, np.inf, 1.0), np.where(k == K - 1, np.nan, 1.0),
           np.where(k == 0, -np.inf, 1.0), np.where(k % 5 == 0, -0.0, 1e-3),
           np.where(k % 32 == 7, 1e6, r.standard_normal(K))]
    for i, row in enumerate(put):
        if i < N:
            w[(i * 5) % N] = row.astype(np.float32)
    return w


STORE = [(1, 1), (1, 31), (3, 33), (32, 64), (33, 65), (70, 256), (5, 257), (131, 1001), (96, 576),
         (64, 2048), (31, 4100)]


@pytest.mark.parametrize("N,K", STORE)
@pytest.mark.parametrize("off", [0, 1])
def test_store_and_read_back(N, K, off):
    r = rng(N * K)
    w = odd_values(weight(r, N, K), r)
    src = at(w, off)
    codes, scales = quantize(src, N, K)
    want_c, want_s, want = OM.hold(w)
    assert np.array_equal(host(codes), want_c) and np.array_equal(host(scales), want_s)
    back = torch.full((N * K + off + 4,), 3.0, device="cuda")
    call("ember_mx4_dequantize", p(codes), p(scales), p(back[off:]), N, K, None)
    got = host(back)
    assert np.array_equal(got[off:off + N * K].reshape(N, K), want.astype(np.float32),
                          equal_nan=True)
    assert (got[:off] == 3.0).all() and (got[off + N * K:] == 3.0).all()


@pytest.mark.parametrize("V,K,n", [(1, 1, 40), (33, 65, 40), (200, 576, 40), (77, 1001, 40),
                                   (5, 300, 40), (40, 700, 3000), (33, 257, 5000), (50, 130, 9000)])
def test_lookup(V, K, n):
    r = rng(V + K)
    c, s, val = OM.hold(odd_values(weight(r, V, K), r))
    ids = np.concatenate([r.integers(0, V, n), [0, V - 1, V - 1, -1, V, 2 ** 40, -2 ** 40]])
    want = np.where(((ids >= 0) & (ids < V))[:, None], val[np.clip(ids, 0, V - 1)], 0.0)
    dids, c, s = dev(ids), dev(c), dev(s)
    for off in (0, 1):
        out = torch.full((len(ids) * K + off + 4,), 3.0, device="cuda")
        call("ember_mx4_embedding", p(dids), p(c), p(s), p(out[off:]), len(ids), K, V,
             None)
        got = host(out)
        assert np.array_equal(got[off:off + len(ids) * K].reshape(-1, K),
                              want.astype(np.float32), equal_nan=True)
        assert (got[:off] == 3.0).all() and (got[off + len(ids) * K:] == 3.0).all()


def held(r, N, K):
    c, s, val = OM.hold(weight(r, N, K))
    return dev(c), dev(s), val


def held_by_kernel(r, N, K):
    """The same by the two kernels, which test_store_and_read_back holds to it bit for bit."""
    c, s = quantize(dev(weight(r, N, K)), N, K)
    back = empty((N, K))
    call("ember_mx4_dequantize", p(c), p(s), p(back), N, K, None)
    return c, s, host(back).astype(np.float64)


def workspace(M, K, N):
    need = capi.lib().ember_mx4_workspace_bytes(M, K, N)
    return (raw(need) if need else None), need


def ptrs(ts):
    return (C.c_void_p * len(ts))(*[t.data_ptr() if t is not None else None for t in ts])


GUARD = 64


def guarded(shape):
    """An output with a band before and behind it, and a check of both."""
    n = int(np.prod(shape))
    t = torch.full((n + 2 * GUARD,), 7.0, device="cuda")

    def intact():
        e = host(t)
        return (e[:GUARD] == 7.0).all() and (e[-GUARD:] == 7.0).all()
    return t[GUARD:GUARD + n].view(shape), intact


def linear(x, M, K, weights, N, norm=None, res=None, stream=None):
    y = [guarded((M, n)) for n in N]
    ws, need = workspace(M, K, sum(N))
    call("ember_mx4_linear", p(x), M, K, p(norm), EPS, len(N), ptrs([w[0] for w in weights]),
         ptrs([w[1] for w in weights]), (C.c_int64 * len(N))(*N), ptrs([v[0] for v in y]),
         ptrs(res) if res else None, p(ws), need, stream)
    assert all(ok() for _, ok in y)
    return [v for v, _ in y]


def gateup(x, M, K, g, u, I, norm=None):
    h, ok = guarded((M, I))
    ws, need = workspace(M, K, 2 * I)
    call("ember_mx4_gateup", p(x), M, K, p(norm), EPS, p(g[0]), p(g[1]), p(u[0]), p(u[1]), I, p(h),
         p(ws), need, None)
    assert ok()
    return h


def check_product(got, xn, val, extra=None, floor=0.0):
    y = xn @ val.T
    bound = OM.product_bound(xn, val, y) + floor
    if extra is not None:
        y = y + extra
        bound = bound + 2.0 ** -24 * np.abs(y)
    err = np.abs(host(got).astype(np.float64) - y)
    assert (err <= bound).all(), (err.max(), (err / bound).max())
    return (err / bound).max()


# (M, K, N per weight, norm, residual): the few-row and many-row kernels, sizes that fill no group,
# tile or block, one of each, and weights of unlike sizes in a call
LINEAR = [
    (1, 1, (1,), False, False), (1, 33, (3,), True, True), (1, 64, (16,), False, False),
    (1, 576, (576, 192, 192), True, False), (2, 2048, (2048, 1024, 1024), True, False),
    (3, 300, (17, 33, 65), True, True), (4, 1001, (129,), False, True), (5, 960, (257, 1), False, False),
    (6, 256, (64,), True, True), (7, 6144, (100,), False, True), (8, 8192, (48, 20), True, True),
    (8, 31, (500,), False, False), (9, 64, (32,), False, True), (9, 1001, (577,), True, False),
    (31, 2048, (40, 300), False, False), (33, 1001, (577,), False, False), (32, 576, (192,), True, True),
    (64, 300, (256, 31, 128), True, True), (65, 4100, (130,), False, True), (100, 5, (9,), True, False),
    (127, 2048, (256,), True, True), (128, 320, (257,), False, False), (129, 256, (255, 256), True, False),
    (257, 1024, (600,), True, True), (300, 192, (1500, 70), False, True), (513, 2049, (129,), True, True),
    (1030, 448, (513,), False, False),
]


# Sizes that take what those do not, by the workgroups that they make: for few rows two and four
# tiles of columns a workgroup, and streams of them (K to 1024 and to 2048, one to three rows of tiles);
# sixteen waves; a K that several workgroups share; tiles of 64 x 128 (K of 1 to 16 tiles) and of 128 x 256
LARGER = [
    (2, 300, (9000,), True, True), (6, 1100, (6000, 3000), True, False), (8, 700, (5000,), False, True),
    (3, 600, (17000,), True, True), (8, 1000, (9000,), True, False), (1, 2100, (33000,), False, True),
    (1, 576, (20000, 13000), True, True), (3, 1030, (33000,), True, False), (2, 64, (33001, 7), False, True),
    (5, 250, (17000,), True, True), (6, 2048, (16500, 700), True, False), (7, 1001, (17000,), False, True),
    (8, 576, (20000, 100, 9000), True, True), (1, 8192, (50, 20), True, True), (3, 4100, (100,), True, True),
    (2, 3841, (4096,), False, False),
    (9, 4096, (40,), True, True), (40, 6200, (100, 33), False, True), (20, 8200, (70,), True, False),
    (700, 37, (4100,), True, True), (900, 100, (3000, 2100), True, False), (600, 190, (4100, 33), False, True),
    (640, 256, (4000,), True, True), (4000, 260, (4090,), False, False), (1921, 1001, (3900, 150), True, True),
    (1500, 333, (2100, 2100), True, True), (3900, 450, (2048,), True, False), (2000, 900, (4096,), False, True),
    (1100, 1600, (4000,), True, True),
]


@pytest.mark.parametrize("M,K,N,norm,res", LINEAR + LARGER)
def test_linear(M, K, N, norm, res):
    r = rng(M + K + sum(N))
    x = activations(r, M, K)
    nw = (1 + 0.1 * r.standard_normal(K)).astype(np.float32) if norm else None
    xn = OM.rms_norm(x, nw, EPS) if norm else x.astype(np.float64)
    weights = [held(r, n, K) if n < 1000 else held_by_kernel(r, n, K) for n in N]
    rs = [r.standard_normal((M, n)).astype(np.float32) for n in N] if res else None
    y = linear(dev(x), M, K, weights, N, dev(nw) if norm else None,
               [dev(v) for v in rs] if res else None)
    for i, (_, _, val) in enumerate(weights):
        check_product(y[i], xn, val, rs[i] if res else None)


GATEUP = [(1, 1, 1, False), (1, 576, 1536, True), (2, 100, 33, True), (3, 2048, 500, True),
          (5, 8192, 40, False), (8, 1001, 65, True), (9, 64, 16, False), (33, 577, 130, True),
          (64, 2048, 129, True), (130, 300, 257, True), (509, 576, 700, True), (600, 1026, 96, False)]

# As LARGER: four tiles a workgroup, a shared K, tiles of 64 x 128 and of 128 x 256
LARGER_GATEUP = [(3, 700, 8300, True), (6, 1100, 8200, False), (8, 300, 4200, True), (2, 2100, 8300, True),
                 (33, 4200, 50, True), (12, 9000, 40, False), (700, 37, 4100, True), (900, 192, 2100, False),
                 (1030, 333, 1900, True), (520, 1001, 1500, True), (2048, 449, 2040, True),
                 (2048, 1200, 2040, False), (2000, 1030, 2048, True), (4000, 1300, 1020, True)]


def check_gateup(h, xn, g, u):
    yg, yu = xn @ g.T, xn @ u.T
    dg, du = OM.product_bound(xn, g, yg), OM.product_bound(xn, u, yu)
    want = OM.silu(yg) * yu
    # |silu'| <= 1.1; exp's, the quotient's and two products' roundings, of which exp's scales with
    # the fp32 argument: 2^-23 |g| more; e^g below 2^-126 counts as 0
    bound = (1.1 * dg * (np.abs(yu) + du) + (np.abs(OM.silu(yg)) + dg) * du +
             2.0 ** -23 * (6 + np.abs(yg)) * np.abs(want) + 2.0 ** -126 * (1 + np.abs(yg * yu)))
    err = np.abs(h - want)
    assert (err <= bound).all(), (err / bound).max()


@pytest.mark.parametrize("M,I", [(1, 5000), (8, 300), (9, 300), (600, 2100), (2048, 2040)])
def test_gates_of_all_sizes(M, I):
    """Gates from -2000 to 2000 and around 0, upwards of 0 and below where e^-|g| ends."""
    r = rng(M)
    K = 64
    x = activations(r, M, K)
    size = np.exp2(r.integers(-20, 9, (I, 1)))
    g, u = [(r.standard_normal((I, K)) * s / 8).astype(np.float32) for s in (size, 1.0)]
    (gc, gs, gv), (uc, us, uv) = OM.hold(g), OM.hold(u)
    h = host(gateup(dev(x), M, K, (dev(gc), dev(gs)), (dev(uc), dev(us)), I)).astype(np.float64)
    yg = x.astype(np.float64) @ gv.T
    assert yg.min() < -200 and yg.max() > 200
    check_gateup(h, x.astype(np.float64), gv, uv)


@pytest.mark.parametrize("M,K,I,norm", GATEUP + LARGER_GATEUP)
def test_gateup(M, K, I, norm):
    r = rng(M + K + I)
    x = activations(r, M, K)
    nw = (1 + 0.1 * r.standard_normal(K)).astype(np.float32) if norm else None
    xn = OM.rms_norm(x, nw, EPS) if norm else x.astype(np.float64)
    g, u = [(held if I < 1000 else held_by_kernel)(r, I, K) for _ in range(2)]
    h = host(gateup(dev(x), M, K, g, u, I, dev(nw) if norm else None)).astype(np.float64)
    check_gateup(h, xn, g[2], u[2])


@pytest.mark.parametrize("M", [1, 5, 8, 9, 40, 300])
def test_closer_than_an_fp32_chain(M):
    """In the 2-norm, beside fp32 products over the values read back (of some other order of sums:
    half as much again is allowed for)."""
    r = rng(M)
    K, N = 2048, 512
    x, w = activations(r, M, K), held(r, N, K)
    y = x.astype(np.float64) @ w[2].T
    chain = host(torch.mm(dev(x), dev(w[2]).t())).astype(np.float64)
    got = host(linear(dev(x), M, K, [w], (N,))[0]).astype(np.float64)
    assert np.linalg.norm(got - y) <= 1.5 * np.linalg.norm(chain - y)


@pytest.mark.parametrize("M", [1, 8, 9, 40, 300])
def test_rows_of_many_sizes_do_not_meet(M):
    """Rows of x 2^200 apart, and a row that is not finite: each row is held by its own scales."""
    r = rng(M)
    K, N = 700, 130
    x = activations(r, M, K)
    x *= np.exp2(r.integers(-90, 90, (M, 1))).astype(np.float32)
    x[M // 2] = 0
    w = held(r, N, K)
    alone = host(linear(dev(x), M, K, [w], (N,))[0])
    check_product(torch.from_numpy(alone), x.astype(np.float64), w[2])
    if M > 2:
        x[M // 2, 5], x[M - 1, K - 1] = np.inf, np.nan
        got = host(linear(dev(x), M, K, [w], (N,))[0])
        bad = np.arange(M)[[M // 2, M - 1]]
        assert not np.isfinite(got[bad]).any()  # inf w or NaN, as the sums come
        rest = np.setdiff1d(np.arange(M), bad)
        assert np.array_equal(got[rest], alone[rest])


@pytest.mark.parametrize("M", [1, 8, 9, 64, 300])
@pytest.mark.parametrize("size", [2.0 ** 120, 2.0 ** 90, 2.0 ** -90, 2.0 ** -115])
def test_ends_of_the_range(M, size):
    """x near fp32's ends, weights on the other side of 1: products of ordinary size."""
    r = rng(M)
    K, N = 256, 70
    x = (size * np.clip(r.standard_normal((M, K)), -3, 3)).astype(np.float32)
    w = (r.standard_normal((N, K)) / min(size, 2.0 ** 110) if size > 1 else
         r.standard_normal((N, K)) * min(1 / size, 2.0 ** 110)).astype(np.float32)
    c, s, val = OM.hold(w)
    # x enters in whole multiples of at least 2^-127: a term may be off by 2^-128 |w| beside
    # product_bound's, which counts steps relative to a group's largest size
    check_product(linear(dev(x), M, K, [(dev(c), dev(s))], (N,))[0], x.astype(np.float64), val,
                  floor=2.0 ** -128 * np.abs(val).sum(1))


def test_x_in_pieces():
    """A long x is taken in pieces of rows: K = 65536 in 1024 at a time."""
    r = rng(3)
    M, K, N = 1100, 65536, 33
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    x = torch.randn((M, K), generator=gen, device="cuda")
    assert capi.lib().ember_mx4_workspace_bytes(M, K, N) < 4.5 * 1100 * K  # not all of it at once
    w = held(r, N, K)
    nw = dev((1 + 0.1 * r.standard_normal(K)).astype(np.float32))
    rs = r.standard_normal((M, N)).astype(np.float32)
    y = linear(x, M, K, [w], (N,), nw, [dev(rs)])[0]
    rows = [0, 1, 1023, 1024, 1025, 1099]
    xn = OM.rms_norm(host(x[rows]), host(nw), EPS)
    check_product(y[rows], xn, w[2], rs[rows])


def test_outputs_past_32_bit_offsets():
    M, K, N = 66000, 33, 33000
    r = rng(4)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(2)
    x = torch.randn((M, K), generator=gen, device="cuda")
    w = held(r, N, K)
    y = empty((M, N))
    assert y.numel() > 2 ** 31
    ws, need = workspace(M, K, N)
    call("ember_mx4_linear", p(x), M, K, None, EPS, 1, ptrs([w[0]]), ptrs([w[1]]),
         (C.c_int64 * 1)(N), ptrs([y]), None, p(ws), need, None)
    rows = [0, 1, 32767, 65073, 65074, 65075, 65998, 65999]
    check_product(y[rows], host(x[rows]).astype(np.float64), w[2])


def test_weights_past_32_bit_offsets():
    """4.5e9 values: 18 GB of fp32, 2.3 GB of codes."""
    N, K = 1100000, 4096
    gen = torch.Generator(device="cuda")
    gen.manual_seed(5)
    w = torch.empty((N, K), device="cuda")
    for part in w.split(100000):
        part.copy_(0.02 * torch.randn(part.shape, generator=gen, device="cuda"))
    codes, scales = quantize(w, N, K)
    assert codes.numel() > 2 ** 31
    ids = np.array([0, 31, 32, 524287, 524288, 1048575, 1048576, N - 1])
    val = OM.hold(host(w[ids]))[2]
    out, dids = empty((len(ids), K)), dev(ids)
    call("ember_mx4_embedding", p(dids), p(codes), p(scales), p(out), len(ids), K, N, None)
    assert np.array_equal(host(out), val.astype(np.float32))
    w.zero_()
    call("ember_mx4_dequantize", p(codes), p(scales), p(w), N, K, None)
    assert np.array_equal(host(w[ids]), val.astype(np.float32))
    del w
    r = rng(6)
    for M in (1, 3, 6, 8, 9, 40):
        x = activations(r, M, K)
        y = linear(dev(x), M, K, [(codes, scales)], (N,))[0]
        check_product(y[:, ids], x.astype(np.float64), val)


@pytest.mark.parametrize("M", [1, 8, 9, 300])
def test_weight_rows_that_are_not_finite(M):
    """Only their own columns of y are NaN."""
    r = rng(M)
    K, N = 500, 100
    w = weight(r, N, K)
    w[3, 7], w[64, 499], w[99, 0] = np.inf, np.nan, -np.inf
    c, s, val = OM.hold(w)
    x = activations(r, M, K)
    got = host(linear(dev(x), M, K, [(dev(c), dev(s))], (N,))[0])
    bad = [3, 64, 99]
    assert np.isnan(got[:, bad]).all()
    good = np.setdiff1d(np.arange(N), bad)
    check_product(torch.from_numpy(got[:, good]), x.astype(np.float64), val[good])


@pytest.mark.parametrize("M", [1, 3, 8, 9, 70, 300])
def test_sums_of_one_sign(M):
    """Nothing cancels: a sum that rounds downwards would show."""
    r = rng(M)
    K, N = 4096, 160
    x = np.abs(activations(r, M, K))
    c, s, val = OM.hold(np.abs(weight(r, N, K)))
    y = x.astype(np.float64) @ val.T
    got = host(linear(dev(x), M, K, [(dev(c), dev(s))], (N,))[0]).astype(np.float64)
    assert (np.abs(got - y) <= 2.0 ** -24 * (24 + 2 * K / 64) * y).all()
    assert np.abs((got - y) / y).mean() <= 4 * 2.0 ** -24


@pytest.mark.parametrize("M,K,N", [(1, 576, (33,)), (8, 1001, (100, 40)), (40, 300, (65,)),
                                   (300, 520, (257,))])
def test_addresses_of_any_float(M, K, N):
    """x, the norm's weight, residuals and outputs one float past an aligned address: the same bits."""
    r = rng(K)
    x, nw = activations(r, M, K), (1 + 0.1 * r.standard_normal(K)).astype(np.float32)
    weights = [held(r, n, K) for n in N]
    rs = [r.standard_normal((M, n)).astype(np.float32) for n in N]
    want = linear(dev(x), M, K, weights, N, dev(nw), [dev(v) for v in rs])
    y = [torch.zeros(M * n + 1, device="cuda") for n in N]
    ws, need = workspace(M, K, sum(N))
    x1, nw1, rs1 = at(x, 1), at(nw, 1), [at(v, 1) for v in rs]
    call("ember_mx4_linear", p(x1), M, K, p(nw1), EPS, len(N),
         ptrs([w[0] for w in weights]), ptrs([w[1] for w in weights]), (C.c_int64 * len(N))(*N),
         ptrs([v[1:] for v in y]), ptrs(rs1), p(ws), need, None)
    for a, b, n in zip(want, y, N):
        assert np.array_equal(host(a), host(b)[1:].reshape(M, n))


@pytest.mark.parametrize("M", [2, 8, 33, 300])
def test_residual_in_place_and_repeats(M):
    r = rng(M)
    K, N = 640, 200
    x, w = dev(activations(r, M, K)), held(r, N, K)
    rs = r.standard_normal((M, N)).astype(np.float32)
    want = host(linear(x, M, K, [w], (N,), None, [dev(rs)])[0])
    ws, need = workspace(M, K, N)
    for _ in range(3):
        y = dev(rs)
        call("ember_mx4_linear", p(x), M, K, None, EPS, 1, ptrs([w[0]]), ptrs([w[1]]),
             (C.c_int64 * 1)(N), ptrs([y]), ptrs([y]), p(ws), need, None)
        assert np.array_equal(host(y), want)


@pytest.mark.parametrize("M", [1, 7, 33, 300])
def test_some_weights_with_a_residual(M):
    r = rng(M)
    K, N = 200, (40, 70, 33)
    x = activations(r, M, K)
    weights = [held(r, n, K) for n in N]
    rs = r.standard_normal((M, N[1])).astype(np.float32)
    y = linear(dev(x), M, K, weights, N, None, [None, dev(rs), None])
    for i, extra in enumerate((None, rs, None)):
        check_product(y[i], x.astype(np.float64), weights[i][2], extra)


@pytest.mark.parametrize("M", [1, 6, 40, 300])
def test_a_row_does_not_depend_on_its_neighbours(M):
    """A weight's rows alone, in another call's second place, give the same bits."""
    r = rng(M)
    K, N = 1000, (96, 70)
    x = dev(activations(r, M, K))
    a, b = held(r, N[0], K), held(r, N[1], K)
    both = linear(x, M, K, [a, b], N)
    assert np.array_equal(host(both[1]), host(linear(x, M, K, [b], N[1:])[0]))


def test_calls_on_two_streams():
    r = rng(1)
    K, N = 1024, 300
    w = held(r, N, K)
    jobs = []
    for M in (4, 64, 300, 5, 200, 8):
        x = dev(activations(r, M, K))
        jobs.append((x, M, host(linear(x, M, K, [w], (N,))[0])))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    out = []
    torch.cuda.synchronize()
    for i, (x, M, _) in enumerate(jobs):
        ws, need = workspace(M, K, N)
        y = empty((M, N))
        torch.cuda.synchronize()
        capi.call("ember_mx4_linear", p(x), M, K, None, EPS, 1, ptrs([w[0]]), ptrs([w[1]]),
                  (C.c_int64 * 1)(N), ptrs([y]), None, p(ws), need,
                  C.c_void_p(streams[i % 2].cuda_stream))
        out.append((y, ws))
    torch.cuda.synchronize()
    for (y, _), (_, _, want) in zip(out, jobs):
        assert np.array_equal(host(y), want)


@pytest.mark.parametrize("M,K,I", [(1, 576, 320), (8, 576, 320), (40, 576, 320), (300, 576, 320),
                                   (1, 600, 17000), (20, 4200, 4300), (2000, 1030, 2048)])
def test_captured_and_replayed(M, K, I):
    """A block's products in a graph, replayed on new inputs between eager calls."""
    r = rng(M)
    nw = dev((1 + 0.1 * r.standard_normal(K)).astype(np.float32))
    g, u, d = [held_by_kernel(r, *s) for s in ((I, K), (I, K), (K, I))]
    x, h, y = empty((M, K)), empty((M, I)), empty((M, K))
    ws1, need1 = workspace(M, K, 2 * I)
    ws2, need2 = workspace(M, I, K)

    def step(st):
        capi.call("ember_mx4_gateup", p(x), M, K, p(nw), EPS, p(g[0]), p(g[1]), p(u[0]), p(u[1]), I,
                  p(h), p(ws1), need1, st)
        capi.call("ember_mx4_linear", p(h), M, I, None, EPS, 1, ptrs([d[0]]), ptrs([d[1]]),
                  (C.c_int64 * 1)(K), ptrs([y]), ptrs([x]), p(ws2), need2, st)
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        step(C.c_void_p(s.cuda_stream))
    for i in range(4):
        new = dev(activations(r, M, K))
        x.copy_(new)
        graph.replay()
        got = host(y).copy()
        y.zero_(), h.zero_()
        torch.cuda.synchronize()
        step(C.c_void_p(torch.cuda.current_stream().cuda_stream))
        assert np.array_equal(host(y), got), i


def test_lookup_block_and_head_together():
    """Token ids to logits through one block's MLP and the tied table, as a decode step uses them."""
    r = rng(5)
    V, K, I, M = 1000, 576, 320, 3
    table, g, u, d = held(r, V, K), held(r, I, K), held(r, I, K), held(r, K, I)
    nw = (1 + 0.1 * r.standard_normal(K)).astype(np.float32)
    ids = np.array([0, 999, 517])
    x, dids = empty((M, K)), dev(ids)
    call("ember_mx4_embedding", p(dids), p(table[0]), p(table[1]), p(x), M, K, V, None)
    h = gateup(x, M, K, g, u, I, dev(nw))
    x2 = linear(h, M, I, [d], (K,), None, [x])[0]
    logits = host(linear(x2, M, K, [table], (V,), dev(nw))[0])
    x64 = table[2][ids]
    xn = OM.rms_norm(x64, nw, EPS)
    x64 = x64 + (OM.silu(xn @ g[2].T) * (xn @ u[2].T)) @ d[2].T
    want = OM.rms_norm(x64, nw, EPS) @ table[2].T
    # four stages (K = 576, 320: at most 24 + 2 * 9 half steps each, oracle.mx4.product_bound) in a
    # row: 4 * 42 * 2^-24
    assert np.linalg.norm(logits - want) <= 168 * 2.0 ** -24 * np.linalg.norm(want)
