"""GPU parity of the few-bit stores: the 4-bit KV cache with its attention, and 8-bit rows.

Codes, offsets and steps are compared with the 64-bit rule (oracle/quant.py) for equality: the
kernels form the same quotient in fp64.  Read-back is one rounding, half an fp32 step (2^-24 of the
value).  The attention's tolerance is written at `attention_bounds`.
"""
import ctypes as C

import numpy as np
import pytest

from oracle import quant as OQ
from tests.helpers import call, dev, empty, host, p

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from emberlm_amd import capi  # noqa: E402

HALF = 2.0 ** -24  # half an fp32 step, relative


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.cuda.init()


def rng(s=0):
    return np.random.default_rng(s)


def words(a):
    """uint32 -> int32 on the GPU, the same bits."""
    return dev(np.ascontiguousarray(a).view(np.int32))


def same(a, b):
    return np.array_equal(a, b, equal_nan=a.dtype.kind == "f")


def close_roundings(got, ref, n=1):
    """n roundings to fp32 of relative size 2^-24 each, or the last subnormal step."""
    got, ref = got.astype(np.float64), np.asarray(ref, np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    ok = ~np.isnan(ref)
    assert (np.abs(got - ref)[ok] <= n * HALF * np.abs(ref)[ok] + 2.0 ** -149).all()


def rows_like_keys(r, *shape):
    """Rows whose channels differ in size and centre."""
    D = shape[-1]
    return (r.standard_normal(shape) * np.exp(0.5 * r.standard_normal(D)) +
            0.5 * r.standard_normal(D)).astype(np.float32)


def odd_rows(x, r):
    """Rows that a quantiser can get wrong, put over some of x [n, D]."""
    n, D = x.shape
    put = [np.full(D, -3.75), np.zeros(D), np.arange(D) % 31 * 0.5, np.arange(D) * 2.0 ** -149,
           np.linspace(-1e38, 1e38, D), 1e4 + 1e-3 * r.standard_normal(D),
           np.where(np.arange(D) == D // 2, 1e30, r.standard_normal(D)),
           2.0 ** -140 * r.standard_normal(D), np.where(np.arange(D) == 0, np.inf, 1.0),
           np.where(np.arange(D) == D - 1, np.nan, 1.0), np.where(np.arange(D) == 3, -np.inf, 0.0)]
    for i, row in enumerate(put[:n]):
        x[i * (n // len(put)) if n >= len(put) else i] = row.astype(np.float32)
    return x


# ------------------------------------------------------------------ cache write and read
WRITE = [  # B, T, Hk, D, S, pos
    (1, 1, 1, 8, 1, 0), (1, 1, 8, 128, 64, 17), (2, 5, 3, 64, 16, 11), (2, 37, 2, 80, 41, 4),
    (1, 3, 5, 16, 9, 0), (3, 7, 1, 256, 7, 0), (1, 130, 8, 128, 200, 70), (4, 33, 4, 40, 64, 1),
    (1, 9, 2, 136, 20, 11),
]


@pytest.mark.parametrize("B,T,Hk,D,S,pos", WRITE)
def test_kv4_write_and_read(B, T, Hk, D, S, pos):
    r = rng(B * T + D)
    src = {n: odd_rows(rows_like_keys(r, B * T * Hk, D), r).reshape(B, T, Hk, D) for n in "kv"}
    old = {n: (r.integers(0, 2 ** 32, (B, Hk, S, D // 8), dtype=np.uint32),
               r.standard_normal((B, Hk, S, 2)).astype(np.float32)) for n in "kv"}
    buf = {n: (words(old[n][0]), dev(old[n][1])) for n in "kv"}
    kd, vd = dev(src["k"]), dev(src["v"])
    call("ember_kv4_write", p(kd), p(vd), p(buf["k"][0]), p(buf["k"][1]), p(buf["v"][0]),
         p(buf["v"][1]), B, T, Hk, D, S, pos, None)
    for n in "kv":
        codes, params = OQ.quantise(src[n].transpose(0, 2, 1, 3), 15)
        ref_w, ref_p = old[n][0].copy(), old[n][1].copy()
        ref_w[:, :, pos:pos + T] = OQ.pack4(codes)
        ref_p[:, :, pos:pos + T] = params
        assert same(host(buf[n][1]), ref_p)
        assert same(host(buf[n][0]).view(np.uint32), ref_w)
        for group, L in ((1, pos + T), (3, max(1, pos + T - 1))):
            out = empty((B, Hk * group, L, D))
            call("ember_kv4_read_expanded", p(buf[n][0]), p(buf[n][1]), p(out), B, Hk, group, L,
                 D, S, None)
            ref = OQ.values(OQ.unpack4(ref_w), ref_p)[:, :, :L]
            close_roundings(host(out), np.repeat(ref, group, axis=1))


# --------------------------------------------------------------------------- attention
def held_cache(r, B, Hk, S, D):
    """A cache's buffers (numpy) and the values it holds, in 64 bits."""
    out = []
    for _ in range(2):
        codes, params = OQ.quantise(rows_like_keys(r, B, Hk, S, D), 15)
        out.append((OQ.pack4(codes), params, OQ.values(codes, params)))
    return out


def attend(q, cache, L, pos, scale, ws_fill=None):
    B, T, H, D = q.shape
    (kw, kp, _), (vw, vp, _) = cache
    Hk, S = kp.shape[1], kp.shape[2]
    t = [dev(q), words(kw), dev(kp), words(vw), dev(vp)]
    o = torch.full((B, T, H, D), 7.0, device="cuda")
    need = capi.lib().ember_attn_kv4_workspace_bytes(B, T, H, Hk, D, L)
    ws = torch.full((max(4, need // 4),), float("nan"), device="cuda")
    call("ember_attn_kv4", *[p(x) for x in t], p(o), B, T, H, Hk, D, L, pos, S, scale,
         p(ws) if need else None, need, None)
    return host(o)


def attention_bounds(q, cache, scale, L):
    """Worst error of an output, and of the outputs' relative L2 norm.

    A score is step (q . c) + lo sum(q) with q in two f16 pieces: each term is off by at most 2^-22
    of itself, and the sums of D terms and the two products round D + 4 times, 2^-24 each, of the
    sum of magnitudes A = scale sum |q| (15 step + |lo|).  So a score is off by delta = A (2^-22 +
    (D + 4) 2^-24), a weight by exp(2 delta) - 1 of itself; the weight times step is held to 2^-22
    and the sums over up to L rows, with rescalings, merges and the division, add (L + 16) 2^-24 of
    the largest value.  The L2 norm averages: independent roundings add up as their square root,
    so sqrt(D) instead of D, and 2 sqrt(L) for L, leaves a factor of 4 for sums whose terms differ.
    """
    (kw, kp, _), (vw, vp, v) = cache
    D = q.shape[-1]
    vmax = np.abs(v[:, :, :L]).max()
    a = abs(scale) * np.abs(q).sum(-1).max() * (15 * kp[:, :, :L, 1] + np.abs(kp[:, :, :L, 0])).max()
    worst = vmax * (np.expm1(2 * a * (2.0 ** -22 + (D + 4) * HALF)) + 2.0 ** -22 + (L + 16) * HALF)
    l2 = 4 * HALF * (4 + a * np.sqrt(D) / 4 + 2 * np.sqrt(L))
    return float(worst), float(l2)


def check_attention(q, cache, L, pos, scale, got=None):
    got = attend(q, cache, L, pos, scale) if got is None else got
    ref = OQ.attention(q, cache[0][2], cache[1][2], pos, scale, L)
    worst, l2 = attention_bounds(q, cache, scale, L)
    assert np.isfinite(got).all()
    err = np.abs(got - ref)
    assert err.max() <= worst, (err.max(), worst)
    rel = np.linalg.norm(err) / np.linalg.norm(ref)
    assert rel <= l2, (rel, l2)
    return got


ATTEND = [  # B, T, H, Hk, D, L, pos, S
    (1, 1, 1, 1, 64, 1, 0, 1),              # one key
    (1, 1, 16, 8, 128, 2, 1, 8),
    (1, 1, 9, 3, 64, 257, 256, 300),        # group 3
    (1, 1, 16, 8, 128, 4096, 4095, 4096),   # split keys
    (2, 1, 32, 8, 64, 1000, 999, 1024),     # group 4
    (1, 1, 15, 3, 64, 63, 62, 64),          # group 5
    (1, 1, 17, 1, 128, 130, 129, 131),      # group 17
    (8, 1, 4, 4, 128, 33, 32, 40),          # no group
    (2, 7, 4, 2, 64, 40, 33, 48),           # a few tokens
    (1, 8, 16, 8, 128, 2010, 2002, 2100),
    (1, 16, 2, 1, 64, 31, 15, 31),          # 32 rows a KV head
    (1, 17, 3, 1, 128, 97, 80, 100),        # 51 rows
    (1, 64, 4, 2, 128, 64, 0, 64),          # a prompt from the start
    (1, 100, 6, 2, 64, 229, 129, 256),      # ragged rows and keys
    (2, 130, 4, 1, 128, 515, 385, 600),
    (1, 33, 8, 8, 64, 1025, 992, 1030),
    (1, 5, 4, 2, 64, 20, 40, 64),           # every row past L's last key
    (1, 40, 4, 2, 128, 30, 3, 64),          # keys end before the queries do
    (1, 300, 2, 2, 64, 700, 400, 701),      # ten tiles of 32 rows
]


@pytest.mark.parametrize("B,T,H,Hk,D,L,pos,S", ATTEND)
def test_attention_over_kv4(B, T, H, Hk, D, L, pos, S):
    r = rng(L + H + T)
    q = r.standard_normal((B, T, H, D)).astype(np.float32)
    cache = held_cache(r, B, Hk, S, D)
    got = check_attention(q, cache, L, pos, D ** -0.5)
    # what lies past a query's last row does not reach it: rows at and past L, and, for all but
    # the last query, the rows that only later ones see
    for w, par, _ in cache:
        par[:, :, L:] = np.nan
        w[:, :, L:] = 0xffffffff
    assert same(attend(q, cache, L, pos, D ** -0.5), got)  # and the same bits again
    if T > 1 and pos + T == L:
        cut = pos + T // 2
        for w, par, _ in cache:
            par[:, :, cut:] = np.nan
        part = attend(q, cache, L, pos, D ** -0.5)
        assert same(part[:, :T // 2], got[:, :T // 2])
        assert np.isnan(part[:, T // 2:]).all()


def attention64(q, k, v, pos, scale, L):
    """OQ.attention on the GPU, in 64 bits, for sizes that take a while in numpy."""
    q, k, v = (torch.from_numpy(np.ascontiguousarray(x)).cuda().double() for x in (q, k, v))
    B, T, H, D = q.shape
    g = H // k.shape[1]
    seen = torch.arange(L, device="cuda")[None] > (pos + torch.arange(T, device="cuda"))[:, None]
    o = torch.empty_like(q)
    for b in range(B):
        for h in range(H):
            z = q[b, :, h] @ k[b, h // g, :L].T.contiguous() * scale
            z[seen] = float("-inf")
            o[b, :, h] = torch.softmax(z, 1) @ v[b, h // g, :L]
    return o.cpu().numpy()


@pytest.mark.parametrize("B,T,H,Hk,D,L,pos,S", [
    (1, 600, 2, 2, 64, 28000, 27400, 28003),   # the shared tiles: 600 rows, ragged
    (1, 2050, 4, 2, 128, 4200, 2150, 4200),    # 4100 rows
    (2, 259, 2, 1, 128, 32500, 32241, 32500),  # the last tile holds 6 rows
    (1, 4099, 1, 1, 64, 4099, 0, 4099),        # a whole prompt
])
def test_attention_of_long_chunks(B, T, H, Hk, D, L, pos, S):
    r = rng(T)
    q = r.standard_normal((B, T, H, D)).astype(np.float32)
    cache = held_cache(r, B, Hk, S, D)
    got = attend(q, cache, L, pos, D ** -0.5)
    ref = attention64(q, cache[0][2], cache[1][2], pos, D ** -0.5, L)
    worst, l2 = attention_bounds(q, cache, D ** -0.5, L)
    err = np.abs(got - ref)
    assert err.max() <= worst and np.linalg.norm(err) <= l2 * np.linalg.norm(ref)
    # rows that only later queries see, and rows past the last, do not reach a query
    cut = pos + T // 2
    for _, par, _ in cache:
        par[:, :, cut:] = np.nan
    part = attend(q, cache, L, pos, D ** -0.5)
    assert same(part[:, :T // 2], got[:, :T // 2]) and np.isnan(part[:, T // 2:]).all()


@pytest.mark.parametrize("T", [1, 6, 70])
def test_attention_of_unlike_sizes(T):
    """Queries and rows of very different magnitude: the f16 pieces are scaled per row."""
    r = rng(T)
    B, H, Hk, D, L = 1, 4, 2, 128, 200
    q = r.standard_normal((B, T, H, D)).astype(np.float32)
    q *= np.exp2(r.integers(-60, 3, (B, T, H, 1))).astype(np.float32)
    q[0, 0, 0] = 0
    q[0, 0, 1, ::3] *= np.float32(1e-20)
    cache = held_cache(r, B, Hk, L, D)
    # value rows of sizes from 2^-60 to 2^60, key by key
    size = np.exp2(r.integers(-60, 61, (B, Hk, L, 1))).astype(np.float32)
    w, par, v = cache[1]
    cache[1] = (w, (par * size).astype(np.float32), v * size)
    check_attention(q, cache, L, L - T, D ** -0.5)


@pytest.mark.parametrize("T", [1, 40])
@pytest.mark.parametrize("scale", [0.0, -0.125, 30.0])
def test_attention_scales(T, scale):
    r = rng(5)
    q = r.standard_normal((1, T, 4, 64)).astype(np.float32) * np.float32(0.3)
    cache = held_cache(r, 1, 2, 90, 64)
    check_attention(q, cache, 90, 90 - T, scale)


@pytest.mark.parametrize("T", [1, 40])
def test_attention_rows_that_are_not_finite_reach_only_who_sees_them(T):
    r = rng(6)
    B, H, Hk, D, L = 2, 4, 2, 64, 150
    q = r.standard_normal((B, T, H, D)).astype(np.float32)
    cache = held_cache(r, B, Hk, L, D)
    clean = attend(q, cache, L, L - T, 0.125)
    cache[0][1][1, 0, 9] = np.nan   # a key of (sequence 1, KV head 0)
    cache[1][1][0, 1, 20] = np.nan  # a value of (sequence 0, KV head 1)
    got = attend(q, cache, L, L - T, 0.125)
    bad = np.zeros((B, T, H, D), bool)
    bad[1, :, :2] = bad[0, :, 2:] = True
    assert np.isnan(got[bad]).all() and same(got[~bad], clean[~bad])
    q[0, T - 1, 1, 5] = np.inf      # and a query
    got = attend(q, cache, L, L - T, 0.125)
    bad[0, T - 1, 1] = True
    assert np.isnan(got[bad]).all() and same(got[~bad], clean[~bad])


@pytest.mark.parametrize("T", [1, 20, 90])
def test_attention_whole_blocks_of_not_finite_rows(T):
    """A split, or a wave's share of one, in which no score is a number still reaches the result."""
    r = rng(7)
    H, Hk, D, L = 2, 2, 128, 1700
    q = r.standard_normal((1, T, H, D)).astype(np.float32)
    cache = held_cache(r, 1, Hk, L, D)
    cache[0][1][0, 1, 600:1300] = np.nan
    got = attend(q, cache, L, L - T, 0.1)
    assert np.isnan(got[:, :, 1]).all() and np.isfinite(got[:, :, 0]).all()


@pytest.mark.parametrize("T,L", [(1, 3000), (3, 700), (96, 1200)])
def test_attention_captured_and_on_another_stream(T, L):
    """A captured call replays to the eager result, with eager work between the replays."""
    r = rng(T)
    B, H, Hk, D = 1, 8, 2, 128
    q = r.standard_normal((B, T, H, D)).astype(np.float32)
    cache = held_cache(r, B, Hk, L, D)
    want = attend(q, cache, L, L - T, 0.1)
    t = [dev(q), words(cache[0][0]), dev(cache[0][1]), words(cache[1][0]), dev(cache[1][1])]
    o = empty((B, T, H, D))
    need = capi.lib().ember_attn_kv4_workspace_bytes(B, T, H, Hk, D, L)
    ws = empty((max(4, need // 4),))

    def go():
        st = C.c_void_p(torch.cuda.current_stream().cuda_stream)
        capi.call("ember_attn_kv4", *[p(x) for x in t], p(o), B, T, H, Hk, D, L, L - T, L, 0.1,
                  p(ws) if need else None, need, st)

    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        go()
    side.synchronize()
    assert same(host(o), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go()
    for _ in range(3):
        o.fill_(0)
        ws.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        assert same(host(o), want)
        go()
        assert same(host(o), want)
    t[0].mul_(0.5)  # new queries in the captured buffers
    graph.replay()
    assert same(host(o), attend(q * np.float32(0.5), cache, L, L - T, 0.1))


def test_kv4_cache_past_int32_offsets():
    """Rows whose words lie past 2^31: written, and seen by a query over the whole cache.  All other
    rows hold zeros, so the output is (sum e^s_j v_j) / (S - 3 + sum e^s_j) over the three."""
    r = rng(8)
    D, H, S, T = 128, 2, 2 ** 27 + 40, 3
    kc, vc = (torch.zeros(S * D // 8, device="cuda", dtype=torch.int32) for _ in range(2))
    kp, vp = (torch.zeros(S * 2, device="cuda") for _ in range(2))
    k, v = (r.standard_normal((1, T, 1, D)).astype(np.float32) for _ in range(2))
    kd, vd = dev(k), dev(v)
    call("ember_kv4_write", p(kd), p(vd), p(kc), p(kp), p(vc), p(vp), 1, T, 1, D, S, S - T, None)
    q = np.stack([k[0, 0, 0] * f for f in (1.0, 1.6)])[None, None].astype(np.float32)
    qd, o = dev(q), empty((1, 1, H, D))
    need = capi.lib().ember_attn_kv4_workspace_bytes(1, 1, H, 1, D, S)
    ws = empty((need // 4,))
    call("ember_attn_kv4", p(qd), p(kc), p(kp), p(vc), p(vp), p(o), 1, 1, H, 1, D, S, S - 1, S,
         0.15, p(ws), need, None)
    held = [OQ.values(*OQ.quantise(x[0, :, 0], 15)) for x in (k, v)]
    e = np.exp(q[0, 0].astype(np.float64) @ held[0].T * 0.15)
    ref = e @ held[1] / (S - T + e.sum(1))[:, None]
    # the rows before add 2^27 ones in splits of fp32 sums of at most 2^18 / 16 terms per lane
    assert np.abs(host(o)[0, 0] - ref).max() <= 1e-3 * np.abs(ref).max()


# --------------------------------------------------------------------------- 8-bit rows
ROWS = [(2100, 36), (2050, 300), (2049, 1030), (2048, 2500), (1, 1), (3, 7), (5, 64), (2, 127), (4, 128), (7, 129), (3, 200), (11, 576), (6, 960),
        (5, 1001), (4, 2048), (2, 5000), (600, 36), (2, 8200), (2048, 17), (2060, 100)]


def quantised(x, offset=0):
    """The 8-bit form of x [rows, H]; `offset` floats shift x's address."""
    rows, H = x.shape
    flat = torch.zeros(x.size + offset, device="cuda")
    flat[offset:] = dev(x).reshape(-1)
    lib = capi.lib()
    codes = torch.full((lib.ember_q8_code_bytes(rows, H),), 9, device="cuda", dtype=torch.uint8)
    params = torch.full((lib.ember_q8_param_bytes(rows, H) // 4,), 9.0, device="cuda")
    call("ember_q8_quantize", p(flat[offset:]), p(codes), p(params), rows, H, None)
    return codes, params


@pytest.mark.parametrize("rows,H", ROWS)
@pytest.mark.parametrize("offset", [0, 1])
def test_q8_rows(rows, H, offset):
    r = rng(rows + H)
    x = odd_rows(rows_like_keys(r, rows, H), r) if H > 3 else rows_like_keys(r, rows, H)
    codes, params = quantised(x, offset)
    ref_c, ref_p = OQ.quantise_rows8(x)
    assert same(host(params).reshape(ref_p.shape), ref_p)
    assert same(host(codes).reshape(ref_c.shape), ref_c)
    ref = OQ.values_rows8(ref_c, ref_p, H)
    guard = torch.full((rows * H + 8,), 5.0, device="cuda")
    out = guard[offset:offset + rows * H]
    call("ember_q8_dequantize", p(codes), p(params), p(out), rows, H, None)
    close_roundings(host(out).reshape(rows, H), ref)
    assert (host(guard)[:offset] == 5).all() and (host(guard)[offset + rows * H:] == 5).all()


@pytest.mark.parametrize("rows,H", ROWS)
@pytest.mark.parametrize("offset", [0, 1])
def test_q8_rows_and_their_norm(rows, H, offset):
    r = rng(rows + H)
    x = rows_like_keys(r, rows, H)
    if rows > 2:
        x[1] = 0
        x[2, H // 2] = np.nan
    w = (1 + 0.1 * r.standard_normal(H)).astype(np.float32)
    eps = 1e-5
    codes, params = quantised(x)
    bufs = [torch.full((rows * H + 8,), 5.0, device="cuda") for _ in range(2)]
    xo, y = (b[offset:offset + rows * H] for b in bufs)
    rstd = empty((rows,))
    wd = dev(w)
    args = (p(codes), p(params), p(wd), p(xo), p(y))
    call("ember_q8_dequantize_rmsnorm", *args, p(rstd), rows, H, eps, None)
    plain = empty((rows, H))
    call("ember_q8_dequantize", p(codes), p(params), p(plain), rows, H, None)
    assert same(host(xo).reshape(rows, H), host(plain))
    ref_c, ref_p = OQ.quantise_rows8(x)
    v = OQ.values_rows8(ref_c, ref_p, H)
    ref = 1 / np.sqrt((v * v).mean(1) + eps)
    # the squares carry 2 roundings of x, the sum at most H, the mean, the sum with eps, the root
    # (which halves all of it) and the quotient
    close_roundings(host(rstd), ref, (H + 5) / 2 + 2)
    close_roundings(host(y).reshape(rows, H), v * ref[:, None] * w, (H + 5) / 2 + 5)
    first = host(y)
    for b in bufs:
        assert (host(b)[:offset] == 5).all() and (host(b)[offset + rows * H:] == 5).all()
    call("ember_q8_dequantize_rmsnorm", *args, None, rows, H, eps, None)
    assert same(host(y), first)


def test_q8_rows_past_int32_offsets():
    rows, H = 2 ** 20 + 3, 2048
    x = torch.randn((rows, H), device="cuda")
    lib = capi.lib()
    codes = torch.empty(lib.ember_q8_code_bytes(rows, H), device="cuda", dtype=torch.uint8)
    params = torch.empty(lib.ember_q8_param_bytes(rows, H) // 4, device="cuda")
    call("ember_q8_quantize", p(x), p(codes), p(params), rows, H, None)
    tail = host(x[-4:])
    ref_c, ref_p = OQ.quantise_rows8(tail)
    assert same(host(codes[-4 * H:]).reshape(4, H), ref_c)
    assert same(host(params[-4 * 32:]).reshape(ref_p.shape), ref_p)
    x.zero_()
    call("ember_q8_dequantize", p(codes), p(params), p(x), rows, H, None)
    close_roundings(host(x[-4:]), OQ.values_rows8(ref_c, ref_p, H))
    y, w = torch.zeros_like(x), torch.ones(H, device="cuda")
    x.zero_()
    call("ember_q8_dequantize_rmsnorm", p(codes), p(params), p(w), p(x), p(y), None, rows, H, 0.0,
         None)
    v = OQ.values_rows8(ref_c, ref_p, H)
    close_roundings(host(x[-4:]), v)
    close_roundings(host(y[-4:]), v / np.sqrt((v * v).mean(1, keepdims=True)), H / 2 + 8)


def test_q8_rows_of_more_than_one_launch():
    rows, H = 2 ** 22 + 37, 8  # the second launch restores 37 rows
    r = rng(5)
    x = rows_like_keys(r, rows, H)
    w = (1 + 0.1 * r.standard_normal(H)).astype(np.float32)
    codes, params = quantised(x)
    out, xo, y = (torch.full((rows, H), 5.0, device="cuda") for _ in range(3))
    rstd, wd = torch.full((rows,), 5.0, device="cuda"), dev(w)
    call("ember_q8_dequantize", p(codes), p(params), p(out), rows, H, None)
    call("ember_q8_dequantize_rmsnorm", p(codes), p(params), p(wd), p(xo), p(y), p(rstd), rows, H,
         1e-5, None)
    assert torch.equal(out, xo)
    v = OQ.values_rows8(*OQ.quantise_rows8(x), H)
    close_roundings(host(xo), v)
    ref = 1 / np.sqrt((v * v).mean(1) + 1e-5)
    close_roundings(host(rstd), ref, (H + 5) / 2 + 2)  # as in test_q8_rows_and_their_norm
    close_roundings(host(y), v * ref[:, None] * w, (H + 5) / 2 + 5)
