"""The attention over a 4-bit cache where values are very large, very small or all alike, what a
query's bits may depend on, and the forms of the few-bit kernels that only large calls take."""
import numpy as np
import pytest

from oracle import quant as OQ
from tests.helpers import call, empty, host, p

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from emberlm_amd import capi  # noqa: E402
from tests.test_gpu_quant import (attend, attention64, attention_bounds, check_attention,  # noqa: E402
                                  close_roundings, held_cache, same)
from tests.test_gpu_quant_model import test_decode_attention_kv4_fold as decode_step  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.cuda.init()


def rng(s=0):
    return np.random.default_rng(s)


def held(x):
    """A cache tensor's buffers and what it holds, of x [B, Hk, S, D]."""
    codes, params = OQ.quantise(x.astype(np.float32), 15)
    return OQ.pack4(codes), params, OQ.values(codes, params)


# ------------------------------------------------------- a query and its neighbours
@pytest.mark.parametrize("B,T,H,Hk,D,L", [
    (1, 16, 2, 2, 128, 512),      # one workgroup of eight waves per head
    (4, 16, 8, 8, 64, 4096),      # one query tile, key splits
    (4, 16, 16, 8, 128, 4096),    # two
    (1, 600, 1, 1, 64, 28000),    # shared tiles
    (1, 600, 1, 1, 128, 28000),
])
def test_a_key_that_only_the_last_query_sees_moves_no_other_bit(B, T, H, Hk, D, L):
    """Every query's scores rise by 3 (log2 units) among the last keys, less than lets its reference
    move; the last key lifts the last query's score by a hundred, and that one's reference."""
    r = rng(D + T)
    d = r.standard_normal(D)
    d /= np.linalg.norm(d)
    q = (4 * d + 0.05 * r.standard_normal((B, T, H, D))).astype(np.float32)
    rise = np.zeros(L)
    rise[L - T:] = 3 * np.log(2) / 4
    k = rise[:, None] * d + 0.02 * r.standard_normal((B, Hk, L, D))
    v = held(r.standard_normal((B, Hk, L, D)))
    quiet = attend(q, [held(k), v], L, L - T, 1.0)
    k[:, :, L - 1] = 25 * d
    loud = [held(k), v]
    got = attend(q, loud, L, L - T, 1.0)
    assert same(got[:, :-1], quiet[:, :-1])
    ref = attention64(q, loud[0][2], v[2], L - T, 1.0, L)
    worst, _ = attention_bounds(q, loud, 1.0, L)
    assert np.abs(got - ref).max() <= worst
    assert np.abs(got[:, -1] - quiet[:, -1]).max() > 0.1


# ---------------------------------------------------------------- sizes of value rows
def check_values(r, v, T, scale=None, Hk=2, G=2, D=64):
    """Queries and keys of the usual size over the value rows v [1, Hk, L, D]."""
    L = v.shape[2]
    q = r.standard_normal((1, T, G * Hk, D)).astype(np.float32)
    cache = [held(r.standard_normal((1, Hk, L, D))), held(v)]
    return check_attention(q, cache, L, L - T, D ** -0.5 if scale is None else scale)


@pytest.mark.parametrize("T,L", [(1, 1), (1, 300), (1, 3000), (20, 40), (70, 3000)])
@pytest.mark.parametrize("power", [-100, -30, 20, 53, 60, 70, 99])
def test_value_rows_of_equal_values(T, L, power):
    """Rows without a step, held as they are: all of one size, and of sizes around it."""
    r = rng(T + L)
    v = np.ones((1, 2, L, 64)) * np.exp2(float(power))
    check_values(r, v, T)
    sign = r.choice([-1.0, 1.0], (1, 2, L, 1))
    check_values(r, v * sign * np.exp2(-r.integers(0, 10, (1, 2, L, 1)).astype(float)), T)


@pytest.mark.parametrize("L", [256, 512, 4096])
@pytest.mark.parametrize("T", [1, 3, 40])
@pytest.mark.parametrize("first,last", [(0, 98), (98, 0), (-80, 98), (-90, 90), (-80, 50)])
@pytest.mark.parametrize("equal", [True, False])
def test_value_rows_of_two_sizes(T, L, first, last, equal):
    """The first half of the keys (or every other run of 128) carries rows of one size, the rest of
    another: the smaller ones count in the weights' sum as much as the larger."""
    r = rng(T + L)
    for large in (np.arange(L) >= L // 2, np.arange(L) // 128 % 2 == 1):
        size = np.exp2(np.where(large, last, first).astype(float))[:, None]
        v = r.standard_normal((1, 2, L, 64)) * size / 8
        if equal:
            small = ~large if first < last else large
            v[:, :, small] = np.exp2(float(min(first, last)))
        check_values(r, v, T, scale=0.05)


@pytest.mark.parametrize("T", [600])
@pytest.mark.parametrize("first,last", [(0, 98), (-80, 90)])
def test_value_rows_of_two_sizes_shared_tiles(T, first, last):
    r = rng(T)
    L, D = 28000, 64
    v = r.standard_normal((1, 1, L, D)) / 8
    v[:, :, :L // 2] = 1
    v *= np.exp2(np.where(np.arange(L) < L // 2, first, last).astype(float))[:, None]
    q = r.standard_normal((1, T, 1, D)).astype(np.float32)
    cache = [held(r.standard_normal((1, 1, L, D))), held(v)]
    got = attend(q, cache, L, L - T, 0.05)
    ref = attention64(q, cache[0][2], cache[1][2], L - T, 0.05, L)
    worst, l2 = attention_bounds(q, cache, 0.05, L)
    err = np.abs(got - ref)
    assert err.max() <= worst and np.linalg.norm(err) <= l2 * np.linalg.norm(ref)


@pytest.mark.parametrize("T,L", [(1, 1), (1, 300), (1, 3000), (20, 40), (70, 3000)])
@pytest.mark.parametrize("power", [-80, -70, -61, 60, 96])
def test_value_rows_all_of_one_size(T, L, power):
    r = rng(T + L)
    check_values(r, r.standard_normal((1, 2, L, 64)) * np.exp2(float(power)), T)


@pytest.mark.parametrize("T,L", [(1, 1), (1, 300), (1, 4096), (20, 40), (16, 512), (70, 3000)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_scores_near_the_largest_that_are_taken(T, L, D, sign):
    """Scores up to 2^21 in steps of some hundreds: each query's output is the value row of its
    largest score, to the weights' 22 bits and the sums' roundings.  Value rows differ in size."""
    r = rng(T + L)
    B, H, Hk = 1, 4, 2
    q = np.abs(r.standard_normal((B, T, H, D))) + 0.5
    k = np.ones((B, Hk, L, D)) + 0.001 * r.standard_normal((B, Hk, L, D))
    level = np.stack([r.permutation(L) for _ in range(Hk)]).reshape(B, Hk, L, 1)
    k *= 1 + level / L  # the order of a query's scores is that of the levels
    q, cache = q.astype(np.float32), [held(k), None]
    v = r.standard_normal((B, Hk, L, D)) * np.exp2(r.integers(-40, 40, (B, Hk, L, 1)).astype(float))
    cache[1] = held(v)
    top = np.einsum("bthd,bhld->bthl", q.astype(np.float64).reshape(B, T, Hk * 2, D),
                    np.repeat(cache[0][2], 2, 1)).max()
    scale = sign * 0.99 * 2.0 ** 21 / top
    got = attend(q, cache, L, L - T, scale)
    for t in range(T):
        n = L - T + t + 1
        for h in range(H):
            kk, vv = cache[0][2][0, h // 2, :n], cache[1][2][0, h // 2, :n]
            s = kk @ q[0, t, h].astype(np.float64) * scale
            j = s.argmax()
            others = np.delete(s, j)
            if others.size and s[j] - others.max() < 120:  # not this one's alone
                continue
            tol = (2.0 ** -22 + 30 * 2.0 ** -24) * (np.abs(vv[j]).max() + 16 * cache[1][1][0, h // 2, j, 1])
            assert np.abs(got[0, t, h] - vv[j]).max() <= tol, (t, h, j)
    assert np.isfinite(got).all()


# ------------------------------------------------------------- forms of large calls
@pytest.mark.parametrize("B,T,H,Hk,D,L,splits", [
    (2, 1024, 32, 8, 64, 6000, 1),    # shared tiles, the output stored by themselves
    (2, 2045, 16, 8, 128, 9003, 1),
    (1, 8200, 16, 8, 128, 8200, 1),   # a whole prompt
    (2, 1021, 16, 8, 128, 17003, 2),  # few splits, merged by a wave per row
    (4, 16, 16, 8, 128, 300, 3),
    (2, 64, 8, 4, 64, 900, 8),
])
def test_attention_of_few_or_no_key_splits(B, T, H, Hk, D, L, splits):
    need = capi.lib().ember_attn_kv4_workspace_bytes(B, T, H, Hk, D, L)
    assert need == (0 if splits == 1 else B * T * H * splits * (D + 2) * 4)
    r = rng(T)
    q = r.standard_normal((B, T, H, D)).astype(np.float32)
    cache = held_cache(r, B, Hk, L, D)
    got = attend(q, cache, L, L - T, D ** -0.5)
    ref = attention64(q, cache[0][2], cache[1][2], L - T, D ** -0.5, L)
    worst, l2 = attention_bounds(q, cache, D ** -0.5, L)
    err = np.abs(got - ref)
    assert err.max() <= worst and np.linalg.norm(err) <= l2 * np.linalg.norm(ref)


@pytest.mark.parametrize("B,T,H,Hk,D,pos,S,qk,factor", [
    (1, 1, 9, 3, 64, 700, 800, True, 0.0),     # heads of 64 over split keys
    (2, 2, 8, 2, 64, 1027, 1030, False, 32.0),
    (1, 1, 32, 8, 64, 6000, 6001, False, 0.0),
])
def test_decode_step_of_split_keys(B, T, H, Hk, D, pos, S, qk, factor):
    assert capi.lib().ember_attn_kv4_workspace_bytes(B, T, H, Hk, D, pos + T) > 0
    decode_step(B, T, H, Hk, D, pos, S, qk, factor)


def test_kv4_write_and_read_of_more_rows_than_32_bits_number():
    """2^31 + 10 head rows of 8 values written in one call, and read back as 2^32 + 20 pieces of
    four.  Rows are checked at the ends, beside 2^31 and at random."""
    torch.cuda.empty_cache()
    T, Hk, D = 2 ** 30 + 5, 2, 8
    rows = T * Hk
    x = torch.empty(rows * D, device="cuda")
    gen = torch.Generator(device="cuda")
    gen.manual_seed(3)
    for a in range(0, x.numel(), 2 ** 30):
        x[a:a + 2 ** 30].normal_(generator=gen)
    x = x.view(T, Hk, D)
    kc, vc = (torch.zeros(rows, device="cuda", dtype=torch.int32) for _ in range(2))
    kp, vp = (torch.zeros(rows * 2, device="cuda") for _ in range(2))
    call("ember_kv4_write", p(x), p(x), p(kc), p(kp), p(vc), p(vp), 1, T, Hk, D, T, 0, None)
    t = np.unique(np.concatenate([np.arange(40), 2 ** 29 + np.arange(-20, 20), T - 1 - np.arange(40),
                                  rng(1).integers(0, T, 2000)]))
    ti = torch.from_numpy(t).cuda()
    codes, params = OQ.quantise(host(x[ti]).transpose(1, 0, 2), 15)
    for c, par in ((kc, kp), (vc, vp)):
        assert same(host(c.view(Hk, T)[:, ti]).view(np.uint32), OQ.pack4(codes)[..., 0])
        assert same(host(par.view(Hk, T, 2)[:, ti]), params)
    # every row of both tensors is written, and alike
    assert torch.equal(kc, vc) and torch.equal(kp, vp)
    assert bool((kp.view(-1, 2)[:, 1] > 0).all())
    del x, vc, vp
    out = empty((Hk, T, D))
    call("ember_kv4_read_expanded", p(kc), p(kp), p(out), 1, Hk, 1, T, D, T, None)
    close_roundings(host(out[:, ti]), OQ.values(codes, params))
    del out, kc, kp
    torch.cuda.empty_cache()
