"""Weights held in 4 bits, as calls that can be timed and checked.

A weight [N, K] is held in microscaled 4-bit floating point: each row in groups of 32 values, one
scale per group, a power of two kept in a byte, and per value a code of a sign and one of the sizes
0, 1/2, 1, 3/2, 2, 3, 4, 6.  The scale is the smallest power of two that the group's largest size is
at most 7 times of (2^-127 at least), a value takes the size nearest to its quotient by the scale, the
one of an even code where two are as near, and 6 above that.

  hold      a weight is brought into that form and read back
  lookup    rows of an embedding table held so, for a list of token ids
  linear    up to three products of the same rows x with weights held so, y = W x (+ a residual),
            x through an RMSNorm first where there is one: from one token to a long prompt
  gateup    the input half of a SwiGLU block, silu(Wg x) * (Wu x), x through an RMSNorm first

The form in memory: tiles of 32 rows by 64 columns, 1024 bytes each, a row of tiles after another.
Byte 16 * (32 * h + r) + i of a tile holds columns 32 * h + 2 * i (low half) and 32 * h + 2 * i + 1 of its
row r.  Scales: 256 bytes for 32 rows by 256 columns, byte 4 * (32 * h + r) + c for row r and columns
64 * c + 32 * h and up.  Rows and columns that fill the last tiles up are zeros of scale 2^-127.
"""
import ctypes as C
import math

import torch

own = False

GROUP = 32
SIZES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _hold(N, K):
    return {"kind": "hold", "N": N, "K": K}


def _lookup(n, V, K):
    return {"kind": "lookup", "n": n, "V": V, "K": K}


def _linear(M, K, N, norm=False, residual=False):
    """N: the weights' rows, as text: "2048" or "2048,1024,1024"."""
    return {"kind": "linear", "M": M, "K": K, "N": N, "norm": norm, "residual": residual}


def _gateup(M, K, I, norm=True):
    return {"kind": "gateup", "M": M, "K": K, "I": I, "norm": norm}


def listed():
    return [
        # a small weight whose rows and columns fill no tile
        dict(_hold(131, 1001), name="hold_131x1001"),
        # a model's embedding table as it is loaded, Qwen3-1.7B
        dict(_hold(151936, 2048), name="hold_qwen3_table"),
        # the token of a decode step, SmolLM2 table
        dict(_lookup(1, 49152, 576), name="lookup_smollm2_1"),
        # a long prompt's tokens, Qwen3-1.7B table
        dict(_lookup(4096, 151936, 2048), name="lookup_qwen3_4096"),
        # Q, K and V of one token, SmolLM2-135M
        dict(_linear(1, 576, "576,192,192", norm=True), name="linear_smollm2_qkv_m1"),
        # the LM head of one token, Qwen3-1.7B
        dict(_linear(1, 2048, "151936", norm=True), name="linear_qwen3_head_m1"),
        # the MLP's output half for eight conversations, LLaMA-3.2-1B
        dict(_linear(8, 8192, "2048", residual=True), name="linear_llama_down_m8"),
        # a short turn through a weight whose sizes are no whole groups or tiles
        dict(_linear(33, 1001, "577"), name="linear_odd_m33"),
        # the MLP's output half for a long prompt, Qwen3-1.7B
        dict(_linear(4096, 6144, "2048", residual=True), name="linear_qwen3_down_m4096"),
        # the MLP's input half of one token, Qwen3-1.7B
        dict(_gateup(1, 2048, 6144), name="gateup_qwen3_m1"),
        # a chat turn's tokens, SmolLM2-135M
        dict(_gateup(509, 576, 1536), name="gateup_smollm2_m509"),
        # a prompt's tokens, Qwen3-1.7B
        dict(_gateup(2048, 2048, 6144), name="gateup_qwen3_m2048"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["hold", "lookup", "linear", "linear", "linear", "gateup", "gateup"])
    K = rng.choice([576, 960, 1024, 2048, 6144]) if rng.random() < 0.5 else _log(rng, 1, 8192)
    if kind == "hold":
        return _hold(_log(rng, 1, min(151936, (1 << 28) // K)), K)
    if kind == "lookup":
        return _lookup(_log(rng, 1, 8192), _log(rng, 1, min(151936, (1 << 28) // K)), K)
    M = rng.randint(1, 8) if rng.random() < 0.5 else _log(rng, 9, 4096)
    most = min(16384, (1 << 35) // (M * K), (1 << 27) // K)
    norm = rng.random() < 0.6
    if kind == "gateup":
        return _gateup(M, K, _log(rng, 1, max(1, most // 2)), norm)
    count = rng.choice([1, 1, 2, 3])
    N = [_log(rng, 1, max(1, most // count)) for _ in range(count)]
    return _linear(M, K, ",".join(map(str, N)), norm, rng.random() < 0.5)


def _rows_of(case):
    return [int(n) for n in case["N"].split(",")] if case["kind"] == "linear" else [case["I"]] * 2


# ---------------------------------------------------------------------- plain form
def _padded(t, rows, cols):
    """t [n, k] in the corner of zeros, both sizes brought up to multiples."""
    n, k = t.shape
    out = torch.zeros((-(-n // rows) * rows, -(-k // cols) * cols), dtype=t.dtype, device=t.device)
    out[:n, :k] = t
    return out


def _quantise(w):
    """Codes [N', K'] (uint8) and scale bytes [N', K' / 32] of w [N, K], filled up to whole tiles."""
    w = _padded(w, 32, 64).unflatten(1, (-1, GROUP))
    bits = w.abs().amax(2).view(torch.int32)
    # the exponent of the largest size, one up where its mantissa is above 1.75
    scale = (((bits + 0x1FFFFF) >> 23) - 2).clamp(min=0)
    bad = bits >= 0x7F800000
    q = torch.ldexp(w.double().abs(), (127 - scale).unsqueeze(2))
    code = torch.zeros_like(q, dtype=torch.uint8)
    for i in range(7):
        border = (SIZES[i] + SIZES[i + 1]) / 2
        # a border value goes to the even code of the two beside it
        code += (q >= border) if i % 2 else (q > border)
    code += 8 * torch.signbit(w).to(torch.uint8)
    code[bad] = 0
    scale = torch.where(bad, torch.full_like(scale, 255), scale)
    return code.flatten(1), scale.to(torch.uint8)


def _tiles(code, scale):
    """The form in memory of codes and scale bytes."""
    n, k = code.shape
    both = (code[:, 0::2] | (code[:, 1::2] << 4)).view(n // 32, 32, k // 64, 2, 16)
    codes = both.permute(0, 2, 3, 1, 4).contiguous()
    scale = _padded(scale, 32, 8).view(n // 32, 32, -1, 4, 2)
    return codes, scale.permute(0, 2, 4, 1, 3).contiguous()


def _held(w):
    return _tiles(*_quantise(w))


def _values(held, N, K):
    """The fp32 values [N, K] of a held weight (or of single rows of its tiles)."""
    codes, scales = held
    nb, kb, _, r = codes.shape[:4]
    table = torch.tensor(SIZES + tuple(-v for v in SIZES), device=codes.device)
    both = codes.permute(0, 3, 1, 2, 4)  # [nb, r, kb, 2, 16]
    vals = torch.stack([table[(both & 15).long()], table[(both >> 4).long()]], -1).flatten(4)
    scale = scales.permute(0, 3, 1, 4, 2).reshape(nb, r, -1, 2)[:, :, :kb].int()
    vals = torch.ldexp(vals, (scale - 127).unsqueeze(-1))
    vals = torch.where((scale == 255).unsqueeze(-1), math.nan, vals)
    return vals.reshape(nb * r, kb * 64)[:N, :K]


def _normed(s, x):
    if not s["case"]["norm"]:
        return x
    return x * (torch.rsqrt((x * x).mean(1, keepdim=True) + s["eps"]) * s["norm_w"])


def _plain(s):
    c = s["case"]
    if c["kind"] == "hold":
        return {"w": _values(_held(s["w"]), c["N"], c["K"]).contiguous()}
    if c["kind"] == "lookup":
        nb, r = s["ids"] // 32, s["ids"] % 32
        codes, scales = s["table"]
        one = (codes[nb, :, :, r].unsqueeze(3), scales[nb, :, :, r].unsqueeze(3))
        return {"x": _values(one, c["n"], c["K"]).contiguous()}
    x = _normed(s, s["x"])
    y = [torch.mm(x, _values(w, N, c["K"]).t()) for w, N in zip(s["weights"], _rows_of(c))]
    if c["kind"] == "gateup":
        g, u = y
        return {"h": g / (1 + torch.exp(-g)) * u}
    if c["residual"]:
        y = [r + v for r, v in zip(s["residual"], y)]
    return {"y%d" % i: v for i, v in enumerate(y)}


# ----------------------------------------------------------------- the framework's calls
def _p(t):
    return C.c_void_p(t.data_ptr())


def _ptrs(ts):
    return (C.c_void_p * len(ts))(*[t.data_ptr() for t in ts])


def _own(s):
    from emberlm_amd import capi
    c, lib = s["case"], capi.lib()
    st = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    new = lambda *shape: torch.empty(shape, device="cuda")  # noqa: E731
    raw = lambda n: torch.empty(n, device="cuda", dtype=torch.uint8)  # noqa: E731
    if c["kind"] == "hold":
        N, K = c["N"], c["K"]
        codes = raw(lib.ember_mx4_code_bytes(N, K))
        scales = raw(lib.ember_mx4_scale_bytes(N, K))
        w = new(N, K)
        capi.call("ember_mx4_quantize", _p(s["w"]), _p(codes), _p(scales), N, K, st)
        capi.call("ember_mx4_dequantize", _p(codes), _p(scales), _p(w), N, K, st)
        return {"w": w}
    if c["kind"] == "lookup":
        x = new(c["n"], c["K"])
        capi.call("ember_mx4_embedding", _p(s["ids"]), _p(s["table"][0]), _p(s["table"][1]), _p(x),
                  c["n"], c["K"], c["V"], st)
        return {"x": x}
    M, K, N = c["M"], c["K"], _rows_of(c)
    need = lib.ember_mx4_workspace_bytes(M, K, sum(N))
    ws = raw(need) if need else None
    norm_w = _p(s["norm_w"]) if c["norm"] else None
    if c["kind"] == "gateup":
        h = new(M, N[0])
        g, u = s["weights"]
        capi.call("ember_mx4_gateup", _p(s["x"]), M, K, norm_w, s["eps"], _p(g[0]), _p(g[1]),
                  _p(u[0]), _p(u[1]), N[0], _p(h), _p(ws) if need else None, need, st)
        return {"h": h}
    y = [new(M, n) for n in N]
    capi.call("ember_mx4_linear", _p(s["x"]), M, K, norm_w, s["eps"], len(N),
              _ptrs([w[0] for w in s["weights"]]), _ptrs([w[1] for w in s["weights"]]),
              (C.c_int64 * len(N))(*N), _ptrs(y), _ptrs(s["residual"]) if c["residual"] else None,
              _p(ws) if need else None, need, st)
    return {"y%d" % i: v for i, v in enumerate(y)}


def run(state):
    return _own(state) if own else _plain(state)


# --------------------------------------------------------------------------- inputs
def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    rand = lambda *shape: torch.randn(shape, generator=gen, device="cuda")  # noqa: E731

    def weight(N, K):
        """Rows and columns of unlike size, as trained weights have them."""
        return rand(N, K) * (0.03 * torch.exp(0.4 * rand(N, 1)) * torch.exp(0.4 * rand(K)))

    s = {"case": c}
    if c["kind"] == "hold":
        s["w"] = weight(c["N"], c["K"])
        return s
    if c["kind"] == "lookup":
        s["table"] = _held(weight(c["V"], c["K"]))
        s["ids"] = torch.randint(c["V"], (c["n"],), generator=gen, device="cuda")
        return s
    M, K = c["M"], c["K"]
    if c["norm"]:  # a residual stream: channels of unlike size, a few of them far larger
        s["x"] = rand(M, K) * torch.exp(rand(K)) + 0.3 * rand(K)
        s["norm_w"] = 1 + 0.1 * rand(K)
    else:  # a product of two activations
        s["x"] = rand(M, K) * rand(M, K)
    s["eps"] = 1e-5
    s["weights"] = [_held(weight(n, K)) for n in _rows_of(c)]
    if c["kind"] == "linear" and c["residual"]:
        s["residual"] = [rand(M, n) for n in _rows_of(c)]
    return s


def work(case):
    c = case
    held = lambda n, k: n * (k / 2 + -(-k // GROUP))  # noqa: E731
    if c["kind"] == "hold":
        n = c["N"] * c["K"]
        return {"bytes": 8 * n + 2 * held(c["N"], c["K"]), "flops": 2 * n}
    if c["kind"] == "lookup":
        rows = min(c["n"], c["V"])
        return {"bytes": held(rows, c["K"]) + c["n"] * (4 * c["K"] + 8), "flops": c["n"] * c["K"]}
    M, K, N = c["M"], c["K"], sum(_rows_of(c))
    out = c["I"] if c["kind"] == "gateup" else N * (2 if c["residual"] else 1)
    return {"bytes": held(N, K) + 4 * M * (K + out) + (4 * K if c["norm"] else 0),
            "flops": 2 * M * K * N}


# ------------------------------------------------------------------------ in 64 bits
def _held64(held, rows, K):
    """Rows `rows` (a tensor of indices) of a held weight in 64 bits, by the place of each byte."""
    codes, scales = held[0].reshape(-1), held[1].reshape(-1)
    k = torch.arange(K, device=rows.device)
    tile = (rows // 32)[:, None] * -(-K // 64) + k // 64
    lane = 32 * (k // 32 % 2) + (rows % 32)[:, None]
    code = codes[tile * 1024 + lane * 16 + k % 32 // 2].to(torch.int16)
    code = torch.where(k % 2 == 1, code >> 4, code & 15)
    sign = 1 - 2 * (code >> 3).to(torch.float64)
    e, m = code >> 1 & 3, (code & 1).to(torch.float64)
    size = torch.where(e > 0, (2 + m) * 2.0 ** (e - 2).to(torch.float64), m / 2)
    at = ((rows // 32)[:, None] * -(-K // 256) + k // 256) * 256 + lane * 4 + k // 64 % 4
    scale = scales[at].to(torch.float64)
    return sign * size * torch.where(scale == 255, math.nan, 2.0 ** (scale - 127))


def _rounded64(w):
    """What the rows of w read back as, group by group, by distances to the sizes."""
    out = torch.empty(w.shape, dtype=torch.float64, device=w.device)
    sizes = torch.tensor(SIZES, dtype=torch.float64, device=w.device)
    for a in range(0, w.shape[1], GROUP):
        x = w[:, a:a + GROUP].to(torch.float64)
        top = x.abs().max(1, keepdim=True).values
        fits = torch.exp2(torch.ceil(torch.log2(top / 7)))
        # log2 may miss a power of two by one
        fits = torch.where(7 * (fits / 2) >= top, fits / 2, fits)
        fits = torch.where(7 * fits < top, fits * 2, fits)
        fits = fits.clamp(min=2.0 ** -127)
        q = (x / fits).abs()
        best, far = torch.zeros_like(q), q.clone()
        for i in range(1, 8):
            d = (q - sizes[i]).abs()
            # the codes of even index take a tie
            nearer = d <= far if i % 2 == 0 else d < far
            best, far = torch.where(nearer, sizes[i], best), torch.where(nearer, d, far)
        out[:, a:a + GROUP] = torch.copysign(best, x) * fits
    return out


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "hold":
        return {"w": torch.cat([_rounded64(r) for r in s["w"].split(16384)])}
    if c["kind"] == "lookup":
        return {"x": _held64(s["table"], s["ids"], c["K"])}
    x = s["x"].to(torch.float64)
    if c["norm"]:
        x = x / (x.square().sum(1, keepdim=True) / c["K"] + s["eps"]).sqrt() * s["norm_w"]
    y = []
    for held, N in zip(s["weights"], _rows_of(c)):
        parts = torch.arange(N, device="cuda").split(8192)
        y.append(torch.cat([x @ _held64(held, p, c["K"]).T for p in parts], dim=1))
    if c["kind"] == "gateup":
        return {"h": y[0] * torch.sigmoid(y[0]) * y[1]}
    if c["residual"]:
        y = [v + r.to(torch.float64) for v, r in zip(y, s["residual"])]
    return {"y%d" % i: v for i, v in enumerate(y)}
