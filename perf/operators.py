"""Activations held in few bits, as calls that can be timed and checked.

Two stores share one rule.  A group of fp32 values is kept as an offset lo (its smallest value), a
step ((largest - smallest) / (levels - 1), rounded to fp32) and one whole code per value,
round((x - lo) / step); it reads back as lo + code * step.

  cache       a key/value cache in 4 bits: new rows are quantised as they are written (one group per
              head row of D values), and the cache is read back with its heads expanded, as the
              attention of head sizes without a kernel of its own reads it
  attend      attention of new queries over such a cache, from one token to a long chunk of a prompt
  checkpoint  a transformer block's saved input in 8 bits (groups of 128 values along a row), and
              what the block's re-run in the backward pass starts with: the restored rows and,
              with a norm, their RMSNorm

Codes are packed eight 4-bit ones to a 32-bit word, the first in the lowest bits, or four 8-bit
ones, a row of H of them padded to 16 bytes.
"""
import ctypes as C
import math

import torch

own = False

GROUP8 = 128


def _cache(B, T, H, Hk, D, S, pos):
    return {"kind": "cache", "B": B, "T": T, "H": H, "Hk": Hk, "D": D, "S": S, "pos": pos}


def _attend(B, T, H, Hk, D, S, pos):
    return {"kind": "attend", "B": B, "T": T, "H": H, "Hk": Hk, "D": D, "S": S, "pos": pos}


def _checkpoint(rows, width, norm):
    return {"kind": "checkpoint", "rows": rows, "width": width, "norm": norm}


def listed():
    return [
        # one new token into a short cache of three heads of 80 values, and the cache read back
        dict(_cache(1, 1, 9, 3, 80, 512, 340), name="cache_step_d80"),
        # a chat turn's prompt behind an earlier turn, Qwen3 heads
        dict(_cache(1, 509, 16, 8, 128, 2048, 515), name="cache_turn_509"),
        # the prompts of a batch, LLaMA-3.2-1B heads, into an empty cache
        dict(_cache(8, 2048, 32, 8, 64, 4096, 0), name="cache_prompts_b8"),
        # one token early in a conversation with the smallest model (three query heads a KV head)
        dict(_attend(1, 1, 9, 3, 64, 512, 256), name="attend_smollm2_l257"),
        # one token of batch-1 generation on the flagship model
        dict(_attend(1, 1, 16, 8, 128, 8192, 4095), name="attend_qwen3_l4096"),
        # one token for each of eight conversations, LLaMA-3.2-1B heads
        dict(_attend(8, 1, 32, 8, 64, 8192, 6000), name="attend_llama_b8_l6001"),
        # one token at the end of a long document
        dict(_attend(1, 1, 16, 8, 128, 131072, 130000), name="attend_qwen3_l130001"),
        # a few drafted tokens checked at once behind a conversation
        dict(_attend(2, 7, 16, 8, 128, 4096, 2010), name="attend_qwen3_t7"),
        # a prompt's later chunk against everything before it
        dict(_attend(1, 1024, 16, 8, 128, 32768, 15360), name="attend_qwen3_chunk1024"),
        # the saved input of one block of a short fine-tuning step, SmolLM2 width
        dict(_checkpoint(511, 576, True), name="checkpoint_smollm2_511"),
        # the same of the flagship step: Qwen3-1.7B, B8 T4096
        dict(_checkpoint(32768, 2048, True), name="checkpoint_qwen3_1.7b"),
        # a function of the user's own under a checkpoint, its rows not whole groups
        dict(_checkpoint(4095, 1001, False), name="checkpoint_plain_1001"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["cache", "attend", "attend", "attend", "checkpoint"])
    if kind == "checkpoint":
        norm = rng.random() < 0.6
        width = rng.choice([576, 960, 1024, 2048]) if rng.random() < 0.5 else _log(rng, 33, 5000)
        return _checkpoint(_log(rng, 1, min(32768, (1 << 26) // width)), width, norm)
    Hk = rng.choice([1, 2, 3, 5, 8])
    group = rng.choice([1, 2, 3, 4])
    if kind == "cache":
        D = rng.choice([16, 40, 64, 80, 96, 128, 256])
        B = rng.randint(1, 4)
        L = _log(rng, 1, 8192 // B)
        T = 1 if rng.random() < 0.3 else _log(rng, 1, L)
        return _cache(B, T, Hk * group, Hk, D, L + rng.randint(0, 300), L - T)
    D = rng.choice([64, 128])
    if rng.random() < 0.6:  # a decode step
        B = _log(rng, 1, 16)
        L = _log(rng, 1, 120000 // B)
        T = min(L, rng.choice([1, 1, 1, 2, 5, 8]))
    else:  # a chunk of a prompt
        B = rng.randint(1, 2)
        L = _log(rng, 16, 12000 // B)
        T = _log(rng, 1, min(L, 1024))
    return _attend(B, T, Hk * group, Hk, D, L + rng.randint(0, 300), L - T)


# ---------------------------------------------------------------------- plain form
def _quantise(x, levels):
    """Offset, step and codes of x [..., n], a group per row.

    The step is rounded to fp32; (x - lo) / step is formed in 64 bits, where values on either side
    of a border between two codes stay apart.
    """
    lo = x.amin(-1, keepdim=True)
    hi = x.amax(-1, keepdim=True)
    n = torch.full_like(lo, levels - 1).double()
    step = ((hi.double() - lo.double()) / n).float()
    inv = torch.ones_like(n) / step.double()
    codes = torch.round((x.double() - lo.double()) * inv).clamp(0, levels - 1)
    codes = torch.where(step > 0, codes, torch.zeros_like(codes))
    return codes.int(), torch.cat([lo, step], -1)


def _pack4(codes):
    """[..., D] codes below 16 -> [..., D / 8] words."""
    shift = 4 * torch.arange(8, device=codes.device, dtype=torch.int32)
    return (codes.unflatten(-1, (-1, 8)) << shift).sum(-1, dtype=torch.int32)


def _unpack4(words):
    shift = 4 * torch.arange(8, device=words.device, dtype=torch.int32)
    return ((words.unsqueeze(-1) >> shift) & 15).flatten(-2)


def _values(codes, params):
    """lo + code * step with one rounding, to fp32."""
    return (params[..., :1].double() + codes.double() * params[..., 1:].double()).float()


def _plain_cache(s):
    c, out = s["case"], {}
    pos, L = c["pos"], c["pos"] + c["T"]
    for name in ("k", "v"):
        words, params = s[name + "_words"], s[name + "_params"]
        codes, par = _quantise(s[name].transpose(1, 2), 16)
        words[:, :, pos:L] = _pack4(codes)
        params[:, :, pos:L] = par
        x = _values(_unpack4(words[:, :, :L]), params[:, :, :L])
        out[name] = x.repeat_interleave(c["H"] // c["Hk"], 1)
    return out


def _plain_attend(s):
    c = s["case"]
    B, T, H, Hk, D, pos = c["B"], c["T"], c["H"], c["Hk"], c["D"], c["pos"]
    L, g = pos + T, H // Hk
    k = _values(_unpack4(s["k_words"][:, :, :L]), s["k_params"][:, :, :L])
    v = _values(_unpack4(s["v_words"][:, :, :L]), s["v_params"][:, :, :L])
    q = s["q"].reshape(B, T, Hk, g, D).permute(0, 2, 1, 3, 4).reshape(B * Hk, T * g, D)
    w = torch.bmm(q, k.reshape(B * Hk, L, D).transpose(1, 2).contiguous()) * s["scale"]
    seen = pos + torch.arange(T, device=q.device).repeat_interleave(g)
    w = w.masked_fill(torch.arange(L, device=q.device)[None] > seen[:, None], -math.inf)
    w = torch.exp(w - w.amax(-1, keepdim=True))
    w = w / w.sum(-1, keepdim=True)
    o = torch.bmm(w, v.reshape(B * Hk, L, D))
    return {"o": o.reshape(B, Hk, T, g, D).permute(0, 2, 1, 3, 4).reshape(B, T, H, D)}


def _plain_checkpoint(s):
    x = s["x"]
    rows, width = x.shape
    pad = -width % GROUP8
    # a short last group repeats its own last value, which moves neither bound
    xp = torch.cat([x, x[:, -1:].expand(rows, pad)], 1).unflatten(1, (-1, GROUP8))
    codes, params = _quantise(xp, 256)
    held = codes.to(torch.uint8)
    x = _values(held, params).flatten(1)[:, :width]
    if not s["case"]["norm"]:
        return {"x": x}
    rstd = torch.rsqrt((x * x).mean(1, keepdim=True) + s["eps"])
    return {"x": x, "y": x * rstd * s["w"], "rstd": rstd[:, 0]}


# ----------------------------------------------------------------- the framework's calls
def _p(t):
    return C.c_void_p(t.data_ptr())


def _own(s):
    from emberlm_amd import capi
    c = s["case"]
    st = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    new = lambda *shape: torch.empty(shape, device="cuda")  # noqa: E731
    if c["kind"] == "checkpoint":
        rows, width = c["rows"], c["width"]
        codes = torch.empty((rows, (width + 15) // 16 * 16), device="cuda", dtype=torch.uint8)
        params = new(rows, (width + GROUP8 - 1) // GROUP8, 2)
        x = new(rows, width)
        capi.call("ember_q8_quantize", _p(s["x"]), _p(codes), _p(params), rows, width, st)
        if not c["norm"]:
            capi.call("ember_q8_dequantize", _p(codes), _p(params), _p(x), rows, width, st)
            return {"x": x}
        y, rstd = new(rows, width), new(rows)
        capi.call("ember_q8_dequantize_rmsnorm", _p(codes), _p(params), _p(s["w"]), _p(x), _p(y),
                  _p(rstd), rows, width, s["eps"], st)
        return {"x": x, "y": y, "rstd": rstd}
    B, T, H, Hk, D, S, pos = (c[n] for n in ("B", "T", "H", "Hk", "D", "S", "pos"))
    L = pos + T
    cache = [_p(s[n]) for n in ("k_words", "k_params", "v_words", "v_params")]
    if c["kind"] == "cache":
        capi.call("ember_kv4_write", _p(s["k"]), _p(s["v"]), *cache, B, T, Hk, D, S, pos, st)
        out = {"k": new(B, H, L, D), "v": new(B, H, L, D)}
        capi.call("ember_kv4_read_expanded", *cache[:2], _p(out["k"]), B, Hk, H // Hk, L, D, S, st)
        capi.call("ember_kv4_read_expanded", *cache[2:], _p(out["v"]), B, Hk, H // Hk, L, D, S, st)
        return out
    o = new(B, T, H, D)
    need = capi.lib().ember_attn_kv4_workspace_bytes(B, T, H, Hk, D, L)
    ws = torch.empty(need, device="cuda", dtype=torch.uint8) if need else None
    capi.call("ember_attn_kv4", _p(s["q"]), *cache, _p(o), B, T, H, Hk, D, L, pos, S, s["scale"],
              _p(ws) if need else None, need, st)
    return {"o": o}


def run(state):
    if own:
        return _own(state)
    return {"cache": _plain_cache, "attend": _plain_attend,
            "checkpoint": _plain_checkpoint}[state["case"]["kind"]](state)


# --------------------------------------------------------------------------- inputs
def _heads(gen, B, n, Hk, D, spread):
    """Projections [B, n, Hk, D] whose channels differ in size and centre, as keys' do."""
    rand = lambda *shape: torch.randn(shape, generator=gen, device="cuda")  # noqa: E731
    return rand(B, n, Hk, D) * torch.exp(spread * rand(Hk, D)) + spread * rand(Hk, D)


def _filled(gen, c, name, spread):
    """A cache of S rows that earlier calls filled: every row holds something."""
    codes, params = _quantise(_heads(gen, c["B"], c["S"], c["Hk"], c["D"], spread).transpose(1, 2),
                              16)
    return {name + "_words": _pack4(codes).contiguous(), name + "_params": params.contiguous()}


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = {"case": c}
    if c["kind"] == "checkpoint":
        rows, width = c["rows"], c["width"]
        rand = lambda *shape: torch.randn(shape, generator=gen, device="cuda")  # noqa: E731
        # a residual stream: channels of unlike size, a few of them far larger
        s["x"] = rand(rows, width) * torch.exp(rand(width)) + 0.3 * rand(width)
        s["w"] = 1 + 0.1 * rand(width)
        s["eps"] = 1e-5
        return s
    s.update(_filled(gen, c, "k", 0.5))
    s.update(_filled(gen, c, "v", 0.25))
    if c["kind"] == "cache":
        s["k"] = _heads(gen, c["B"], c["T"], c["Hk"], c["D"], 0.5)
        s["v"] = _heads(gen, c["B"], c["T"], c["Hk"], c["D"], 0.25)
    else:
        s["q"] = torch.randn((c["B"], c["T"], c["H"], c["D"]), generator=gen, device="cuda")
        s["scale"] = 1.0 / math.sqrt(c["D"])
    return s


def work(case):
    c = case
    if c["kind"] == "checkpoint":
        n = c["rows"] * c["width"]
        held = c["rows"] * ((c["width"] + 15) // 16 * 16 + 8 * ((c["width"] + 127) // 128))
        # the rows in, the codes out and, at the re-run, in again; the restored rows (and norm) out
        out = (8 * n + 4 * c["rows"] + 4 * c["width"]) if c["norm"] else 4 * n
        return {"bytes": 4 * n + 2 * held + out, "flops": (10 if c["norm"] else 6) * n}
    B, T, H, Hk, D, pos = (c[n] for n in ("B", "T", "H", "Hk", "D", "pos"))
    L, row = pos + T, D // 2 + 8
    if c["kind"] == "cache":
        return {"bytes": 2 * B * Hk * (T * (4 * D + row) + L * row) + 8 * B * H * L * D,
                "flops": 2 * B * Hk * D * (4 * T + 2 * L)}
    pairs = T * pos + T * (T + 1) // 2
    return {"bytes": 2 * B * Hk * L * row + 8 * B * T * H * D, "flops": 4 * B * H * D * pairs}


# ------------------------------------------------------------------------ in 64 bits
def _groups64(x, levels):
    """What the groups x [..., n] read back as: bounds and codes in 64 bits, the step as held."""
    x = x.to(torch.float64)
    lo, hi = x.aminmax(dim=-1, keepdim=True)
    step = torch.div(hi - lo, torch.tensor(float(levels - 1), dtype=torch.float64,
                                           device=x.device).expand_as(lo))
    step = step.to(torch.float32).to(torch.float64)
    inverse = torch.where(step > 0, torch.div(torch.ones_like(step), step), torch.zeros_like(step))
    return lo + step * ((x - lo) * inverse).round().clamp(min=0, max=levels - 1)


def _held64(words, params):
    """The values of cache rows, in 64 bits, word by word."""
    cols = [torch.bitwise_and(torch.bitwise_right_shift(words, 4 * i), 15) for i in range(8)]
    codes = torch.stack(cols, dim=-1).flatten(-2).to(torch.float64)
    p = params.to(torch.float64)
    return p[..., 0].unsqueeze(-1) + codes * p[..., 1].unsqueeze(-1)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "checkpoint":
        cuts = list(range(0, c["width"], GROUP8)) + [c["width"]]
        x = torch.cat([_groups64(s["x"][:, a:b], 256) for a, b in zip(cuts, cuts[1:])], dim=1)
        if not c["norm"]:
            return {"x": x}
        rstd = (x.square().sum(1) / c["width"] + s["eps"]) ** -0.5
        return {"x": x, "y": x * rstd[:, None] * s["w"].to(torch.float64), "rstd": rstd}
    B, T, H, Hk, D, pos = (c[n] for n in ("B", "T", "H", "Hk", "D", "pos"))
    L, g = pos + T, H // Hk
    if c["kind"] == "cache":
        out = {}
        for name in ("k", "v"):
            old = _held64(s[name + "_words"][:, :, :pos], s[name + "_params"][:, :, :pos])
            rows = torch.cat([old, _groups64(s[name].permute(0, 2, 1, 3), 16)], dim=2)
            out[name] = rows[:, :, None].expand(B, Hk, g, L, D).reshape(B, H, L, D)
        return out
    o = torch.empty((B, T, H, D), device="cuda", dtype=torch.float64)
    last = pos + torch.arange(T, device="cuda")
    for b in range(B):
        for n in range(Hk):
            k = _held64(s["k_words"][b, n, :L], s["k_params"][b, n, :L])
            v = _held64(s["v_words"][b, n, :L], s["v_params"][b, n, :L])
            for h in range(n * g, n * g + g):
                z = s["q"][b, :, h].to(torch.float64) @ k.T * s["scale"]
                z[torch.arange(L, device="cuda") > last[:, None]] = -math.inf
                o[b, :, h] = torch.softmax(z, dim=1) @ v
    return {"o": o}
