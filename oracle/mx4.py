"""Weights in microscaled 4-bit floating point, and products with them, in 64 bits.

Rows in groups of 32 values (the last may be shorter): a scale byte b per group, 2^(b - 127), the
smallest power of two that 7 times reaches the group's largest size (b >= 0), and per value a sign
and the nearest of SIZES to its quotient by the scale, of two as near the one of even index.  b = 255,
codes 0: a group with a value that is not finite; it reads back as NaN.
"""
import numpy as np

SIZES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
GROUP = 32


def quantise(w):
    """Codes [N, K] uint8 and scale bytes [N, ceil(K / 32)] uint8 of w [N, K] (float32)."""
    w = np.asarray(w, np.float32)
    N, K = w.shape
    codes, scales = np.zeros((N, K), np.uint8), np.zeros((N, -(-K // GROUP)), np.uint8)
    for i, a in enumerate(range(0, K, GROUP)):
        x = w[:, a:a + GROUP].astype(np.float64)
        bad = ~np.isfinite(x).all(1)
        x = np.where(bad[:, None], 0.0, x)
        top = np.abs(x).max(1)
        m, e = np.frexp(top / 7)  # top / 7 = m 2^e, m in [1/2, 1): 2^(e - 1) only if m is 1/2
        b = np.where(top > 0, np.where(7 * np.ldexp(0.5, e) >= top, e - 1, e), -127)
        b = np.maximum(b, -127)
        q = np.ldexp(np.abs(x), -b[:, None])
        d = np.abs(q[..., None] - SIZES)
        d[..., 1::2] = np.nextafter(d[..., 1::2], np.inf)  # a tie goes to the even index
        c = np.where(q > 6, 7, d.argmin(-1)) + 8 * np.signbit(w[:, a:a + GROUP])
        codes[:, a:a + GROUP] = np.where(bad[:, None], 0, c)
        scales[:, i] = np.where(bad, 255, b + 127)
    return codes, scales


def values(codes, scales):
    """What codes [N, K] and scales read back as, in 64 bits."""
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    v = SIZES[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    return v * np.repeat(s, GROUP, 1)[:, :codes.shape[1]]


def _grown(a, rows, cols):
    out = np.zeros((-(-a.shape[0] // rows) * rows, -(-a.shape[1] // cols) * cols), a.dtype)
    out[:a.shape[0], :a.shape[1]] = a
    return out


def pack(codes, scales):
    """The two buffers as flat uint8 arrays: tiles of 32 rows by 64 columns, 256 scales a block."""
    c = _grown(codes, 32, 64)
    both = (c[:, 0::2] | c[:, 1::2] << 4).reshape(c.shape[0] // 32, 32, -1, 2, 16)
    s = _grown(scales, 32, 8)
    s = s.reshape(s.shape[0] // 32, 32, -1, 4, 2)
    return both.transpose(0, 2, 3, 1, 4).ravel(), s.transpose(0, 2, 4, 1, 3).ravel()


def hold(w):
    """The two buffers and the values in 64 bits of w."""
    codes, scales = quantise(w)
    return (*pack(codes, scales), values(codes, scales))


def rms_norm(x, w, eps):
    x = np.asarray(x, np.float64)
    return x / np.sqrt((x * x).mean(1, keepdims=True) + eps) * w


def silu(g):
    return g / (1 + np.exp(np.minimum(-g, 700.0)))


def product_bound(x, w, y):
    """How far an fp32-accurate product y = x w^T [M, N] may be from 64 bits.

    An element is the sum of K terms.  Two kinds of roundings go into it, each at most half a
    step, 2^-24, of something:
      - one operand's, per term: x as the kernels hold it is off by 2^-24 of its group's largest
        size at most (products of it with the codes are exact), and by 2^-24 of itself where a norm's
        weight is multiplied in.  Independent of each other: 7 times the root of the sum of their
        squares is passed once in 10^10 (Hoeffding).
      - the running sum's: twice per 64 columns (an MFMA each for the upper and the lower part of x),
        and 24 for the split of K, the norm's factor and the store.  The running sum is
        below |y| and 7 times the root of its terms' squares.
    """
    x, w = np.abs(x), np.abs(np.nan_to_num(w))
    K = x.shape[1]
    top = np.repeat(np.maximum.reduceat(x, np.arange(0, K, GROUP), axis=1), GROUP, 1)[:, :K]
    terms = np.sqrt((x * x) @ (w * w).T)
    groups = np.sqrt((top * top) @ (w * w).T)
    n = 24 + 2 * -(-K // 64)
    return 2.0 ** -24 * (7 * groups + 7 * terms + n * (np.abs(y) + 7 * terms)) + 2.0 ** -126


def rms_bound(x, w, y):
    """What the error of each element of y = x w^T [M, N] is below in the mean of its square's root.

    The roundings of product_bound, each at most half a step, 2^-24, of its value and independent of
    each other, so that their squares add up: one a term, of x's group's largest size, and one where a
    norm's weight is multiplied in; 24 for the split of K, the norm's factor and the store; and K / 32
    of running sums, one a group (of the upper digits; the lower ones' sums are 2^-9 of these), which
    grow up to y and to the root of their terms' squares, their squares half of that on average.  (A
    rounding's own mean square is a third of what is counted here.  What the matrix cores drop, below
    2^-27 of a running sum, is an eighth of a half step a time.)
    """
    x, w = np.abs(x), np.abs(w)
    K = x.shape[1]
    top = np.repeat(np.maximum.reduceat(x, np.arange(0, K, GROUP), axis=1), GROUP, 1)[:, :K]
    terms = (x * x) @ (w * w).T
    groups = (top * top) @ (w * w).T
    return 2.0 ** -24 * np.sqrt(groups + terms + (24 + K / 64) * (y * y + terms))


def gateup_rms_bound(x, g, u):
    """The same of silu(x g^T) * (x u^T): either factor's error through the product (|silu'| <= 1.1),
    and six roundings and the exponential's of the result."""
    yg, yu = x @ g.T, x @ u.T
    own = 2.0 ** -23 * (6 + np.abs(yg)) * np.abs(silu(yg) * yu)
    return np.sqrt((1.1 * rms_bound(x, g, yg) * yu) ** 2 + (silu(yg) * rms_bound(x, u, yu)) ** 2 +
                   own ** 2)


def in_digits(x, digits):
    """x as the first of its base-32 digits: a group's scale is 2^-3 of its largest size's power of two."""
    K = x.shape[1]
    top = np.repeat(np.maximum.reduceat(np.abs(x), np.arange(0, K, GROUP), axis=1), GROUP, 1)[:, :K]
    unit = np.ldexp(1.0, np.frexp(np.where(top > 0, top, 1.0))[1] - 4 - 5 * (digits - 1))
    return np.rint(x / unit) * unit
