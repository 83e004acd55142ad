"""Row operators in binary64, from their definitions, for the tests.  Arrays are (d, rows, ...): the
first axis is a row, as in the package's column-major arrays."""
import math

import ml_dtypes
import numpy as np

BF16 = np.dtype(ml_dtypes.bfloat16)
TYPES = {"f16": np.dtype(np.float16), "bf16": BF16, "f32": np.dtype(np.float32)}
HALF = {np.dtype(np.float16): 2.0 ** -11, BF16: 2.0 ** -8, np.dtype(np.float32): 2.0 ** -24}   # half a step, relative
TINY = {np.dtype(np.float16): 2.0 ** -25, BF16: 2.0 ** -134, np.dtype(np.float32): 2.0 ** -150}         # half the least subnormal
U = 2.0 ** -24                                                                                          # of the arithmetic


def rounded(x, dtype):
    """`x` in the type, and back."""
    return np.asarray(x).astype(dtype).astype(np.float64)


def within(got, want, slack, what=""):
    """|got - want| <= half a step of got's type + slack (the error of the binary32 arithmetic)."""
    got_type = got.dtype
    got, want = got.astype(np.float64), np.asarray(want, dtype=np.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert np.array_equal(np.isnan(got), np.isnan(want)), (what, "NaN in other places")
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)]), (what, "infinities differ")
    slack = np.broadcast_to(slack, want.shape)[fine]
    off = np.abs(got[fine] - want[fine])
    # the rounded value is the one with the slack on it
    tol = HALF[got_type] * (np.abs(want[fine]) + slack) + slack + TINY[got_type]
    assert (off <= tol).all(), (what, "off by %.3g, allowed %.3g" % (off[np.argmax(off - tol)], tol[np.argmax(off - tol)]))


# ---- layer norm
def norm(x, gamma, beta, eps):
    """x: (d, rows)."""
    mean = x.mean(0)
    rstd = 1.0 / np.sqrt(((x - mean) ** 2).mean(0) + eps)
    hat = (x - mean) * rstd
    return hat * gamma[:, None] + beta[:, None], mean, rstd, hat


def norm_grad(dy, hat, rstd, gamma):
    g = dy * gamma[:, None]
    dx = rstd * (g - g.mean(0) - hat * (g * hat).mean(0))
    return dx, (dy * hat).sum(1), dy.sum(1)


def norm_steps(d):
    """Roundings on the way to a row's sum: 16 terms in a thread, 5 exchanges, up to 16 warps; rows of
    more than 8192 elements: d / 1024 terms and two times 5 exchanges."""
    return max(16 + 5 + 16, d / 1024 + 11) + 3


# ---- 8 bits
def blocks(x):
    n = -(-x.shape[0] // 32)
    p = np.zeros((n * 32,) + x.shape[1:], dtype=np.float64)
    p[: x.shape[0]] = x
    return p.reshape((n, 32) + x.shape[1:])


def exponents(x, form):
    """Scale bytes of rows."""
    top = 127.0 if form == "int8" else 448.0
    with np.errstate(invalid="ignore"):
        big = np.abs(blocks(x)).max(1)
    m, e = np.frexp(np.where(np.isfinite(big), big, 1.0))
    mt, et = math.frexp(top)
    k = np.where(m == 0, -127, np.maximum(e - et + (m > mt), -127))
    return np.where(np.isfinite(big), k + 127, 255).astype(np.uint8)


def quantize(x, form):
    e = exponents(x, form)
    with np.errstate(invalid="ignore", over="ignore"):
        v = np.ldexp(blocks(x), 127 - e.astype(np.int32)[:, None]).reshape((-1,) + x.shape[1:])[: x.shape[0]]
    v = np.where(np.repeat(e, 32, axis=0)[: x.shape[0]] == 255, 0.0, v)
    if form == "int8":
        return np.rint(v).astype(np.int8), e
    step = np.ldexp(1.0, np.maximum(np.frexp(v)[1] - 1, -6) - 3)
    return (np.rint(v / step) * step).astype(ml_dtypes.float8_e4m3fn).view(np.uint8), e


def restore(codes, scales):
    v = codes.astype(np.float64) if codes.dtype == np.int8 else codes.view(ml_dtypes.float8_e4m3fn).astype(np.float64)
    e = np.repeat(scales.astype(np.int32), 32, axis=0)[: codes.shape[0]]
    return np.where(e == 255, np.nan, np.ldexp(v, e - 127))


def saturated(x, dtype):
    top = float(np.float64(ml_dtypes.finfo(dtype).max))
    return np.clip(x, -top, top)


# ---- activations
def act(name, a):
    """f and f'."""
    def sig(u):
        with np.errstate(over="ignore"):
            return 1.0 / (1.0 + np.exp(-u))
    if name == "silu":
        q = sig(a)
        return a * q, q + a * q * (1.0 - q)
    c = math.sqrt(2.0 / math.pi)
    u = c * (a + 0.044715 * a ** 3)
    q, p = sig(2 * u), sig(-2 * u)        # (1 + tanh u) / 2 = sig(2u): 1 + tanh u itself would lose what is below 2^-53
    return a * q, q + a * q * p * 2 * c * (1.0 + 3 * 0.044715 * a * a)


# ---- rotary positions
def turn(x, pos, freq, factor, layout, adjoint=False):
    """x: (d, heads, tokens, ...), pos: (tokens, ...), freq: (rot/2,)."""
    rot = 2 * len(freq)
    a = np.multiply.outer(np.asarray(freq, dtype=np.float64), pos.astype(np.float64))[:, None]
    c, s = np.cos(a) * factor, np.sin(a) * factor * (-1 if adjoint else 1)
    y = x.astype(np.float64).copy()
    if layout == "half":
        i, j = slice(0, rot // 2), slice(rot // 2, rot)
    else:
        i, j = slice(0, rot, 2), slice(1, rot, 2)
    u, v = y[i].copy(), y[j].copy()
    y[i], y[j] = u * c - v * s, v * c + u * s
    return y


def turn_slack(x, rot, factor, layout):
    """Error of a turned element in binary32, less the store: sine and cosine are good to 6 u (angle
    rounded twice, series, factor), products and sum to 3 u, both against the pair's magnitudes."""
    y = np.zeros(x.shape)
    if layout == "half":
        i, j = slice(0, rot // 2), slice(rot // 2, rot)
    else:
        i, j = slice(0, rot, 2), slice(1, rot, 2)
    m = np.abs(x[i]).astype(np.float64) + np.abs(x[j]).astype(np.float64)
    y[i] = y[j] = 9 * U * abs(factor) * m
    return y
