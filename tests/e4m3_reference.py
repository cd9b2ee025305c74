"""Plain numpy forms of the e4m3 block-scaled operators, in 64 bits where a value is computed."""

import numpy as np

BLOCK = 128
MAX = 448.0


def decode(bytes_):
    """e4m3 bytes -> the float64 values they stand for (0x7f and 0xff: NaN)."""
    b = np.asarray(bytes_, dtype=np.int64)
    sign = np.where(b & 0x80, -1.0, 1.0)
    e, m = (b >> 3) & 15, b & 7
    v = np.where(e == 0, m * 2.0**-9, (8 + m) * 2.0 ** (e - 10.0))
    return np.where((b & 0x7F) == 0x7F, np.nan, sign * v)


def encode(v):
    """float64 -> e4m3 bytes, to nearest, ties to even, clamped to +-448."""
    v = np.asarray(v, dtype=np.float64)
    a = np.minimum(np.abs(v), MAX)
    _, e = np.frexp(np.where(a > 0, a, 1.0))
    e = np.maximum(e - 1, -6)  # exponent of the value's step: 2^(e - 3)
    m = np.rint(np.ldexp(a, 3 - e)).astype(np.int64)  # rint: ties to even
    e = np.where(m == 16, e + 1, e)
    m = np.where(m == 16, 8, m)
    byte = np.where(m < 8, m, ((e + 7) << 3) | (m - 8))
    byte = np.where(np.isnan(v), 0x7F, byte | np.where(np.signbit(v), 0x80, 0))
    return byte.astype(np.uint8)


def encode_exact(v):
    """encode() of extended-precision values: cut to float64 with what is cut off in the last bit, so that no tie
    is made of a value beside one."""
    d = v.astype(np.float64)
    rest = v - d.astype(np.longdouble)
    low = np.where(rest < 0, np.nextafter(d, -np.inf), np.where(rest > 0, np.nextafter(d, np.inf), d))
    return encode(np.where(np.isfinite(d) & (rest != 0), low, d))


def scale_of(amax):
    """float32 scale of blocks with these maxima."""
    amax = np.asarray(amax, dtype=np.float32)
    s = (amax / np.float32(MAX)).astype(np.float32)
    s = np.where(s < np.float32(2.0**-126), np.float32(2.0**-126), s)
    return np.where(amax == 0, np.float32(1), s).astype(np.float32)


def _blocks(x, tall):
    rows, K = x.shape
    rb, kb = -(-rows // tall), -(-K // BLOCK)
    full = np.zeros((rb * tall, kb * BLOCK), dtype=np.float32)
    full[:rows, :K] = x
    return full.reshape(rb, tall, kb, BLOCK)


def quantize(x, tall):
    """x float32 [rows x K] -> (bytes [rows x K], scales [row blocks x K blocks]); `tall` rows share a scale."""
    rows, K = x.shape
    f = _blocks(x, tall)
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        amax = np.abs(f).max(axis=(1, 3))  # a NaN propagates
        s = scale_of(amax)
        # the exact quotient 448 x / amax, in extended precision (the product is exact; the quotient keeps 64 bits,
        # and one that is no tie is at least 2^-50 of itself away from one)
        least, x = s == np.float32(2.0**-126), f.astype(np.longdouble)
        over = np.where(least | (amax == 0), np.longdouble(1), amax.astype(np.longdouble))
        by = np.where(least, np.longdouble(2.0**126), np.where(amax == 0, np.longdouble(1), np.longdouble(448)))
        q = encode_exact(x * by[:, None, :, None] / over[:, None, :, None])
    return q.reshape(f.shape[0] * tall, -1)[:rows, :K], s


def dense(xq, xs, wq, ws):
    """float64 product of the values that e4m3 bytes and scales (xs [K blocks x M], ws [N blocks x K blocks])
    stand for, and the same with absolute values (the scale of its rounding errors)."""
    K = xq.shape[1]
    x = decode(xq) * np.repeat(xs.T.astype(np.float64), BLOCK, 1)[:, :K]
    w = decode(wq) * np.repeat(np.repeat(ws.astype(np.float64), BLOCK, 0)[: wq.shape[0]], BLOCK, 1)[:, :K]
    return x @ w.T, np.abs(x) @ np.abs(w).T
