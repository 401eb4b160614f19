"""MXFP4 by its definition, in 64 bits on the CPU: the oracle of the quantiser's and the product's tests."""
import numpy as np

VALUES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
BETWEEN = (VALUES[1:] + VALUES[:-1]) / 2


def quantize(x):
    """(codes [rows, k], scale bytes [rows, blocks]) of the rows of x, blocks of 32."""
    x = np.asarray(x, dtype=np.float64)
    rows, k = x.shape
    blocks = -(-k // 32)
    v = np.zeros((rows, blocks * 32))
    v[:, :k] = x
    v = v.reshape(rows, blocks, 32)
    bad = ~np.isfinite(v).all(-1)
    v = np.where(bad[..., None], 0, v)
    most = np.abs(v).max(-1)
    exponent = np.frexp(np.where(most > 0, most, 2.0**-200))[1] - 1  # most = 2^exponent * [1, 2)
    s = np.clip(exponent - 2, -127, 127)
    size = np.abs(np.ldexp(v, -s[..., None]))
    # a border between two codes goes to the even one: the upper code where the lower one is odd
    code = sum((size > b) if i % 2 == 0 else (size >= b) for i, b in enumerate(BETWEEN)).astype(np.uint8)
    code |= np.signbit(v).astype(np.uint8) << 3
    code = np.where(bad[..., None], 0, code).astype(np.uint8).reshape(rows, -1)[:, :k]
    return code, np.where(bad, 255, s + 127).astype(np.uint8)


def values(codes, scales):
    """What codes and scales stand for, float64."""
    rows, k = codes.shape
    v = np.where(codes & 8, -1.0, 1.0) * VALUES[codes & 7]
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(int) - 127))
    return v * np.repeat(s, 32, axis=1)[:, :k]


def round_trip(x):
    return values(*quantize(x))
