"""The block-scaled 8-bit format in 64 bits (numpy): what tests/test_blocks.py and tests/test_gpu_blocks.py hold the kernels to."""
import numpy as np

BLOCK = 128


def up(n, to):
    return -(-n // to) * to


def e4m3_values():
    """The value of each of the 256 codes: sign, 4 exponent bits (bias 7), 3 mantissa bits; exponent 15 with mantissa 7 is NaN, there is no infinity."""
    v = np.zeros(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        a = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        v[c] = np.nan if e == 15 and m == 7 else (-a if c & 128 else a)
    return v


def round_e4m3(v):
    """The nearest e4m3, ties to even, for |v| <= 448: steps of 2^-9 below 2^-6, eight to a power of two above.  np.rint ties to even."""
    a = np.abs(v)
    _, e = np.frexp(np.maximum(a, 2.0 ** -6))         # a = m 2^e, 1/2 <= m < 1
    step = np.ldexp(1.0, e - 4)
    return np.copysign(np.rint(a / step) * step, v)


def quantize(x, block_rows):
    """x float64 [rows][cols] -> (values [rows][padded], scale bytes [row blocks][blocks padded to 4])"""
    rows, cols = x.shape
    R, K = up(rows, block_rows), up(cols, BLOCK)
    big = np.zeros((R, K))
    big[:rows, :cols] = x
    t = big.reshape(R // block_rows, block_rows, K // BLOCK, BLOCK)
    finite = np.isfinite(t)
    top = np.where(finite, np.abs(t), 0.0).max((1, 3))
    byte = np.full((R // block_rows, up(K // BLOCK, 4)), 127, np.int64)
    m, e = np.frexp(top)                                     # top = m 2^e, 1/2 <= m < 1; 448 = 0.875 * 2^9: the smallest power p >= -127 with top <= 448 * 2^p
    power = np.maximum(e - 9 + (m > 0.875), -127)
    byte[:, :K // BLOCK] = np.where(top > 0, power + 127, 127)
    s = byte[:, None, :K // BLOCK, None] - 127
    v = np.where(finite, round_e4m3(np.ldexp(np.where(finite, t, 0.0), -s)), np.nan)
    return v.reshape(R, K)[:rows], byte.astype(np.uint8)


def values(v, byte, cols, block_rows):
    """[rows][cols] float64"""
    rows = v.shape[0]
    nb = -(-cols // BLOCK)
    s = np.where(byte[:, :nb] == 255, np.nan, np.ldexp(1.0, byte[:, :nb].astype(np.int64) - 127))
    wide = np.repeat(np.repeat(s, block_rows, 0)[:rows], BLOCK, 1)
    return (v[:, :nb * BLOCK] * wide)[:, :cols]


def dense(x, w, bias=None, clip=None):
    y = x @ w.T
    if bias is not None:
        y = y + bias
    if clip is not None:
        y = np.where(np.isnan(y), y, np.clip(y, 0.0, clip))
    return y
