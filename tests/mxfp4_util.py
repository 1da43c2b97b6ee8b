"""Microscaled 4-bit floating point from its definition, in 64 bits on the CPU, and what 32-bit sums over it may be off (ffn_util says how errors are counted)."""
import numpy as np

from ffn_util import U

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
VALUES = np.concatenate([GRID, -GRID])  # of the 16 codes


def blocks(n):
    return -(-n // 32)


def scale_of(amax):
    """b of the least power of two 2^(b - 127), b from 1 on, with amax < 7 * 2^(b - 127); 255 for what is not finite."""
    out = np.full(np.shape(amax), 255, np.uint8)
    for i in np.ndindex(np.shape(amax)):
        if np.isfinite(amax[i]):
            b = 1
            while not amax[i] < 7 * 2.0 ** (b - 127):
                b += 1
            out[i] = b
    return out


def power(b):
    b = np.asarray(b, np.int64)
    return np.where(b == 255, np.nan, np.exp2(b - 127.0))


def encode(v):
    """The code nearest to v (magnitude below 7), the even one of two as near; 0 for what is not finite."""
    a = np.where(np.isfinite(v), np.abs(v), 0)
    d = np.abs(a[..., None] - GRID)
    best = d.min(-1, keepdims=True)
    near = d == best
    even = near & (np.arange(8) % 2 == 0)
    code = np.where(even.any(-1), even.argmax(-1), near.argmax(-1))
    return np.where(np.isfinite(v), code | np.where(np.signbit(v), 8, 0), 0).astype(np.uint8)


def quantize(x):
    """x [M, K] (64 bits) -> (codes [M, K], b [M, blocks(K)])."""
    M, K = x.shape
    pad = np.zeros((M, blocks(K) * 32))
    pad[:, :K] = x
    p = pad.reshape(M, -1, 32)
    b = scale_of(np.where(np.isfinite(p).all(-1), np.abs(p).max(-1), np.inf))
    with np.errstate(invalid="ignore"):
        return encode(p / power(b)[:, :, None]).reshape(M, -1)[:, :K], b


def values(codes, b):
    return VALUES[codes] * np.repeat(power(b), 32, 1)[:, :codes.shape[1]]


def pairs(codes):
    """Codes [M, K] two a byte, the lower k in the low half."""
    c = np.pad(codes, ((0, 0), (0, codes.shape[1] % 2)))
    return (c[:, 0::2] | c[:, 1::2] << 4).astype(np.uint8)


def single(q, K):
    return np.stack((q & 15, q >> 4), -1).reshape(q.shape[0], -1)[:, :K]


def unpack(packed, rows, K):
    """Packed bytes -> (codes [rows, K], b [rows, blocks(K)], codes between K and the end of the chunk, the scales there)."""
    chunks, panels = -(-K // 256), -(-rows // 32)
    p = np.asarray(packed, np.uint8)[:panels * chunks * 4352].reshape(panels, chunks, 4352)
    v = p[:, :, :4096].reshape(panels, chunks, 4, 2, 32, 16)  # step, half, row, byte
    q = v.transpose(0, 4, 1, 2, 3, 5).reshape(panels * 32, chunks * 128)[:rows]
    s = p[:, :, 4096:].reshape(panels, chunks, 2, 32, 4).transpose(0, 3, 1, 4, 2).reshape(panels * 32, chunks * 8)[:rows]  # (half, row, step)
    codes = single(q, chunks * 256)
    return codes[:, :K], s[:, :blocks(K)], codes[:, K:], s[:, blocks(K):]


def product(a, b, sums=0):
    """a [M, K] . b [N, K]^T of such values, and what the matrix cores may be off.

    Within a block the products are multiples of 1/4 of its scales and their sum at most 32 * 36: 13 bits, exact in 32.  Beside it there is a
    rounding for each block, and `sums` further ones."""
    n = blocks(a.shape[1]) + 4 + sums
    return a @ b.T, n * U * (np.abs(a) @ np.abs(b).T)
