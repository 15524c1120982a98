"""The 8-bit KV cache in 64 bits, in numpy: the numbers of the codes, the quantiser, attention over the values, and how far a
correct kernel may be from it."""
import math

import numpy as np


def _number(byte):
    size, fraction = byte >> 3 & 15, (byte & 7) / 8
    if size == 15 and byte & 7 == 7:
        return math.nan
    value = fraction * 2.0 ** -6 if size == 0 else (1 + fraction) * 2.0 ** (size - 7)
    return -value if byte & 128 else value


NUMBERS = np.array([_number(b) for b in range(256)])


def scale_row(block_size):
    return -(-block_size // 16) * 16


def quantise(x):
    """(codes, scale bytes) of rows [..., D] in float64: the nearest number, ties to the even code."""
    size = np.abs(x)
    most = np.minimum(np.max(np.where(np.isnan(size), 0.0, size), -1), 57344.0)
    e = np.full(most.shape, -14)
    for step in range(-14, 7):
        e += most > 448.0 * 2.0 ** step
    scaled = np.minimum(size * 2.0 ** -e[..., None].astype(np.float64), 448.0)
    positive = NUMBERS[:127]
    middle = (positive[1:] + positive[:-1]) / 2
    code = np.searchsorted(middle, scaled)  # a tie goes to the lower one
    tie = (code < 126) & (scaled == middle[np.minimum(code, 125)]) & (code % 2 == 1)
    code = np.where(np.isnan(x), 127, code + tie + 128 * np.signbit(x))
    return code.astype(np.uint8), (e + 15).astype(np.uint8)


def values(codes, scales):
    """[blocks, block_size, heads, D] in float64."""
    bs = codes.shape[1]
    return NUMBERS[codes] * 2.0 ** (scales[:, :, :bs].transpose(0, 2, 1).astype(np.float64) - 15)[..., None]


def half_step(bits16):
    """Half a step of a 16-bit type relative to the value, and the smallest it can be."""
    return (2.0 ** -8, 2.0 ** -134) if bits16 == "bf16" else (2.0 ** -11, 2.0 ** -25)


def attention(q, k, v, visible, scale, bits16):
    """q [rows, D], k / v [keys, D], visible [rows, keys]. Returns the output and the bound on a kernel's distance from it that the
    roundings add up to: P to fp16 (2^-11 of each weight; below 2^-14 of the largest 2^-25 of it), scores and sums in fp32 whose additions
    are off by at most a whole step (2^-23) each, the exponential (2^-21), and the output's type."""
    d, keys = q.shape[1], k.shape[0]
    k = np.where(visible.any(0)[:, None], k, 0.0)  # what no row sees may be NaN
    v = np.where(visible.any(0)[:, None], v, 0.0)
    s = np.where(visible, q @ k.T * scale, -np.inf)
    top = s.max(-1, keepdims=True, initial=-np.inf)
    p = np.exp(s - np.where(np.isinf(top), 0.0, top))
    total = p.sum(-1, keepdims=True)
    safe = np.where(total > 0, total, 1.0)
    out = p @ v / safe
    spread = p @ np.abs(v) / safe
    largest = np.where(visible, np.abs(q) @ np.abs(k).T * scale, 0.0).max(-1, keepdims=True)
    weight = 2 * ((d + 8) * 2.0 ** -23 * largest + 2.0 ** -21)  # relative, of a weight and of their sum
    few = keys * 2.0 ** -25 * np.abs(v).max(initial=0.0) / safe
    rel, least = half_step(bits16)
    near = spread * (2.0 ** -11 + weight + 2 * keys * 2.0 ** -23) + few
    return out, near + rel * (np.abs(out) + near) + least
