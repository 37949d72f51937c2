"""AdamW and its 8-bit states in double precision (numpy), written from the formulas in include/gcn_uelb_hip.h."""
import numpy as np

BLOCK = 128

# value of every e4m3 code: sign, 4 exponent bits (bias 7), 3 mantissa bits; exponent 0 holds multiples of 2^-9, 0x7f is NaN
E4M3 = np.array([(-1.0) ** (c >> 7) * (2.0 ** ((c >> 3 & 15) - 10) * (8 + (c & 7)) if c & 0x78 else 2.0 ** -9 * (c & 7)) for c in range(256)])
E4M3[[0x7F, 0xFF]] = np.nan


def _mix(x):
    x = x.astype(np.uint32)
    x = (x ^ (x >> np.uint32(16))) * np.uint32(0x7FEB352D)
    x = (x ^ (x >> np.uint32(15))) * np.uint32(0x846CA68B)
    return x ^ (x >> np.uint32(16))


def random32(n, seed, step, tensor):
    """The 32 random bits of each of a tensor's n elements (n < 2^32)."""
    with np.errstate(over="ignore"):
        word = lambda v: np.array([v & 0xFFFFFFFF], dtype=np.uint32)
        key = _mix(word(seed) ^ word(0x9E3779B9))
        for v in (seed >> 32, step, step >> 32):
            key = _mix(key ^ word(v))
        key = _mix(key ^ word(tensor * 0x85EBCA6B))
        return _mix(key ^ np.arange(n, dtype=np.uint32))


def decode(codes, exps):
    scale = np.repeat(np.exp2(exps.astype(np.float64) - 127), BLOCK)[:codes.size]
    return E4M3[codes.reshape(-1)] * scale


def encode(x, random16, never_zero):
    """(values, exponent bytes, margin): the rounded values, the blocks' exponent bytes, and how far the decision between the two
    neighbours was from turning, in steps between them."""
    n = x.size
    rows = np.zeros(-(-n // BLOCK) * BLOCK)
    rows[:n] = x
    rows = rows.reshape(-1, BLOCK)
    top = np.abs(rows).max(1)
    exps = np.ones(len(rows), dtype=np.int64)
    exps[top > 0] = np.maximum(np.floor(np.log2(top[top > 0])).astype(np.int64) + 127 - 7, 1)
    scale = np.repeat(np.exp2(exps - 127.0), BLOCK)[:n]
    y = np.abs(x) / scale
    step = np.exp2(np.floor(np.log2(np.maximum(y, 2.0 ** -6))) - 3)
    low = np.floor(y / step)
    total = (y / step - low) + random16 / 65536.0
    value = (low + (total >= 1)) * step
    if never_zero:
        value = np.where((value == 0) & (x > 0), 2.0 ** -9, value)
    return np.sign(x) * value * scale, exps, np.minimum(np.abs(total - 1), np.minimum(total, np.abs(2 - total))), step * scale


def step(p, g, m, v, *, t, lr, b1, b2, eps, wd, scale=1.0):
    """(p, m, v) after one step on double-precision arrays."""
    g = g * scale
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    p = p * (1 - lr * wd) - lr / (1 - b1 ** t) * m / (np.sqrt(v / (1 - b2 ** t)) + eps)
    return p, m, v
