"""AdamW with 32- and 8-bit moments in 64-bit numpy, from the formulas: what the kernels of csrc/adamw.hip are held to."""
import numpy as np

BLOCK = 256


def mix(x):
    x = np.uint32(x) if np.isscalar(x) else x.astype(np.uint32)
    with np.errstate(over="ignore"):
        x = (x ^ (x >> np.uint32(16))) * np.uint32(0x6A09E667)
        x = (x ^ (x >> np.uint32(15))) * np.uint32(0xBB67AE85)
    return x ^ (x >> np.uint32(16))


def dither(seed, t, first_block, blocks):
    """(blocks, 256) pairs of 16-bit numbers"""
    k = mix((seed + t * 0x9E3779B9) & 0xFFFFFFFF)
    key = mix(np.array([(int(k) + first_block + b) & 0xFFFFFFFF for b in range(blocks)], np.uint64))
    lanes = (np.arange(BLOCK, dtype=np.uint64) * np.uint64(0x9E3779B9)) & np.uint64(0xFFFFFFFF)
    r = mix((key.astype(np.uint64)[:, None] + lanes[None]) & np.uint64(0xFFFFFFFF))
    return (r >> np.uint32(16)).astype(np.float64), (r & np.uint32(0xFFFF)).astype(np.float64)


def exponent(x):
    """floor(log2 |x|) of the fp32 value, -127 for what fp32 holds as zero or a denormal"""
    a = np.abs(x)
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.where(a > 0, np.frexp(a)[1] - 1, -127)
    return np.maximum(e, -127)


def quantise(x, signed, d):
    """x (blocks, 256) -> (stored values, grid step): three mantissa bits; linear below `octaves` powers of two under the largest"""
    finite = np.isfinite(x)
    top = np.where(finite, exponent(x), -127).max(1, keepdims=True)
    lowest = top - (13 if signed else 29)
    step = 2.0 ** (np.maximum(np.where(finite, exponent(x), -127), lowest) - 3)
    units = np.where(finite, np.abs(x), 0) / step
    up = np.floor(units + (d + 0.5) / 65536)
    if not signed:
        up = np.where((x > 0) & (up == 0), 1, up)
    q = np.sign(np.where(finite, x, 0)) * up * step
    return np.where(finite, q, np.nan if signed else np.inf), step


def blocks_of(x, fill=0.0):
    n = -(-x.size // BLOCK) * BLOCK
    out = np.full(n, fill)
    out[:x.size] = x.reshape(-1)
    return out.reshape(-1, BLOCK)


def step(p, g, m, v, t, lr, b1, b2, eps, wd, clip=1.0):
    g = g * clip
    m = m + (g - m) * (1 - b1)
    v = b2 * v + (1 - b2) * g * g
    p = p * (1 - lr * wd) - lr / (1 - b1 ** t) * m / (np.sqrt(v) / np.sqrt(1 - b2 ** t) + eps)
    return p, m, v
