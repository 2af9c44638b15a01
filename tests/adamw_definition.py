"""The AdamW step of geomae_amd.optim in numpy, 64 bits: what tests/test_multi_adamw_cpu.py and test_gpu_multi_adamw.py hold
the kernels to.  A code's value comes from a table of the 256 codes; a rounding picks the code below or above."""
import numpy as np

BLOCK = 32
M32 = np.uint64(0xFFFFFFFF)


def code_values(digits, signed):
    out = np.zeros(256)
    top = 128 if signed else 256
    for c in range(256):
        size = c % top
        field, rest = size >> digits, size % (1 << digits)
        v = rest * 2.0 ** (-6 - digits) if field == 0 else (1 + rest / 2.0 ** digits) * 2.0 ** (field - 7)
        out[c] = -v if signed and c >= top else v
    if signed:
        out[127] = out[255] = np.nan
    else:
        out[255] = np.nan
    return out


SIGNED, ROOT = code_values(3, True), code_values(4, False)


def decode(codes, exponents, table):
    return table[codes.astype(np.int64)] * np.repeat(2.0 ** (exponents.astype(np.float64) - 135), BLOCK)[:codes.size]


def mix(x):
    x = x & M32
    x = ((x ^ (x >> np.uint64(15))) * np.uint64(0xBB67AE85)) & M32
    x = ((x ^ (x >> np.uint64(13))) * np.uint64(0x243F6A89)) & M32
    return x ^ (x >> np.uint64(16))


def draws(seed, index, step, n):
    """(16 bits of the first moment, 16 of the second) of elements 0 .. n - 1."""
    old = np.seterr(over="ignore")
    key = mix(mix(np.uint64(seed) + np.uint64(0x9E3779B9) * np.uint64(index)) ^ np.uint64(step & 0xFFFFFFFF))
    h = mix(key + np.arange(n, dtype=np.uint64))
    np.seterr(**old)
    return h & np.uint64(0xFFFF), h >> np.uint64(16)


def exponent(block, table):
    """The exponent byte of a block: the smallest E >= 16 whose largest code is not below the block's largest magnitude."""
    fin = np.abs(block[np.isfinite(block)])
    a = float(fin.max()) if fin.size else 0.0
    if a == 0.0:
        return 16
    top = np.nanmax(table[:128] if table is SIGNED else table)            # 448, 480
    return int(np.clip(np.ceil(np.log2(a / top)) + 135, 16, 254))


def encode(x, u, table):
    """(codes' values, exponents, and for each element the distance of its position from the draw's border in units of the
    step: below ~1e-6 an fp32 computation may land on the other side)."""
    signed = table is SIGNED
    digits = 3 if signed else 4
    n = x.size
    val, exps, margin = np.zeros(n), np.zeros(-(-n // BLOCK), dtype=np.int64), np.ones(n)
    for b in range(exps.size):
        s = slice(b * BLOCK, min(n, (b + 1) * BLOCK))
        e = exps[b] = exponent(x[s], table)
        y = np.abs(x[s]) * 2.0 ** (135 - e)
        with np.errstate(divide="ignore", invalid="ignore"):
            place = np.where(y > 0, np.floor(np.log2(np.where(y > 0, y, 1))), -6)
            place = np.maximum(place, -6)
            step = 2.0 ** (place - digits)
            t = y / step + (u[s].astype(np.float64) + 0.5) / 65536
            k = np.floor(t)
            q = k * step
        margin[s] = np.minimum(t - k, k + 1 - t)
        if not signed:
            q = np.where((q == 0) & (y > 0), 2.0 ** -10, q)
        q = np.where(np.isfinite(x[s]), q, np.nan)
        val[s] = np.copysign(q, x[s]) * 2.0 ** (e - 135.0)
    return val, exps, margin


def step(p, g, m, v, steps, lr, betas, eps, wd, coef=1.0):
    """One update in 64 bits: (p, m, v) of flat arrays; v the second moment itself."""
    b1, b2 = betas
    g = g * coef
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    p = p * (1 - lr * wd) - lr / (1 - b1 ** steps) * m / (np.sqrt(v) / np.sqrt(1 - b2 ** steps) + eps)
    return p, m, v
