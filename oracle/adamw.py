"""AdamW from the formulas (numpy): the step in 64 bits, and the 8-bit moments with their codes.

The codes' arithmetic is in 64 bits with the roundings to fp32 that the definition has written
out, apart from the bit operations by which the kernels do the same."""

import numpy as np

BLOCK = 256


def step(g, p, m, v, t, lr, beta1, beta2, eps, weight_decay, inv_scale=1.0, clip=1.0):
    """(p, m, v) after step t, in 64 bits."""
    g, p, m, v = (np.asarray(x, np.float64) for x in (g, p, m, v))
    g = g * inv_scale * clip
    m = beta1 * m + (1 - beta1) * g
    v = beta2 * v + (1 - beta2) * g * g
    update = (m / (1 - beta1 ** t)) / (np.sqrt(v / (1 - beta2 ** t)) + eps)
    return p - lr * weight_decay * p - lr * update, m, v


def magnitude(c):
    """F(c) of codes without their sign."""
    c = np.asarray(c, np.int64)
    return np.where(c < 8, c / 8.0, (1 + (c & 7) / 8.0) * np.exp2((c >> 3) - 1.0))


def random_words(blocks, seed, first=0):
    """The words of `blocks` blocks from number `first` on, [blocks, 256], as integers below 2^32."""
    low = 0xFFFFFFFF
    q = [(b * 64 + i) for b in range(first, first + blocks) for i in range(64)]
    out = np.empty((blocks * 64, 4), np.int64)
    for row, n in enumerate(q):
        x = ((n & low) ^ (seed & low)) * 0x9E3779B9 & low
        x = ((x ^ x >> 16) + (seed >> 32 & low) + (n >> 32)) * 0x6A09E667 & low
        x ^= x >> 15
        for e, c in enumerate((0xBB67AE85, 0x510E527F, 0x1F83D9AB, 0x5BE0CD19)):
            w = x * c & low
            out[row, e] = w ^ w >> 16
    return out.reshape(blocks, BLOCK)


def exponent(largest):
    """E of a block whose largest magnitude is the fp32 number `largest`."""
    largest = float(largest)
    if not np.isfinite(largest):
        return 255
    mantissa, e = np.frexp(largest)          # 1/2 <= mantissa < 1
    if largest < 2.0 ** -126:                # denormal: the exponent field is 0, or 1 from 1.875 units on
        return 1 if largest >= 0.875 * 2.0 ** -126 else 0
    return int(e + 126 + (mantissa >= 0.9375))


def encode(x, e, bias, u, least):
    """Codes of magnitudes x (fp32) in a block with exponent e; u in [0, 1): the place between two codes
    from which on the upper one is taken is 1 - u."""
    # units of F; fp32 holds them to 2^-23 below 1
    y = np.asarray(x, np.float64) * 2.0 ** (bias - e)
    y = np.where(y < 1, np.rint(y * 2.0 ** 23) / 2.0 ** 23, y)
    octave = np.maximum(np.floor(np.log2(np.maximum(y, 1e-300))), 0).astype(np.int64)
    steps = np.floor(y / np.exp2(octave - 3.0) + u).astype(np.int64)      # 8 to 16 of them, below 1: 0 to 8
    code = np.where(y < 1, steps, (octave + 1) * 8 + steps - 8)
    if least:
        code = np.where((code == 0) & (np.asarray(x) > 0), 1, code)
    return code


def decode(codes, exponents):
    """(m, v) of codes [blocks, 512] and exponents [blocks, 2], [blocks, 256] in 64 bits."""
    c = np.asarray(codes, np.int64).reshape(-1, 64, 2, 4)
    e = np.asarray(exponents, np.int64)
    cm, cv = (c[:, :, i].reshape(-1, BLOCK) for i in (0, 1))
    m = magnitude(cm & 127) * np.exp2(e[:, :1] - 141.0) * np.where(cm & 128, -1.0, 1.0)
    v = magnitude(cv) * np.exp2(e[:, 1:] - 157.0)
    return np.where(e[:, :1] == 255, np.nan, m), np.where(e[:, 1:] == 255, np.nan, v)


def quantize(m, v, words):
    """(codes [blocks, 512], exponents [blocks, 2]) of fp32 moments [blocks, 256]."""
    blocks = m.shape[0]
    codes, exponents = np.zeros((blocks, 64, 2, 4), np.uint8), np.zeros((blocks, 2), np.uint8)
    for b in range(blocks):
        for i, (x, bias, u) in enumerate(((m[b], 141, words[b] & 0xFFFF), (v[b], 157, words[b] >> 16))):
            e = exponent(np.abs(x).max())
            exponents[b, i] = e
            if e == 255:
                continue
            c = encode(np.abs(x), e, bias, (u + 0.5) / 65536, i == 1)
            if i == 0:
                c = c | np.where(x < 0, 128, 0)
            codes[b, :, i] = c.reshape(64, 4)
    return codes.reshape(blocks, 2 * BLOCK), exponents


def moments_step(g, m, v, beta1, beta2, inv_scale=1.0, clip=1.0):
    """(m, v) after a step, every product and sum rounded to fp32 by itself."""
    f = np.float32
    with np.errstate(over="ignore", invalid="ignore"):
        g = np.asarray(g, f) * f(inv_scale) * f(clip)
        m = m + (g - m) * f(1.0 - beta1)
        v = v * f(beta2) + f(1.0 - beta2) * g * g
    assert m.dtype == v.dtype == f
    return m, v


def step8(g, p, codes, exponents, seed, t, lr, beta1, beta2, eps, weight_decay, inv_scale=1.0, clip=1.0, first=0):
    """(p in 64 bits, codes, exponents) of one tensor's step; its first block has number `first`."""
    n, blocks = len(p), len(exponents)
    pad = lambda x: np.concatenate([np.asarray(x, np.float32), np.zeros(blocks * BLOCK - n, np.float32)]).reshape(blocks, BLOCK)  # noqa: E731
    m0, v0 = (x.astype(np.float32) for x in decode(codes, exponents))
    m, v = moments_step(pad(g), m0, v0, beta1, beta2, inv_scale, clip)
    behind = np.arange(blocks * BLOCK).reshape(blocks, BLOCK) >= n
    m[behind] = v[behind] = 0
    m64, v64 = (x.reshape(-1)[:n].astype(np.float64) for x in (m, v))
    p = np.asarray(p, np.float64)
    update = (m64 / (1 - beta1 ** t)) / (np.sqrt(v64 / (1 - beta2 ** t)) + eps)
    return (p - lr * weight_decay * p - lr * update, *quantize(m, v, random_words(blocks, seed, first)))
