"""Plain references of the AdamW step: the formulas in 64 bits, and the 8-bit moments operation by operation in numpy fp32."""
import math

import numpy as np

BLOCK = 256
M_BASE, V_BASE = 889, 761        # code c > 0: the float whose exponent and three mantissa bits are base + c


def code_values(base, n):
    bits = (np.arange(1, n + 1, dtype=np.int64) + base) << 20
    return np.concatenate([[0.0], bits.astype(np.uint32).view(np.float32)]).astype(np.float64)


def encode(t, base, least):
    """Nearest code of t in [0, 1] by the float's value (numpy's frexp, rint: ties to even), not by its bits."""
    t = np.asarray(t, np.float32).astype(np.float64)
    f, e = np.frexp(t)
    q = np.ldexp(np.rint(f * 16) / 16, e)
    smallest = float((np.array([base + 1], np.uint32) << 20).view(np.float32)[0])
    f, e = np.frexp(np.maximum(q, smallest))
    code = (e.astype(np.int64) + 126) * 8 + np.rint((f * 2 - 1) * 8).astype(np.int64) - base
    code = np.where(q < smallest, least, code)
    return np.where(t > 0, code, 0).astype(np.int64)


def decode(code, scale, base, signed):
    c = np.asarray(code).astype(np.int64)
    k = c & 127 if signed else c
    t = np.where(k > 0, ((k + base) << 20), 0).astype(np.uint32).view(np.float32)
    x = (t * np.float32(scale)).astype(np.float32)
    return np.where(c > 127, -x, x).astype(np.float32) if signed else x


def to8(x, base, least, signed):
    """One tensor's values (fp32 array) -> codes, scales."""
    n = len(x)
    pad = np.zeros(-(-n // BLOCK) * BLOCK, np.float32)
    pad[:n] = x
    blocks = pad.reshape(-1, BLOCK)
    scale = np.abs(blocks).max(1).astype(np.float32)
    with np.errstate(invalid="ignore", divide="ignore"):
        t = (np.abs(blocks) / np.where(scale > 0, scale, np.float32(1))[:, None]).astype(np.float32)
    code = encode(t, base, least)
    if signed:
        code = code + 128 * (blocks < 0)
    return code.reshape(-1)[:n].astype(np.uint8), scale


def from8(code, scale, base, signed):
    return decode(code, np.repeat(scale, BLOCK)[:len(code)], base, signed)


def factor_and_norm(grads, grad_scale, max_norm):
    norm = math.sqrt(sum(float((g.astype(np.float64) ** 2).sum()) for g in grads if g is not None)) * abs(grad_scale)
    c = min(1.0, max_norm / (norm + 1e-6)) if max_norm else 1.0
    return grad_scale * c, norm


def step64(p, m, v, g, t, lr, b1, b2, eps, wd):
    """The definition, in 64 bits; returns new (p, m, v)."""
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    return p * (1 - lr * wd) - lr / (1 - b1 ** t) * m / (np.sqrt(v) / math.sqrt(1 - b2 ** t) + eps), m, v


def moments32(m, v, g, factor, b1, b2):
    """The moments with every operation rounded to fp32 on its own, as the kernel does."""
    f = np.float32
    g = g.astype(f) * f(factor)
    return (m * f(b1)) + (g * f(1 - b1)), (v * f(b2)) + ((g * g) * f(1 - b2))
