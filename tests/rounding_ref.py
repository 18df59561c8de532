"""The random rounding of the 8-bit moments, operation by operation in numpy: which bits decide, and the codes they give."""
import numpy as np

from optim_ref import BLOCK

M_SALT, V_SALT = 0, 2            # a quad of elements takes two words for its first moments, two for its second
U32 = np.uint32


def word(quad, step, salt):
    """32 bits for a quad of elements (its number among all of the state), a step count and a salt."""
    quad = np.asarray(quad, np.uint64)
    lo, hi = (quad & np.uint64(0xFFFFFFFF)).astype(U32), (quad >> np.uint64(32)).astype(U32)
    with np.errstate(over="ignore"):
        h = lo ^ (hi * U32(0xA54FF53B)) ^ (U32(4 * step + salt & 0xFFFFFFFF) * U32(0xBB67AE85))
        for shift, factor in ((16, 0x3C6EF373), (15, 0xBB67AE85), (16, 0xA54FF53B)):
            h = (h ^ (h >> U32(shift))) * U32(factor)
        return h ^ (h >> U32(15))


def offsets(n, first_quad, step, salt):
    """For each of n elements from quad first_quad on: 16 random bits in the middle of the 20 that a code drops."""
    quads = np.arange(first_quad, first_quad + -(-n // 4), dtype=np.uint64)
    a, b = word(quads, step, salt), word(quads, step, salt + 1)
    r = np.stack([a & U32(0xFFFF), a >> U32(16), b & U32(0xFFFF), b >> U32(16)], 1).reshape(-1)[:n]
    return (r << U32(4)) | U32(8)


def to8_random(x, base, least, signed, first_block, step):
    """One tensor's values (fp32 array) -> codes, scales."""
    n = len(x)
    pad = np.zeros(-(-n // BLOCK) * BLOCK, np.float32)
    pad[:n] = x
    blocks = pad.reshape(-1, BLOCK)
    scale = np.abs(blocks).max(1).astype(np.float32)
    t = (np.abs(blocks) / np.where(scale > 0, scale, np.float32(1))[:, None]).astype(np.float32).reshape(-1)
    r = offsets(len(pad), first_block * BLOCK // 4, step, M_SALT if signed else V_SALT)
    bits = t.view(U32)
    code = ((bits + r) >> U32(20)).astype(np.int64) - base
    smallest = np.array([(base + 1) << 20], U32).view(np.float32)[0]
    below = np.full(t.shape, 1) if least else (r.astype(np.float32) < t * (np.float32(2.0 ** 20) / smallest)).astype(np.int64)
    code = np.where(t < smallest, below, code)
    code = np.where(t > 0, code, 0)
    if signed:
        code = code + 128 * ((pad < 0) & (code > 0))
    return code[:n].astype(np.uint8), scale
