"""4-bit microscaled matrices in 64-bit numpy, from the definitions (test infrastructure only)."""
import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
NAN_SCALE = 255


def philox_words(rows, cols, key, counter=0):
    """32 random bits an element: word c % 4 of Philox4x32-10 at counter + r * ceil(cols / 4) + c // 4."""
    quads = (cols + 3) // 4
    at = [counter + i for i in range(rows * quads)]
    c = [np.array([(a >> (32 * w)) & 0xFFFFFFFF for a in at], dtype=np.uint64) for w in range(4)]
    k0, k1 = key & 0xFFFFFFFF, (key >> 32) & 0xFFFFFFFF
    u = np.uint64
    for _ in range(10):
        p0, p1 = u(0xD2511F53) * c[0], u(0xCD9E8D57) * c[2]
        c = [(p1 >> u(32)) ^ c[1] ^ u(k0), p1 & u(0xFFFFFFFF), (p0 >> u(32)) ^ c[3] ^ u(k1), p0 & u(0xFFFFFFFF)]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(c, 1).reshape(rows, quads * 4)[:, :cols]


def quantize(x, words=None):
    """codes (rows x padded columns, one a byte) and scale bytes (rows x blocks) of x; words: stochastic."""
    rows, cols = x.shape
    nb = (cols + 31) // 32
    p = np.zeros((rows, nb * 32))
    p[:, :cols] = x
    p = p.reshape(rows, nb, 32)
    bad = ~np.isfinite(p).all(2)
    p = np.where(bad[:, :, None], 0.0, p)
    top = np.abs(p).max(2)
    mant, e = np.frexp(top)   # top = mant 2^e, 0.5 <= mant < 1
    e = e - 3
    if words is not None:
        e = e + (mant > 0.75)
    e = np.clip(np.where(top == 0, -127, e), -127, 125)
    v = np.minimum(np.ldexp(np.abs(p), -e[:, :, None]), 6.0)
    low = np.searchsorted(GRID, v.ravel(), side="right").reshape(v.shape) - 1
    high = np.minimum(low + 1, 7)
    gap = np.where(high > low, GRID[high] - GRID[low], 1.0)
    part = (v - GRID[low]) / gap
    if words is None:
        up = (part > 0.5) | ((part == 0.5) & (low % 2 == 1))   # ties to the even code
    else:
        w = np.zeros((rows, nb * 32))
        w[:, :cols] = words
        up = w.reshape(v.shape) < np.floor(part * 2.0 ** 32)
    code = low + up + 8 * np.signbit(p)
    code = np.where(bad[:, :, None], 0, code).astype(np.uint8)
    scale = np.where(bad, NAN_SCALE, e + 127).astype(np.uint8)
    return code.reshape(rows, nb * 32), scale


def pack(code):
    return (code[:, 0::2] | (code[:, 1::2] << 4)).astype(np.uint8)


def values(codes, scales, cols):
    """The matrix that packed codes and scales stand for, in 64 bits."""
    c = np.stack((codes & 15, codes >> 4), 2).reshape(codes.shape[0], -1)
    v = np.where(c & 8, -1.0, 1.0) * GRID[c & 7]
    s = np.where(scales == NAN_SCALE, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return (v * np.repeat(s, 32, 1)[:, : c.shape[1]])[:, :cols]


def random_mx4(rng, rows, cols, low=120, high=130):
    """Random codes and scales in [low, high], the padding zero: (packed codes, scales)."""
    nb = (cols + 31) // 32
    code = rng.integers(0, 16, (rows, nb * 32)).astype(np.uint8)
    code[:, cols:] = 0
    return pack(code), rng.integers(low, high + 1, (rows, nb)).astype(np.uint8)
