"""Philox 4x32-10 (Salmon, Moraes, Dror and Shaw, 2011) on numpy words, and the dropout mask made
of it."""
import numpy as np

M32 = np.uint64(0xFFFFFFFF)


def philox(counter, key):
    """counter: 4 arrays (or ints) of 32-bit words, key: 2 ints; 4 arrays of words."""
    c = [np.atleast_1d(np.asarray(v, dtype=np.uint64)) for v in counter]
    k0, k1 = key
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), p1 & M32,
             (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), p0 & M32]
        k0, k1 = (k0 + 0x9E3779B9) % 2 ** 32, (k1 + 0xBB67AE85) % 2 ** 32
    return c


def bits16(rows, cols, seed, offset):
    """The 16 random bits of each element of a [rows, cols] matrix."""
    groups = -(-cols // 8)
    n = np.arange(rows * groups, dtype=np.uint64)
    w = philox([n & M32, n >> np.uint64(32), np.full_like(n, offset % 2 ** 32),
                np.full_like(n, offset >> 32)], (seed % 2 ** 32, seed >> 32))
    b = np.stack([v >> np.uint64(s) & np.uint64(0xFFFF) for v in w for s in (0, 16)], -1)
    return b.reshape(rows, groups * 8)[:, :cols].astype(np.int64)


def keep_mask(rows, cols, seed, offset, p):
    return bits16(rows, cols, seed, offset) >= round(p * 65536)
