"""Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC'11)
in Python integers, and the dropout mask drawn from it."""

import numpy as np


def philox4x32(counter, key, rounds=10):
    """The four output words of one counter block."""
    c, k = list(counter), list(key)
    for _ in range(rounds):
        a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def keep_mask(rows, cols, p, seed, call):
    """bool [len(rows), cols]: the elements that dropout keeps."""
    limit = round(p * 2 ** 32)
    key = (seed & 0xFFFFFFFF, seed >> 32)
    out = np.empty((len(rows), (cols + 3) // 4 * 4), dtype=bool)
    for i, r in enumerate(rows):
        for b in range((cols + 3) // 4):
            words = philox4x32((b, int(r) & 0xFFFFFFFF, call & 0xFFFFFFFF, call >> 32), key)
            out[i, 4 * b:4 * b + 4] = [w >= limit for w in words]
    return out[:, :cols]
