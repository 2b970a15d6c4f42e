"""Philox4x32-10 (Salmon, Moraes, Dror and Shaw, 2011) in numpy, and the dropout mask made from it."""
import math

import numpy as np

M0, M1 = np.uint64(0xD2511F53), np.uint64(0xCD9E8D57)
LOW, S32 = np.uint64(0xFFFFFFFF), np.uint64(32)


def philox4x32(counter, key):
    """counter [n, 4], key (2 words) -> [n, 4] uint32."""
    c = [np.asarray(counter)[:, i].astype(np.uint64) for i in range(4)]
    k = [int(key[0]), int(key[1])]
    for _ in range(10):
        p0, p1 = c[0] * M0, c[2] * M1
        c = [(p1 >> S32) ^ c[1] ^ np.uint64(k[0]), p1 & LOW, (p0 >> S32) ^ c[3] ^ np.uint64(k[1]), p0 & LOW]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, 1).astype(np.uint32)


def keep_mask(start, n, rate, seed, call):
    """Which of the elements start .. start + n - 1 are kept."""
    j = np.arange(start // 4, (start + n + 3) // 4, dtype=np.uint64)
    seed, call = seed % 2 ** 64, call % 2 ** 64
    ctr = np.stack([j & LOW, j >> S32, np.full_like(j, call & 0xFFFFFFFF), np.full_like(j, call >> 32)], 1)
    words = philox4x32(ctr, (seed & 0xFFFFFFFF, seed >> 32)).reshape(-1)
    off = start - 4 * (start // 4)
    return words[off:off + n] >= np.uint32(math.floor(rate * 2.0 ** 32))
