"""Philox-4x32 with ten rounds in numpy (Salmon, Moraes, Dror, Shaw: Parallel Random Numbers: As Easy as 1, 2, 3, SC 2011)."""
import numpy as np

_WORD = np.uint64(0xffffffff)


def philox(counter, key):
    """[n, 4] words for [n, 4] counters and a pair of key words."""
    c = [np.asarray(counter, dtype=np.uint64)[:, i] for i in range(4)]
    k0, k1 = (int(k) for k in key)
    for r in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64((k0 + r * 0x9E3779B9) & 0xffffffff), b & _WORD,
             (a >> np.uint64(32)) ^ c[3] ^ np.uint64((k1 + r * 0xBB67AE85) & 0xffffffff), a & _WORD]
    return np.stack(c, 1).astype('<u4')


def keep(count, seed, offset, limit, first=0):
    """keep[i] of the decisions from 8 * first on."""
    block = np.arange(first, first + (count + 7) // 8, dtype=np.uint64)
    counter = np.stack([block & _WORD, block >> np.uint64(32), np.full_like(block, offset & 0xffffffff),
                        np.full_like(block, offset >> 32)], 1)
    words = philox(counter, (seed & 0xffffffff, seed >> 32))
    return words.reshape(-1).view('<u2')[:count] >= limit
