"""Philox4x32-10 in numpy, and the dropout mask made from it."""

from __future__ import annotations

import numpy as np


def philox4x32_10(counter, key):
    """counter: four uint32 arrays (or numbers), key: two numbers; four uint32 arrays."""
    c = [np.atleast_1d(np.asarray(v, dtype=np.uint64)) for v in counter]
    k = [int(v) for v in key]
    low = np.uint64(0xFFFFFFFF)
    for _ in range(10):
        p, q = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(q >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), q & low, (p >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), p & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return [v.astype(np.uint32) for v in c]


def dropout_words(seed: int, offset: int, begin: int, count: int) -> np.ndarray:
    """The 16-bit words of elements begin .. begin + count - 1."""
    first, last = begin // 8, (begin + count + 7) // 8
    i = np.arange(first, max(last, first + 1), dtype=np.uint64)
    seed, offset = seed % 2**64, offset % 2**64
    words = philox4x32_10((i & np.uint64(0xFFFFFFFF), i >> np.uint64(32), offset & 0xFFFFFFFF, offset >> 32),
                          (seed & 0xFFFFFFFF, seed >> 32))
    w = np.stack(words, 1)
    halves = np.stack((w & np.uint32(0xFFFF), w >> np.uint32(16)), 2).reshape(-1)
    return halves[begin - 8 * first:][:count]
