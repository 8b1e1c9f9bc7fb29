"""Philox4x32-10 (Salmon, Moraes, Dror, Shaw, SC 2011) in numpy, and the dropout mask defined on it."""
import numpy as np


def philox(counter, key):
    """counter: four uint32 arrays (or integers); key: two integers -> four uint32 arrays."""
    c = [np.asarray(v, dtype=np.uint64) for v in counter]
    k = [int(v) for v in key]
    low, hi = np.uint64(0xFFFFFFFF), np.uint64(32)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> hi) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> hi) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    return [v.astype(np.uint32) for v in c]


def bits16(n, seed, offset):
    """The 16 random bits of elements 0 .. n - 1."""
    at = [(offset + b) % 2 ** 64 for b in range((n + 7) // 8)]
    lo, up = np.array([v % 2 ** 32 for v in at]), np.array([v >> 32 for v in at])
    seed %= 2 ** 64
    r = philox([lo, up, np.zeros_like(lo), np.zeros_like(lo)], [seed % 2 ** 32, seed >> 32])
    halves = [h for w in r for h in (w & np.uint32(0xFFFF), w >> np.uint32(16))]
    return np.stack(halves, 1).reshape(-1)[:n].astype(np.int64)
