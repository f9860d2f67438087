"""Philox4x32 with ten rounds (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011) in numpy's
unsigned integers: the words that decide which elements dropout keeps."""
import numpy as np

M0, M1, W0, W1, LOW = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85, 0xFFFFFFFF


def block(counter, key):
    """counter: four arrays of 32-bit words (uint64), key: two integers -> four arrays"""
    u = np.uint64
    c = [np.asarray(v, dtype=u) for v in counter]
    k0, k1 = key
    for _ in range(10):
        a, b = c[0] * u(M0), c[2] * u(M1)
        c = [(b >> u(32)) ^ c[1] ^ u(k0), b & u(LOW), (a >> u(32)) ^ c[3] ^ u(k1), a & u(LOW)]
        k0, k1 = (k0 + W0) & LOW, (k1 + W1) & LOW
    return c


def words(n, seed, call, first=0):
    """the words of elements first .. first+n-1 (first a multiple of 4)"""
    at = np.arange(first // 4, first // 4 + (n + 3) // 4, dtype=np.uint64)
    same = np.ones_like(at)
    c = block([at & np.uint64(LOW), at >> np.uint64(32), same * np.uint64(call & LOW), same * np.uint64(call >> 32)], (seed & LOW, seed >> 32))
    return np.stack(c, 1).reshape(-1)[:n].astype(np.uint32)
