"""Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as
easy as 1, 2, 3", SC 2011) from its definition, and dropout's use of it."""
import numpy as np

LOW = np.uint64(0xFFFFFFFF)


def philox(ctr, key):
    """ctr: four arrays or numbers of 32 bits, key: two numbers.  Four arrays of 32 bits."""
    c = [np.asarray(x, np.uint64) for x in ctr]
    k = [int(x) for x in key]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & LOW, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & LOW]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return [x.astype(np.uint32) for x in c]


def numbers(rows, width, seed, offset, row0=0):
    """The 16-bit numbers of [rows, width]."""
    chunks = (width + 7) // 8
    c, r = np.meshgrid(np.arange(chunks), np.arange(row0, row0 + rows))
    ctr = (c, r, np.full_like(c, offset & 0xFFFFFFFF), np.full_like(c, offset >> 32))
    words = np.stack(philox(ctr, (seed & 0xFFFFFFFF, seed >> 32)), -1)
    return np.stack([words & 0xFFFF, words >> 16], -1).reshape(rows, chunks * 8)[:, :width].astype(np.int64)


def kept(rows, width, p, seed, offset):
    return numbers(rows, width, seed, offset) >= round(65536 * p)
