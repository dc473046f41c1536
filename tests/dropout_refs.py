"""The random bits of dropout with numpy's unsigned integers: Philox 4x32 with 7 rounds (Salmon, Moraes, Dror, Shaw, "Parallel
random numbers: as easy as 1, 2, 3", 2011)."""
import numpy as np


def philox(counter, key, rounds=7):
    """counter: four arrays of 32-bit values in uint64; key: two integers."""
    low, up = np.uint64(0xFFFFFFFF), np.uint64(32)
    c = list(counter)
    for r in range(rounds):
        k = [np.uint64((key[i] + r * w) % 2 ** 32) for i, w in enumerate((0x9E3779B9, 0xBB67AE85))]
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> up) ^ c[1] ^ k[0], b & low, (a >> up) ^ c[3] ^ k[1], a & low]
    return c


def bits_of(n, seed, offset, first=0):
    """16 bits of each of the elements first .. first + n - 1; first a multiple of 8."""
    assert first % 8 == 0
    at = np.arange(-(-n // 8), dtype=np.uint64) + np.uint64(first // 8)
    counter = [at & np.uint64(0xFFFFFFFF), at >> np.uint64(32), np.full_like(at, offset % 2 ** 32), np.full_like(at, offset // 2 ** 32)]
    words = philox(counter, (seed % 2 ** 32, seed // 2 ** 32))
    halves = [h for w in words for h in (w & np.uint64(0xFFFF), w >> np.uint64(16))]
    return np.stack(halves, axis=1).reshape(-1)[:n].astype(np.int64)
