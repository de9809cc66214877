"""Dropout's mask by its definition, in numpy, for the tests of the residual
stream's operators: Philox4x32-10 (Salmon et al., SC'11) from its paper."""

import numpy as np
import torch


def philox(counter, key):
    """Blocks of counters [n, 4] under the key (k0, k1): [n, 4] uint64 words."""
    c = [counter[:, i].astype(np.uint64) for i in range(4)]
    k0, k1 = np.uint64(key[0]), np.uint64(key[1])
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    for i in range(10):
        if i:
            k0, k1 = (k0 + np.uint64(0x9E3779B9)) & low, (k1 + np.uint64(0xBB67AE85)) & low
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> half) ^ c[1] ^ k0, b & low, (a >> half) ^ c[3] ^ k1, a & low]
    return np.stack(c, axis=1)


def bits(first, n, seed, call):
    """The 32 bits of elements first .. first + n - 1."""
    e = np.arange(first, first + n, dtype=np.uint64)
    halves = []
    for stream in (0, 1):
        blocks = np.unique(e >> np.uint64(3))
        counter = np.stack([blocks & np.uint64(0xFFFFFFFF), blocks >> np.uint64(32),
                            np.full_like(blocks, stream), np.full_like(blocks, call)], axis=1)
        words = philox(counter, (seed & 0xFFFFFFFF, seed >> 32 & 0xFFFFFFFF))
        half = np.stack([words >> np.uint64(s) & np.uint64(0xFFFF) for s in (0, 16)], axis=2)
        half = half.reshape(len(blocks), 8)
        halves.append(half[(e >> np.uint64(3)) - blocks[0], e & np.uint64(7)])
    return (halves[0] << np.uint64(16)) | halves[1]


def kept(shape, p, seed, call, first=0):
    """Whether each element is kept, a bool tensor on the CPU."""
    n = int(np.prod(shape))
    limit = np.uint64(int(np.floor(p * 2.0 ** 32 + 0.5)))
    return torch.from_numpy(bits(first, n, seed, call) >= limit).view(shape)
