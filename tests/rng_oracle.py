"""Independent host reference of the dropout generator: Philox4x32-10 in numpy uint64."""
import numpy as np


def philox(ctr, key):
    """ctr [n, 4], key (2,) -> [n, 4] uint32."""
    c = [ctr[:, j].astype(np.uint64) for j in range(4)]
    k = [int(key[0]), int(key[1])]
    m = np.uint64(0xFFFFFFFF)
    s = np.uint64(32)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> s) ^ c[1] ^ np.uint64(k[0]), b & m, (a >> s) ^ c[3] ^ np.uint64(k[1]), a & m]
        k = [(k[0] + 0x9E3779B9) % 2**32, (k[1] + 0xBB67AE85) % 2**32]
    return np.stack(c, 1).astype(np.uint32)


def keep(index, rate, seed, step):
    """bool keep bit of each mask index (any integer array)."""
    idx = np.asarray(index, dtype=np.uint64).reshape(-1)
    seed, step = seed % 2**64, step % 2**64
    blk, inv = np.unique(idx >> np.uint64(3), return_inverse=True)
    ctr = np.stack([blk & np.uint64(0xFFFFFFFF), blk >> np.uint64(32), np.full(len(blk), step % 2**32, np.uint64),
                    np.full(len(blk), step >> 32, np.uint64)], 1)
    w = philox(ctr, (seed % 2**32, seed >> 32))[inv]
    j = (idx & np.uint64(7)).astype(np.int64)
    piece = (w[np.arange(len(idx)), j // 2] >> (16 * (j % 2)).astype(np.uint32)) & np.uint32(0xFFFF)
    return (piece >= round(rate * 65536)).reshape(np.shape(index))


def scale(rate):
    thr = round(rate * 65536)
    return 65536.0 / (65536 - thr) if thr < 65536 else 0.0


def shared_index(shape, noise):
    """Mask index of every element of ``shape`` under the mask shape ``noise``."""
    return np.broadcast_to(np.arange(int(np.prod(noise))).reshape(noise), shape)
