"""The layer operators in 64 bits with numpy: what tests hold the kernels to.

Philox4x32-10 as published by Salmon, Moraes, Dror and Shaw ("Parallel random numbers: as easy as 1, 2, 3", SC 2011),
section 2 and table 2; the mask's layout as include/epi.h defines it."""
import numpy as np

M32 = 0xFFFFFFFF


def philox4x32(counter, key, rounds=10):
    """One block with Python's integers."""
    c, k = [int(v) for v in counter], [int(v) for v in key]
    for _ in range(rounds):
        p0, p1 = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(p1 >> 32) ^ c[1] ^ k[0], p1 & M32, (p0 >> 32) ^ c[3] ^ k[1], p0 & M32]
        k = [(k[0] + 0x9E3779B9) & M32, (k[1] + 0xBB67AE85) & M32]
    return c


def draws(rows, cols, seed, offset, first_row=0):
    """The 16-bit draws of rows first_row .. first_row + rows - 1."""
    u = np.uint64
    n = -(-cols // 8)
    c = [np.broadcast_to(np.arange(n, dtype=u)[None, :], (rows, n)).copy(),
         np.broadcast_to(np.arange(first_row, first_row + rows, dtype=u)[:, None], (rows, n)).copy(),
         np.full((rows, n), offset & M32, u), np.full((rows, n), (offset >> 32) & M32, u)]
    k = [seed & M32, (seed >> 32) & M32]
    for _ in range(10):
        p0, p1 = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = [(p1 >> u(32)) ^ c[1] ^ u(k[0]), p1 & u(M32), (p0 >> u(32)) ^ c[3] ^ u(k[1]), p0 & u(M32)]
        k = [(k[0] + 0x9E3779B9) & M32, (k[1] + 0xBB67AE85) & M32]
    out = np.stack([h for w in c for h in (w & u(0xFFFF), w >> u(16))], axis=-1)
    return out.reshape(rows, 8 * n)[:, :cols]


def threshold(p):
    return int(np.rint(p * 65536.0))


def factors(rows, cols, p, seed, offset, first_row=0):
    """0 where a unit is dropped, else what it is multiplied by."""
    t = threshold(p)
    if t >= 65536:
        return np.zeros((rows, cols))
    return np.where(draws(rows, cols, seed, offset, first_row) >= t, 65536.0 / (65536 - t), 0.0)


def apply_factors(x, f):
    return np.where(f > 0, x, 0.0) * f


def norm_forward(x, weight, bias, eps):
    """(y, unit values, mean, 1 / deviation)"""
    m = x.mean(axis=1, keepdims=True)
    c = x - m
    c = c - c.mean(axis=1, keepdims=True)
    r = 1.0 / np.sqrt((c * c).mean(axis=1, keepdims=True) + eps)
    u = c * r
    return u * weight + bias, u, m, r


def norm_backward(dy, u, r, weight):
    g = dy * weight
    dh = r * (g - g.mean(axis=1, keepdims=True) - u * (g * u).mean(axis=1, keepdims=True))
    return dh, (dy * u).sum(axis=0), dy.sum(axis=0)
