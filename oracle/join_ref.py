"""The end of a block in 64 bits and its generator on the host: the oracle of the tests."""
from __future__ import annotations

import numpy as np
import torch


def philox(counter, key):
    """Philox 4x32 of ten rounds (Salmon et al., SC 2011), one counter, in Python's integers."""
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def kept(rows, D, p, seed, salt=0):
    """Which places dropout keeps, (rows, D) bool, for any list of row numbers."""
    key = (seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF)
    least = round(p * 2 ** 32)
    words = [[w for b in range(-(-D // 4)) for w in philox((b, row, salt, 0), key)][:D]
             for row in rows]
    return torch.from_numpy(np.array(words, np.int64).reshape(len(rows), D) >= least)


def block_join(f, h, post=None, gate=None, kind="sigmoid", scale=1.0, pre=None, eps=1e-6,
               mask=None):
    """``(h', x or None)`` in fp64, differentiable; ``mask`` dropout's factors."""
    f, h = f.double(), h.double()
    y = f
    if post is not None:
        y = post.double() * f / torch.sqrt(f.pow(2).mean(-1, keepdim=True) + eps)
    if gate is not None:
        z = gate.double()
        y = y * {"linear": lambda: z, "sigmoid": lambda: torch.sigmoid(z),
                 "silu": lambda: torch.nn.functional.silu(z)}[kind]()
    if mask is not None:
        y = y * mask.double()
    h2 = h + (scale.double() if torch.is_tensor(scale) else scale) * y
    if pre is None:
        return h2, None
    return h2, pre.double() * h2 / torch.sqrt(h2.pow(2).mean(-1, keepdim=True) + eps)
