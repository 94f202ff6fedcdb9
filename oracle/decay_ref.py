"""Linear attention with a decay for each head in 64 bits, token by token: the oracle of the tests.

Plain torch on whatever device the inputs are on; inputs of any type are taken to fp64 as they
are, so a comparison sees the kernels' arithmetic alone.
"""
from __future__ import annotations

import torch


def head_decay_scan(Q, K, V, logA, scale=1.0, state=None, offsets=None):
    """``(o, state_out)`` of ``head_decay_scan`` in fp64, differentiable; ``offsets`` the
    segments' borders (then states have the leading segment axis)."""
    Q, K, V, logA = (t.double() for t in (Q, K, V, logA))
    nb, group = V.shape[0], V.shape[0] // Q.shape[0]
    Q, K = (t.repeat_interleave(group, 0) for t in (Q, K))
    a = torch.exp(logA).repeat(nb // len(logA))[:, None, None]
    off = offsets if offsets is not None else [0, V.shape[1]]
    outs, states = [], []
    for i, (t0, t1) in enumerate(zip(off, off[1:])):
        if state is None:
            S = V.new_zeros(nb, Q.shape[2], V.shape[2])
        else:
            S = (state[i] if offsets is not None else state).double()
        for t in range(t0, t1):
            S = a * S + K[:, t, :, None] * V[:, t, None]
            outs.append(scale * (Q[:, t, :, None] * S).sum(1))
        states.append(S)
    o = torch.stack(outs, 1) if outs else V.new_zeros(nb, 0, V.shape[2])
    return o, torch.stack(states) if offsets is not None else states[0]
