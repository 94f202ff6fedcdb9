"""The gated delta rule and drafted trees in 64 bits, token by token: the oracle of the tests.

Plain torch on whatever device the inputs are on; inputs of any type are taken to fp64 as they
are, so a comparison sees the kernels' arithmetic alone.
"""
from __future__ import annotations

import torch


def delta_scan(Q, K, V, logA, beta, scale=1.0, state=None, offsets=None):
    """``(o, state_out)`` of ``gated_delta_scan`` in fp64, differentiable; ``offsets`` the
    segments' borders (then states have the leading segment axis)."""
    Q, K, V, logA, beta = (t.double() for t in (Q, K, V, logA, beta))
    nb, group = V.shape[0], V.shape[0] // Q.shape[0]
    Q, K = (t.repeat_interleave(group, 0) for t in (Q, K))
    off = offsets if offsets is not None else [0, V.shape[1]]
    outs, states = [], []
    for i, (t0, t1) in enumerate(zip(off, off[1:])):
        if state is None:
            S = V.new_zeros(nb, Q.shape[2], V.shape[2])
        else:
            S = (state[i] if offsets is not None else state).double()
        for t in range(t0, t1):
            S = S * torch.exp(logA[:, t])[:, None, None]
            u = beta[:, t, None] * (V[:, t] - (K[:, t, :, None] * S).sum(1))
            S = S + K[:, t, :, None] * u[:, None]
            outs.append(scale * (Q[:, t, :, None] * S).sum(1))
        states.append(S)
    o = torch.stack(outs, 1) if outs else V.new_zeros(nb, 0, V.shape[2])
    return o, torch.stack(states) if offsets is not None else states[0]


def tree_nodes(Phi, Psi, Vb, parents, S, U, at):
    """``(out, states)`` of one request's sequences (heads, M, .): the outputs of every node and
    the state behind each, node by node; ``at`` the position of the first drafted token."""
    Phi, Psi, Vb, S, U = (t.double() for t in (Phi, Psi, Vb, S, U))
    out, states, depth = [], [], []
    for j, a in enumerate(parents):
        if a == -2:
            out.append(torch.zeros_like(Vb[:, j, :-1]))
            states.append(None)
            depth.append(None)
            continue
        depth.append(0 if a < 0 else depth[a] + 1)
        Sj = (S if a < 0 else states[a]) + Psi[:, j, :, None] * Vb[:, j, None]
        states.append(Sj)
        N = (Phi[:, j, :, None] * (Sj + U[:, (at + depth[j]) % U.shape[1]])).sum(1)
        out.append(N[:, :-1] / N[:, -1:])
    return torch.stack(out, 1), states
