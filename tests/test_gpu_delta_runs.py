"""Sequences cut into runs, and the gates' gradients, to the bits that fp32 sums leave.

Roundings are independent and at most 2^-24 of the value, 2^-24 / sqrt(3) in the root mean
square: after n of them sqrt(n / 3) 2^-24 is left, and the tests allow twice that of a result's
norm, beside the rounding of what is stored in 16 bits.

Runs.  Slow decays, weak writes (beta <= 0.03) and a state larger than them let the runs'
transitions carry what a sequence ends with.  What K S and U round enters a state through beta
and is lost beside it; a state is rounded where K^T U is added to it, two steps of 32 tokens
for up to 6 pairs of terms, and where it is scaled by a decay that is itself off by up to two:
13 + 4, and 20 with the runs' products (6 ceil(r / 32) for 4 chunks or more) spread over them.
Its gradient takes two such sums, Q^T dO and K^T Z: 32.  What is formed from both takes 52, and
four chunks more stand for the one product that a result is.  With transitions of two terms
(2^-17) the states and their gradients are beyond these limits, which
`test_the_limit_sees_two_terms` shows.

Whole sequences of few chunks: every sum's roundings count, 6 ceil(r / 32) in K S, 12 in T, 12
in K^T U and a few in the factors, in the state's chunks and in its gradient's.  dlogA with
resets is measured against the terms of its sums, which cancel there.
"""
import math

import pytest
import torch

import oracle.delta_ref as O
from test_gpu_delta import BF16, DEV, FP16, FP32, _inputs

if torch.cuda.is_available():
    from smat_attention_amd import attention as A

NAMES = ("dq", "dk", "dv", "dlogA", "dbeta", "dS0")


def _noise(n):
    return 2 * math.sqrt(n / 3) * 2.0 ** -24


def _limit(name, chunks):
    a_chunk = {"S": 20, "o": 20, "dq": 20, "dS0": 32, "dv": 32}.get(name, 52)
    return _noise(a_chunk * (chunks + 4))


def _near(name, got, ref, lim, size=None):
    got, ref = got.detach(), ref.detach()
    assert torch.isfinite(got).all(), name
    off = (got.double() - ref).norm().item()
    once = (ref.to(got.dtype).double() - ref).norm().item() if got.dtype != FP32 else 0.0
    size = ref.norm().item() if size is None else size
    assert off <= once + lim * size, (name, off, once, size)


def _weak(nb, nbk, T, r, p, dtype, seed, lead):
    """Inputs whose states live long: about a third of S0 is left after 2600 tokens."""
    q, k, v, logA, beta, S = _inputs(nb, nbk, T, r, p, dtype, seed=seed, state=lead, decay=1e-3)
    return q, k, v, logA, beta * 0.03, S * 4


SHAPES = [
    # nb, nbk, T, r, p, offsets
    (2, 2, 64 * 41 + 9, 24, 40, None),
    (4, 2, 64 * 38, 96, 72, None),
    (1, 1, 64 * 40 + 1, 64, 64, None),
    (2, 1, 64 * 45 + 1, 128, 48, [0, 64 * 30 + 3, 64 * 30 + 3, 64 * 45 + 1]),
    (2, 2, 64 * 44, 80, 100, [0, 64 * 22 + 40, 64 * 44]),
    (3, 1, 64 * 36 + 50, 17, 200, [0, 64 * 36 + 40, 64 * 36 + 50]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("nb,nbk,T,r,p,off", SHAPES)
def test_runs(dtype, nb, nbk, T, r, p, off):
    """Outputs, states and every gradient, with gradients of o and of the returned state."""
    from smat_attention_amd.kernels.hip_delta import _Plan
    lead = () if off is None else (len(off) - 1,)
    x = [t.requires_grad_(True) for t in _weak(nb, nbk, T, r, p, dtype, T + r, lead)]
    seg = None if off is None else A.Segments(off, DEV)
    assert _Plan("test", x[0], x[2], seg).nruns > (len(seg) if seg else 1)
    got = A.gated_delta_scan(*x[:5], state=x[5], segments=seg, return_state=True)
    y = [t.detach().double().requires_grad_(True) for t in x]
    ref = O.delta_scan(*y[:5], state=y[5], offsets=off)
    chunks = max(-(-(b - a) // 64) for a, b in zip(off or [0], (off or [0, T])[1:]))
    _near("o", got[0], ref[0], _limit("o", chunks))
    _near("S", got[1], ref[1], _limit("S", chunks))
    g = torch.Generator().manual_seed(14)
    d = [torch.randn(t.shape, generator=g).to(t.dtype).to(DEV) for t in got]
    got = torch.autograd.grad(got, x, d)
    ref = torch.autograd.grad(ref, y, [t.double() for t in d])
    for name, a, b in zip(NAMES, got, ref):
        _near(name, a, b, _limit(name, chunks))


def _dlogA_terms(y, d):
    """The norm of what dlogA is summed from.  In a chunk dlogA_t is the sum over i >= t of
    q_i.dq_i, of k_i against its gradient as it reads the state and against that as it writes,
    plus <dS', S'> at the chunk's end (which is dlogA of the token behind it).  Those terms are
    off by their own roundings, whatever they sum to; ahead of a reset, whose sum is zero, they
    cancel."""
    q, k, v, logA, beta, S = y
    group = v.shape[0] // q.shape[0]
    heads = lambda t: t.detach().repeat_interleave(group, 0).requires_grad_(True)
    Q, read, write = heads(q), heads(k), heads(k)
    S, out = S.detach(), []
    la = logA.detach().clone().requires_grad_(True)
    T = v.shape[1]
    for t in range(T):
        S = S * torch.exp(la[:, t])[:, None, None]
        u = beta[:, t, None].detach() * (v[:, t].detach() - (read[:, t, :, None] * S).sum(1))
        S = S + write[:, t, :, None] * u[:, None]
        out.append((Q[:, t, :, None] * S).sum(1))
    g = torch.autograd.grad((torch.stack(out, 1), S), (Q, read, write, la),
                            [t.double() for t in d])
    x = sum((a * b).sum(-1) ** 2 for a, b in zip((Q, read, write), g)).detach()
    last = (S.detach().flatten(1).norm(dim=1) * d[1].double().flatten(1).norm(dim=1)
            / math.sqrt(S[0].numel()))
    total = 0.0
    for t0 in range(0, T, 64):
        t1 = min(t0 + 64, T)
        end = (last if t1 == T else g[3][:, t1].abs()) ** 2
        total += (x[:, t0:t1].flip(1).cumsum(1) + end[:, None]).sum().item()
    return math.sqrt(total)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("kind", ["plain", "resets", "only the state's"])
@pytest.mark.parametrize("nb,nbk,T,r,p", [(2, 2, 129, 128, 256), (2, 1, 63, 128, 128),
                                          (3, 3, 140, 40, 64), (2, 2, 7, 96, 33)])
def test_gradients_with_a_state_gradient(dtype, kind, nb, nbk, T, r, p):
    """Whole sequences, where a gradient comes in through the returned state."""
    x = _inputs(nb, nbk, T, r, p, dtype, seed=T, state=())
    if kind == "resets":
        x[3][:, [0, 3, T // 2, T - 1]] = -math.inf
    x = [t.requires_grad_(True) for t in x]
    y = [t.detach().double().requires_grad_(True) for t in x]
    got = A.gated_delta_scan(*x[:5], state=x[5], return_state=True)
    ref = O.delta_scan(*y[:5], state=y[5])
    g = torch.Generator().manual_seed(15)
    d = [torch.randn(t.shape, generator=g).to(t.dtype).to(DEV) for t in got]
    at = slice(1, 2) if kind == "only the state's" else slice(0, 2)
    # (with the state's alone q has no gradient)
    wrt = range(1, 6) if kind == "only the state's" else range(6)
    got = torch.autograd.grad(got[at], [x[i] for i in wrt], d[at])
    ref = torch.autograd.grad(ref[at], [y[i] for i in wrt], [t.double() for t in d[at]])
    for i, a, b in zip(wrt, got, ref):
        size = _dlogA_terms(y, d) if kind == "resets" and NAMES[i] == "dlogA" else None
        _near(NAMES[i], a, b, _noise(2 * (-(-T // 64) + 2) * (6 * -(-r // 32) + 32)), size)


def _terms(x, n):
    """x as the sum of its first n bf16 terms."""
    got, left = torch.zeros_like(x), x
    for _ in range(n):
        t = left.float().to(BF16).double()
        got, left = got + t, left - t
    return got


@pytest.mark.parametrize("nb,nbk,T,r,p,off", [s for s in SHAPES if s[5] is None])
def test_the_limit_sees_two_terms(nb, nbk, T, r, p, off):
    """On the CPU in 64 bits: states carried over runs of four chunks by transitions of one and
    of two bf16 terms are beyond the limit, of three far below it; so are their gradients."""
    g = torch.Generator().manual_seed(T + r)
    k = torch.nn.functional.normalize(torch.randn(T, r, generator=g).double(), dim=-1)
    v = torch.randn(T, p, generator=g).double()
    a = torch.exp(-1e-3 * torch.nn.functional.softplus(torch.randn(T, generator=g).double() - 2))
    b = 0.03 * torch.sigmoid(torch.randn(T, generator=g).double())
    S0, dS0 = 4 * torch.randn(r, p, generator=g).double(), torch.randn(r, p, generator=g).double()
    runs = []                                        # of each: S' = M S + E
    for t0 in range(0, T, 256):
        M, E = torch.eye(r, dtype=torch.float64), torch.zeros(r, p, dtype=torch.float64)
        for t in range(t0, min(t0 + 256, T)):
            M = a[t] * (M - b[t] * torch.outer(k[t], k[t] @ M))
            E = a[t] * (E - b[t] * torch.outer(k[t], k[t] @ E)) + b[t] * torch.outer(k[t], v[t])
        runs.append((M, E))
    for n in (1, 2, 3):
        S = ref = S0
        dS = dref = dS0
        for M, E in runs:
            S, ref = _terms(M, n) @ S + E, M @ ref + E
        for M, _ in reversed(runs):
            dS, dref = _terms(M, n).T @ dS, M.T @ dref
        for name, x, y in (("S", S, ref), ("dS0", dS, dref)):
            off = ((x - y).norm() / y.norm()).item() / _limit(name, -(-T // 64))
            assert off > 1.5 if n < 3 else off < 0.1, (name, n, off)
