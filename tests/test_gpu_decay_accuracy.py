"""How many bits the head decay's 16-bit results carry before they are rounded, in the mean over
the values.

A rounding to the nearest is off by at most 2^-24 of the value in fp32, by 2^-24 / sqrt(3) in
the root mean square, and roundings of sums are independent: a value that meets n of them on
its way is off by about sqrt(n / 3) 2^-24 of the root of its terms' squares.  ``_noise(n)`` is
twice that.  A result meets r or p products with the state, and T with the chunk's tokens.
"""
import math

import pytest
import torch

import oracle.decay_ref as O
from test_gpu_decay import BF16, DEV, FP16

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from smat_attention_amd import attention as A

BIG = 2.0 ** 14


def _noise(n):
    return 2 * math.sqrt(n / 3) * 2.0 ** -24


def _hold(name, got, ref, terms, n):
    """``got`` within the noise of ``ref`` and the rounding of its storing."""
    off = (got.double() - ref).norm().item()
    once = (ref.to(got.dtype).double() - ref).norm().item()
    lim = once + _noise(n) * terms.norm().item()
    assert off <= lim, (name, off, once, lim)


def _pairs(g, nb, r, p, dim):
    """Large fp32 values whose halves along ``dim`` are each other's negatives, nearly."""
    x = torch.randn(nb, r, p, generator=g)
    a, b = (BIG * x).chunk(2, dim)
    return torch.cat([a, x.chunk(2, dim)[1] - a], dim)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("r,p,T", [(64, 64, 64), (16, 40, 17), (128, 96, 50), (32, 128, 9)])
@pytest.mark.parametrize("group", [1, 2])
@pytest.mark.parametrize("name", ["o", "dq", "dk", "dv"])
def test_differences_of_the_state(dtype, r, p, T, group, name):
    """Results that are small differences of a large state's rows or columns (o and dq of the
    state entering, dv and dk of the gradient behind): both halves meet the same factors."""
    g = torch.Generator().manual_seed(r + p + T)
    nb, nbk = 8, 8 // group
    rn = lambda *s: torch.randn(*s, generator=g)
    x = {"q": rn(nbk, T, r), "k": rn(nbk, T, r), "v": rn(nb, T, p), "do": rn(nb, T, p)}
    by = {"o": "q", "dq": "do", "dk": "v", "dv": "k"}[name]
    x[by] = x[by][..., :x[by].shape[-1] // 2].repeat(1, 1, 2)
    q, k, v, dO = (x[n].to(dtype).to(DEV) for n in ("q", "k", "v", "do"))
    far = _pairs(g, nb, r, p, 1 if name in ("o", "dv") else 2).to(DEV)
    near = torch.randn(nb, r, p, generator=g).to(DEV)
    S, dS = (far, near) if name in ("o", "dq") else (near, far)
    logA = torch.tensor([-0.003, -0.02], device=DEV)
    a = [t.clone().requires_grad_(True) for t in (q, k, v)]
    b = [t.double().requires_grad_(True) for t in (q, k, v)]
    o, So = A.head_decay_scan(*a, logA, state=S, return_state=True)
    ro, rS = O.head_decay_scan(*b, logA, state=S)
    if name == "o":
        got, ref = o.detach(), ro.detach()
    else:
        i = ("dq", "dk", "dv").index(name)
        got, = torch.autograd.grad((o, So), a[i], (dO, dS))
        ref, = torch.autograd.grad((ro, rS), b[i], (dO.double(), dS.double()))
    # the terms' squares: of the large state alone, its decay at most one
    w = {"o": q, "dq": dO, "dk": v, "dv": k}[name].double().pow(2)
    if w.shape[0] < nb:
        w = w.repeat_interleave(group, 0)
    sq = far.double().pow(2)
    terms = (w @ (sq if name in ("o", "dv") else sq.transpose(1, 2).contiguous())).sqrt()
    if got.shape[0] < nb:                            # (summed over a key head's value heads)
        terms = terms.pow(2).view(nbk, group, *terms.shape[1:]).sum(1).sqrt()
    _hold(name, got, ref, terms, T + (r if name in ("o", "dv") else p))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("r,p,T", [(64, 64, 64), (128, 96, 50), (16, 40, 18)])
def test_differences_of_tokens(dtype, r, p, T):
    """Results that are small differences of a chunk's tokens: one key, and values that change
    sign from token to token, under a slow decay.  Every second output is near zero."""
    g = torch.Generator().manual_seed(r + p)
    nb = 8
    q, k = torch.randn(nb, T, r, generator=g), torch.randn(nb, 1, r, generator=g)
    w = torch.randn(nb, 1, p, generator=g)
    q, k, w = (t.to(dtype).to(DEV) for t in (q, k, w))
    sign = 1.0 - 2.0 * (torch.arange(T, device=DEV) % 2)[None, :, None]
    k, v = k.repeat(1, T, 1), w * sign.to(dtype)
    logA = torch.full((1,), -2.0 ** -14, device=DEV)
    o = A.head_decay_scan(q, k, v, logA)
    ro, _ = O.head_decay_scan(q, k, v, logA)
    t = torch.arange(1, T, 2, device=DEV)
    P = (q.double() * k.double()).sum(-1, keepdim=True)[:, t]
    terms = P.abs() * w.double().abs() * (t + 1.0).double().sqrt()[None, :, None]
    _hold("o", o[:, t], ro[:, t], terms, T + r)
