"""How many bits the gated delta rule's results carry, in the mean over the values.

A rounding to the nearest is off by at most 2^-24 of the value in fp32, by 2^-24 / sqrt(3) in
the root mean square, and roundings of sums are independent: a value that meets n of them on
its way is off by about sqrt(n / 3) 2^-24 of the largest magnitude involved.  ``_noise(n)`` is
twice that.
"""
import math

import pytest
import torch

import oracle.delta_ref as O
from test_gpu_delta import BF16, DEV, FP16, FP32

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from smat_attention_amd import attention as A


def _noise(n):
    return 2 * math.sqrt(n / 3) * 2.0 ** -24


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("r,p,T", [(64, 64, 64), (16, 40, 17), (64, 200, 50)])
def test_outputs_are_rounded_once(dtype, r, p, T):
    """Outputs that are small differences of large sums.  With unit keys, beta = 1, no decay and
    q = k the output is v whatever the state held; here that is 2^14 times v, and what is
    rounded before the sum shows.  (Keys of +-1/sqrt(r) are exact in every type.)  A value
    meets r + T products on the way to U, and r + T more."""
    g = torch.Generator().manual_seed(r + p)
    nb, big = 8, 2.0 ** 14
    k = (torch.randint(0, 2, (nb, T, r), generator=g) * 2 - 1) * r ** -0.5
    v = torch.randn(nb, T, p, generator=g)
    k, v = k.to(dtype).to(DEV), v.to(dtype).to(DEV)
    S = (big * torch.randn(nb, r, p, generator=g)).to(DEV)
    logA, beta = torch.zeros(nb, T, device=DEV), torch.ones(nb, T, device=DEV)
    o = A.gated_delta_scan(k, k, v, logA, beta, state=S)
    ro, _ = O.delta_scan(k, k, v, logA, beta, state=S)
    read = k.double() @ S.double()                   # the large magnitudes
    off = (o.double() - ro).norm().item()
    once = (ro.to(dtype).double() - ro).norm().item()
    assert off <= once + _noise(2 * (r + T)) * read.norm().item(), (off, once, read.norm().item())
