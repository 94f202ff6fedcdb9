"""What dropout drops counts for nothing, whatever it holds: results and gradients are the bits
of a call with zeros there."""
import math

import pytest
import torch

import oracle.join_ref as O
from test_gpu_join import BF16, DEV, FP16, FP32, inputs

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from smat_attention_amd import attention as A


def _run(x, kind, dh, dx, **kw):
    x = [None if t is None else t.clone().requires_grad_(True) for t in x]
    o = A.block_join(x[0], x[1], post_weight=x[2], gate=x[3], gate_kind=kind, scale=x[4],
                     pre_weight=x[5], **kw)
    o, ups = ([t for t in o if t is not None], [dh] if x[5] is None else [dh, dx])
    got = torch.autograd.grad(o, [t for t in x if t is not None], ups)
    return [t.detach() for t in o] + list(got)


@pytest.mark.parametrize("dtype,stream", [(BF16, FP32), (BF16, BF16), (FP16, FP32), (FP32, FP32)])
@pytest.mark.parametrize("rows,D", [(9, 96), (5, 1531), (4, 4100)])
@pytest.mark.parametrize("kind", [None, "linear", "sigmoid", "silu"])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_dropped_places_that_are_not_finite(dtype, stream, rows, D, kind, bad):
    """f without a norm after the block, the gate, and a gradient arriving at h' alone."""
    p, seed = 0.3, torch.tensor([77 + D], device=DEV)
    kw = dict(dropout=p, seed=seed, salt=3)
    away = ~O.kept(range(rows), D, p, int(seed), 3).to(DEV)
    away[:, 8:] &= torch.rand(rows, D - 8, generator=torch.Generator().manual_seed(2)).to(DEV) < 0.2
    assert away.any()
    g = torch.Generator().manual_seed(1)
    dh = torch.randn(rows, D, generator=g).to(stream).to(DEV)
    dx = torch.randn(rows, D, generator=g).to(dtype).to(DEV)
    f, h, w1, z, s, w2 = inputs(rows, D, dtype, stream, kind, True, True, True, seed=D)
    zero = lambda t: t.masked_fill(away, 0)
    spoilt = lambda t: t.masked_fill(away, bad)
    want = _run((zero(f), h, None, z, s, w2), kind or "sigmoid", dh, dx, **kw)
    got = _run((spoilt(f), h, None, z, s, w2), kind or "sigmoid", dh, dx, **kw)
    for i, (a, b) in enumerate(zip(got, want)):
        assert torch.isfinite(a).all(), i
        # (dz at a dropped place is a zero of either sign)
        assert torch.equal(a + 0, b + 0), i
    if kind:
        want = _run((f, h, w1, zero(z), s, w2), kind, dh, dx, **kw)
        got = _run((f, h, w1, spoilt(z), s, w2), kind, dh, dx, **kw)
        for i, (a, b) in enumerate(zip(got, want)):
            assert torch.isfinite(a).all(), i
            assert torch.equal(a + 0, b + 0), i
    # the gradient of h' alone: f's and the gate's do not see it where they were dropped
    def back(dh):
        a, c = f.clone().requires_grad_(True), None if z is None else z.clone().requires_grad_(True)
        o, _ = A.block_join(a, h, gate=c, gate_kind=kind or "sigmoid", scale=0.5, **kw)
        return torch.autograd.grad(o, [a] if c is None else [a, c], dh)
    for a, b in zip(back(spoilt(dh)), back(zero(dh))):
        assert torch.isfinite(a).all() and torch.equal(a + 0, b + 0)
