"""The block's end at gates that are infinite or at their type's ends, against the oracle in 64
bits, with the tolerances of test_gpu_join."""
import math

import pytest
import torch

import oracle.join_ref as O
from test_gpu_join import BF16, DEV, FP16, FP32, check, inputs, magnitudes

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from smat_attention_amd import attention as A

NAMES = ("df", "dh", "dpost", "dz", "ds", "dpre")


@pytest.mark.parametrize("dtype,stream", [(BF16, FP32), (BF16, BF16), (FP16, FP32), (FP32, FP32)])
@pytest.mark.parametrize("D", [64, 1531, 4100])
@pytest.mark.parametrize("kind", ["sigmoid", "silu"])
@pytest.mark.parametrize("post", [True, False])
def test_gates_at_the_ends(dtype, stream, D, kind, post):
    """Closed gates give zero and open ones one (silu: z): single places of a row, whole rows.
    Under a silu gate the large places have a small f, so that rows stay within fp32's squares;
    the oracle takes -2^100 for -inf there (its own quotient is inf / inf)."""
    f, h, w1, z, s, w2 = inputs(6, D, dtype, stream, kind, post, True, True, seed=D)
    ends = [v for v in (200.0, 65504.0, 2.3e38, 2.4e38, 3.3e38) if v <= torch.finfo(dtype).max]
    if kind == "silu":
        f[:, :8] = 2.0 ** -14 if dtype == FP16 else 1e-30
        s[:8] = 2.0 ** -6                            # (and gradients within fp32's range)
    low = [-v for v in ends] + [-math.inf]
    high = ends + ([math.inf] if kind == "sigmoid" else [])
    for i, v in enumerate(high):
        z[i % 4, i] = v
    for i, v in enumerate(low):
        z[(i + 1) % 4, 9 + i] = v
    z[4] = -math.inf
    z[5, 1::2] = -torch.finfo(dtype).max
    x = [None if t is None else t.clone().requires_grad_(True) for t in (f, h, w1, z, s, w2)]
    y = [None if t is None else t.double() for t in (f, h, w1, z, s, w2)]
    if kind == "silu":
        y[3] = y[3].clamp(min=-2.0 ** 100)
    y = [None if t is None else t.requires_grad_(True) for t in y]
    o = A.block_join(x[0], x[1], post_weight=x[2], gate=x[3], gate_kind=kind, scale=x[4],
                     pre_weight=x[5])
    r = O.block_join(*y[:4], kind, *y[4:])
    g = torch.Generator().manual_seed(1)
    dh = torch.randn(6, D, generator=g).to(stream).to(DEV)
    dx = torch.randn(6, D, generator=g).to(dtype).to(DEV)
    m = [None if t is None else t.detach() for t in y]
    big = magnitudes(*m[:4], kind, *m[4:], 1e-6, None, dh, dx)
    check("h", o[0].detach(), r[0].detach(), big["h"], 64)
    check("x", o[1].detach(), r[1].detach(), big["x"], 64)
    wrt = [i for i, t in enumerate(x) if t is not None]
    got = torch.autograd.grad(o, [x[i] for i in wrt], (dh, dx))
    ref = torch.autograd.grad(r, [y[i] for i in wrt], (dh.double(), dx.double()))
    for i, a, b in zip(wrt, got, ref):
        check(NAMES[i], a, b, big[NAMES[i]], 134)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_an_infinite_silu_gate(dtype):
    """silu(inf) is inf with slope one; what is not a number stays that, under either gate."""
    f = torch.ones(1, 64, device=DEV, dtype=dtype)
    f[0, 3] = -2.0
    z, h = torch.ones_like(f), torch.zeros(1, 64, device=DEV)
    z[0, 2:4] = math.inf
    f, z, h = (t.requires_grad_(True) for t in (f, z, h))
    o, _ = A.block_join(f, h, gate=z, gate_kind="silu")
    df, dz, dh = torch.autograd.grad(o, (f, z, h), torch.ones_like(o))
    assert o[0, 2] == math.inf and o[0, 3] == -math.inf
    assert torch.isfinite(torch.cat([o[:, :2], o[:, 4:]], 1)).all()
    assert dz[0, 2] == 1 and dz[0, 3] == -2 and (df[0, 2:4] == math.inf).all() and (dh == 1).all()
    z = z.detach().clone()
    z[0, 5] = math.nan
    for kind in ("sigmoid", "silu"):
        bad = torch.isnan(A.block_join(f.detach(), h.detach(), gate=z, gate_kind=kind)[0])
        assert bad[0, 5] and bad.sum() == 1
