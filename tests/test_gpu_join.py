"""The end of a block (block_join) and its gradient against the oracle in 64 bits.

Tolerances.  A result is off by the rounding to its type and by fp32 arithmetic of fewer than
64 roundings of 2^-24 (forward: 8 squares a lane, 6 steps across lanes, 8 across waves, the
root, an exp, a dozen products), 128 (gradient), of the magnitudes that were added up: for h'
|h| + |s u|, for x that times pre / rms, and so on (``magnitudes``).  The columns' sums add a
rounding for every row of a group (at most rows) of the terms' magnitudes.  Relative roundings
end at fp32's smallest normal: below it a rounding is off by up to 2^-150 absolutely (sigmoid(-100)
= 3.8e-44 is 27 steps of 2^-149), and what it is multiplied by later here (the next gradients, the
norm's factor) stays below 8, so each allows 2^-147.
"""
import pytest
import torch

import oracle.join_ref as O

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from smat_attention_amd import attention as A

DEV = "cuda:0"
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24


def check(name, got, ref, big, roundings):
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    if not ref.numel():
        return
    assert torch.isfinite(got).all(), name
    info = torch.finfo(got.dtype)
    lim = info.eps / 2 * ref.abs() + 1.01 * roundings * U * big + info.smallest_normal * info.eps
    lim = lim + roundings * 2.0 ** -147
    worst = ((got.double() - ref).abs() - lim).max().item()
    assert worst <= 0, f"{name}: {worst:.3e} beyond the bound"


def inputs(rows, D, dtype, stream, gate, post, vector, pre, seed=0, wtype=FP32):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)
    f, h, z = (0.5 * rn(rows, D)).to(dtype), (2 * rn(rows, D)).to(stream), rn(rows, D).to(dtype)
    w1, s, w2 = ((c + 0.1 * rn(D)).to(wtype) for c in (1.0, 0.25, 1.0))
    t = [f, h, w1 if post else None, z if gate else None, s if vector else None, w2 if pre else None]
    return [None if x is None else x.to(DEV) for x in t]


def magnitudes(f, h, post, z, kind, s, pre, eps, mask, dh, dx):
    """The sums over magnitudes of h', x, df, dh, dz, dpost, ds, dpre."""
    f, h, dh = f.double(), h.double(), dh.double().abs()
    one = lambda t: (t.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    r1 = one(f) if post is not None else torch.ones_like(f[:, :1])
    w1 = post.double().abs() if post is not None else 1.0
    y = f.abs() * r1 * w1
    a, slope = torch.ones_like(f), torch.zeros_like(f)
    if z is not None:
        z = z.double()
        sg = torch.sigmoid(z)
        a, slope = {"linear": (z.abs(), torch.ones_like(z)), "sigmoid": (sg, sg * (1 - sg)),
                    "silu": (z.abs() * sg, sg * (1 + z.abs() * (1 - sg)))}[kind]
    m = mask.double() if mask is not None else 1.0
    s = s.double().abs() if torch.is_tensor(s) else abs(s)
    u = m * a * y
    h2 = h.abs() + s * u
    hh = O.block_join(f, h, post, z, kind, s, None, eps, mask)[0]
    r2 = one(hh)
    got = {"h": h2}
    g = dh
    if pre is not None:
        got["x"] = pre.double().abs() * r2 * h2
        t = pre.double().abs() * dx.double().abs()
        g = dh + r2 * t + h2 * r2 ** 3 * (t * h2).mean(-1, keepdim=True)
        got["dpre"] = (dx.double().abs() * h2 * r2).sum(0)
    dy = g * m * s * a
    v = w1 * dy
    got["df"] = r1 * v + f.abs() * r1 ** 3 * (v * f.abs()).mean(-1, keepdim=True) \
        if post is not None else dy
    got["dh"], got["dz"] = g, g * m * s * y * slope
    got["dpost"], got["ds"] = (dy * f.abs() * r1).sum(0), (g * u).sum(0)
    return got


CASES = [
    # rows, D, gate, post, vector, pre, dropout
    (1, 8, "sigmoid", True, True, True, 0.0),
    (3, 9, "silu", True, True, True, 0.3),
    (5, 64, None, True, False, True, 0.0),
    (70, 65, "linear", False, True, True, 0.5),
    (33, 511, "sigmoid", True, True, False, 0.1),
    (17, 512, "silu", False, False, True, 0.0),
    (9, 513, "sigmoid", True, True, True, 0.1),
    (40, 768, "sigmoid", True, True, True, 0.1),
    (6, 1531, "silu", True, False, True, 0.25),
    (4, 4096, None, False, False, False, 0.2),
    (3, 4097, "sigmoid", True, True, True, 0.1),
    (2, 8191, "linear", True, True, True, 0.0),
    (2, 8192, "silu", True, True, True, 0.1),
    (5000, 40, "sigmoid", True, True, True, 0.1),
    # more rows than workgroups at a time, sixteen waves a row
    (515, 4100, "sigmoid", True, True, True, 0.1),
    (600, 8192, None, True, False, True, 0.0),
]


@pytest.mark.parametrize("dtype,stream", [(BF16, FP32), (BF16, BF16), (FP16, FP32), (FP16, FP16),
                                          (FP32, FP32)])
@pytest.mark.parametrize("rows,D,kind,post,vector,pre,p", CASES)
def test_join_and_gradients(dtype, stream, rows, D, kind, post, vector, pre, p):
    f, h, w1, z, s, w2 = x = inputs(rows, D, dtype, stream, kind, post, vector, pre, seed=D)
    scale = s if vector else 0.3
    seed, salt = (torch.tensor([2 ** 61 + 12345 * D], device=DEV), 7) if p else (None, 0)
    mask = None
    if p:
        keep = O.kept(range(min(rows, 64)), D, p, int(seed), salt)
        if rows > 64:                                # the rest of the mask from the kernel itself
            one = torch.ones(rows, D, device=DEV)
            got = A.block_join(one, 0 * one, dropout=p, seed=seed, salt=salt)[0] != 0
            assert torch.equal(got[:64].cpu(), keep)
            keep = got
        mask = keep.double().to(DEV) / (1 - p)
    kw = dict(gate_kind=kind or "sigmoid", dropout=p, seed=seed, salt=salt)
    h2, x2 = A.block_join(f, h, post_weight=w1, gate=z, scale=scale, pre_weight=w2, **kw)
    assert h2.dtype == stream and (x2 is None) == (not pre) and (x2 is None or x2.dtype == dtype)
    g = torch.Generator().manual_seed(1)
    dh = torch.randn(rows, D, generator=g).to(stream).to(DEV)
    dx = torch.randn(rows, D, generator=g).to(dtype).to(DEV)
    big = magnitudes(f, h, w1, z, kind, scale, w2, 1e-6, mask, dh, dx)
    leaves = [None if t is None else t.double().requires_grad_(True) for t in x]
    rf, rh, rw1, rz, rs, rw2 = leaves
    r = O.block_join(rf, rh, rw1, rz, kind, rs if vector else scale, rw2, 1e-6, mask)
    check("h", h2, r[0].detach(), big["h"], 64)
    if pre:
        check("x", x2, r[1].detach(), big["x"], 64)
    mine = [None if t is None else t.clone().requires_grad_(True) for t in x]
    o = A.block_join(mine[0], mine[1], post_weight=mine[2], gate=mine[3],
                     scale=mine[4] if vector else scale, pre_weight=mine[5], **kw)
    assert torch.equal(o[0].detach(), h2) and (not pre or torch.equal(o[1].detach(), x2))
    ups = (dh, dx) if pre else (dh,)
    wrt = [i for i, t in enumerate(x) if t is not None]
    got = torch.autograd.grad(o[:len(ups)], [mine[i] for i in wrt], ups)
    ref = torch.autograd.grad(r[:len(ups)], [leaves[i] for i in wrt], [t.double() for t in ups])
    for i, a, b in zip(wrt, got, ref):
        name = ("df", "dh", "dpost", "dz", "ds", "dpre")[i]
        assert a.dtype == x[i].dtype
        check(name, a, b, big[name], 128 + (rows if a.dim() == 1 else 0))


def test_only_one_result_has_a_gradient():
    x = inputs(20, 100, FP32, FP32, "silu", True, True, True)
    for k in (0, 1):
        a = [t.clone().requires_grad_(True) for t in x]
        b = [t.double().requires_grad_(True) for t in x]
        o = A.block_join(a[0], a[1], post_weight=a[2], gate=a[3], gate_kind="silu", scale=a[4],
                         pre_weight=a[5])
        r = O.block_join(b[0], b[1], b[2], b[3], "silu", b[4], b[5])
        d = torch.randn(20, 100, generator=torch.Generator().manual_seed(3)).to(DEV)
        got = torch.autograd.grad(o[k], a, d, allow_unused=True)
        ref = torch.autograd.grad(r[k], b, d.double(), allow_unused=True)
        zero = torch.zeros_like(d)
        big = magnitudes(*x[:4], "silu", *x[4:], 1e-6, None, d if k == 0 else zero,
                         d if k == 1 else zero)
        for name, s, t in zip(("df", "dh", "dpost", "dz", "ds", "dpre"), got, ref):
            if t is None:
                assert not s.any()                   # x's weight, when only h' has a gradient
            else:
                check(name, s, t, big[name], 148)


@pytest.mark.parametrize("wtype", [BF16, FP16])
def test_weights_of_16_bits(wtype):
    x = inputs(12, 96, BF16, FP32, "sigmoid", True, True, True, wtype=wtype)
    y = [t if i < 2 or i == 3 else t.float() for i, t in enumerate(x)]

    def run(x):
        x = [t.clone().requires_grad_(True) for t in x]
        o = A.block_join(x[0], x[1], post_weight=x[2], gate=x[3], scale=x[4], pre_weight=x[5])
        return list(o), torch.autograd.grad(o[0].sum() + o[1].float().sum(), x)
    (a, ga), (b, gb) = run(x), run(y)
    assert all(torch.equal(s, t) for s, t in zip(a, b))
    assert all(torch.equal(s, t.to(s.dtype)) for s, t in zip(ga, gb))


def test_generator_and_rate():
    """The mask is the generator's; other salts, seeds and rows have others; the rate is p's, to
    five standard deviations of as many draws."""
    rows, D, p = 300, 1001, 0.2
    one = torch.ones(rows, D, device=DEV)

    def mask(seed, salt=0, t=one):
        return A.block_join(t, torch.zeros_like(t), dropout=p, salt=salt,
                            seed=torch.tensor([seed], device=DEV))[0]
    m = mask(-5)
    assert torch.equal((m != 0)[:20].cpu(), O.kept(range(20), D, p, -5))
    assert ((m == 0) | (m == torch.tensor(1 / (1 - p), device=DEV, dtype=FP32))).all()
    dropped = (m == 0).double().mean().item()
    assert abs(dropped - p) <= 5 * (p * (1 - p) / (rows * D)) ** 0.5
    for other in (mask(-4), mask(-5, 1), mask(-5 + 2 ** 32)):
        same = ((other == 0) == (m == 0)).double().mean().item()
        q = p * p + (1 - p) * (1 - p)
        assert abs(same - q) <= 5 * (q * (1 - q) / (rows * D)) ** 0.5
    # a row's places do not depend on how many rows there are
    assert torch.equal(mask(-5, t=one[:7]), m[:7])


def test_layouts_and_shapes():
    """Leading axes, rows apart, transposed columns, an expanded gate: what contiguous copies
    give."""
    B, T, D = 3, 7, 72
    f, h, w1, z, s, w2 = inputs(B * T, D, BF16, FP32, "sigmoid", True, True, True)
    want = A.block_join(f, h, post_weight=w1, gate=z, scale=s, pre_weight=w2)
    buf = torch.full((B * T, D + 5), float("nan"), device=DEV, dtype=BF16)
    fs = buf[:, 3:3 + D]
    fs.copy_(f)
    ht = h.t().contiguous().t()
    got = A.block_join(fs.unflatten(0, (B, T)), ht.view(B, T, D), post_weight=w1,
                       gate=z.view(B, T, D), scale=torch.stack([s, s], 1)[:, 0], pre_weight=w2)
    assert got[0].shape == (B, T, D)
    assert all(torch.equal(a.reshape(-1, D), b) for a, b in zip(got, want))
    z1 = z[:B, None].clone().requires_grad_(True)
    o = A.block_join(f.view(B, T, D), h.view(B, T, D), gate=z1.expand(B, T, D))[0]
    z2 = z1.detach().repeat(1, T, 1).requires_grad_(True)
    o2 = A.block_join(f.view(B, T, D), h.view(B, T, D), gate=z2)[0]
    assert torch.equal(o, o2)
    a, = torch.autograd.grad(o.sum(), z1)
    b, = torch.autograd.grad(o2.sum(), z2)
    # the expanded gate's gradient: T rounded values and their sum's rounding
    lim = (T + 2) * 2.0 ** -9 * b.double().abs().sum(1, keepdim=True)
    assert ((a.double() - b.double().sum(1, keepdim=True)).abs() <= lim).all()
    row = A.block_join(f[0], h[0], post_weight=w1, gate=z[0], scale=s, pre_weight=w2)
    assert all(torch.equal(a, b[0]) for a, b in zip(row, want))


@pytest.mark.parametrize("rows", [0, 1])
def test_no_rows_and_one(rows):
    x = [t.requires_grad_(True) for t in inputs(rows, 24, FP32, FP32, "sigmoid", True, True, True)]
    o = A.block_join(x[0], x[1], post_weight=x[2], gate=x[3], scale=x[4], pre_weight=x[5])
    got = torch.autograd.grad(o[0].sum() + o[1].sum(), x)
    assert [g.shape for g in got] == [t.shape for t in x]
    if not rows:
        assert all(not g.any() for g in got)


def test_zero_rows_and_far_gates():
    """Rows of zeros (rms is eps's), gates far into both ends, values at the type's ends."""
    f, h, w1, z, s, w2 = inputs(8, 64, FP32, FP32, "sigmoid", True, True, True)
    f[0], h[0] = 0, 0
    f[1] = 1e-30
    h[2] = 1e15
    z[3], z[4] = 100.0, -100.0
    for kind in ("sigmoid", "silu"):
        x = [t.detach().clone().requires_grad_(True) for t in (f, h, w1, z, s, w2)]
        y = [t.detach().double().requires_grad_(True) for t in x]
        o = A.block_join(x[0], x[1], post_weight=x[2], gate=x[3], gate_kind=kind, scale=x[4],
                         pre_weight=x[5])
        r = O.block_join(y[0], y[1], y[2], y[3], kind, y[4], y[5])
        g = torch.Generator().manual_seed(1)
        d = [torch.randn(8, 64, generator=g).to(DEV) for _ in range(2)]
        big = magnitudes(*[t.detach() for t in x[:4]], kind, *[t.detach() for t in x[4:]], 1e-6,
                         None, *d)
        check("h", o[0].detach(), r[0].detach(), big["h"], 64)
        check("x", o[1].detach(), r[1].detach(), big["x"], 64)
        got = torch.autograd.grad(o, x, d)
        ref = torch.autograd.grad(r, y, [t.double() for t in d])
        for name, a, b in zip(("df", "dh", "dpost", "dz", "ds", "dpre"), got, ref):
            check(name, a, b, big[name], 136)


def test_rates_at_the_ends():
    """A rate whose threshold is the generator's last word, and one below half a step, which
    keeps everything: both within the documented range."""
    f, h = torch.ones(64, 512, device=DEV), torch.zeros(64, 512, device=DEV)
    seed = torch.tensor([5], device=DEV)
    y, _ = A.block_join(f, h, dropout=1 - 2.0 ** -40, seed=seed)
    assert ((y == 0) | (y == 2.0 ** 40)).all()
    y, _ = A.block_join(f, h, dropout=2.0 ** -40, seed=seed)
    assert torch.equal(y, f)


def test_seed_steps_before_the_backward():
    """The gradient belongs to the forward's mask, whatever the seed holds by then."""
    f, h = (torch.randn(9, 50, device=DEV) for _ in range(2))
    f.requires_grad_(True)
    seed = torch.tensor([11], device=DEV)
    o = A.block_join(f, h, dropout=0.4, seed=seed)[0]
    seed += 1
    g, = torch.autograd.grad(o.sum(), f)
    assert torch.equal(g != 0, (o - h) != 0)
