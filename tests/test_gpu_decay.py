"""Linear attention with a decay for each head (head_decay_scan, its gradient, head_decay_step,
HeadDecayDecoder) against the token-by-token oracle in 64 bits.

Tolerances.  A result stored in type t is off by its rounding, eps(t) / 2 of its value, and by
the arithmetic before it: fp32 sums of products whose operands carry 24 bits.  Every value is a
sum of terms; ``big`` is the same sum over the terms' magnitudes (the oracle on absolute values),
and each term has passed at most r + p + 128 roundings of 2^-24 of what it was added to in its own
chunk, and 72 (64 tokens, the decay, the splits) in each of the chunks the state took it through.
(The products of an output of 16 bits take the state and P to 17 bits, 2^-17 = 128 * 2^-24 of each
term: as much as the count has beyond the r + p + 72 roundings of a chunk's own sums.)
"""
import math

import pytest
import torch

import oracle.decay_ref as O

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from smat_attention_amd import attention as A

DEV = "cuda:0"
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def check(name, got, ref, big, chunks, r, p):
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    if not ref.numel():
        return
    assert torch.isfinite(got).all(), name
    info = torch.finfo(got.dtype)
    tol = (r + p + 128 + 72 * chunks) * 2.0 ** -24 * big
    lim = info.eps / 2 * ref.abs() + (1 + info.eps) * tol + info.smallest_normal * info.eps
    worst = ((got.double() - ref).abs() - lim).max().item()
    assert worst <= 0, f"{name}: {worst:.3e} beyond the bound"


def inputs(nb, nbk, T, r, p, heads, dtype, seed=0, lead=None, slow=1 / 64):
    """Normal rows; decays from ``slow`` to 1/2 a token; a state where ``lead`` says its leading
    axes."""
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)
    q, k, v = (x.to(dtype) for x in (rn(nbk, T, r), rn(nbk, T, r), rn(nb, T, p)))
    logA = -slow * torch.exp(torch.rand(heads, generator=g) * math.log(0.5 / slow))
    S = None if lead is None else rn(*lead, nb, r, p)
    return [None if t is None else t.to(DEV) for t in (q, k, v, logA, S)]


def oracle(q, k, v, logA, S, scale, off, dO=None, dS=None):
    """``(o, S, grads)`` and the same over magnitudes."""
    both = []
    for mag in (False, True):
        f = (lambda t: t.double().abs()) if mag else (lambda t: t.double())
        x = [f(q), f(k), f(v), logA.double()] + ([] if S is None else [f(S)])
        x = [t.clone().requires_grad_(True) for t in x]
        o, So = O.head_decay_scan(*x[:4], scale=abs(scale) if mag else scale,
                                  state=x[4] if len(x) > 4 else None, offsets=off)
        grads = None
        if dO is not None:
            grads = torch.autograd.grad((o, So), x, (f(dO), f(dS)))
        both.append((o.detach(), So.detach(), grads))
    return both


def chunks_of(T, off):
    return max(sum(-(-(b - a) // 64) for a, b in zip(off or [0], (off or [0, T])[1:])), 1)


SHAPES = [
    # nb, nbk, T, r, p, heads, offsets, state
    (3, 3, 1, 64, 64, 3, None, True),
    (4, 2, 7, 40, 50, 2, None, False),
    (300, 150, 16, 128, 128, 6, None, True),
    (2, 2, 17, 33, 9, 1, None, True),
    (2, 2, 63, 128, 128, 2, None, False),
    (2, 1, 64, 64, 64, 2, None, True),
    (4, 2, 65, 96, 80, 4, None, True),
    (1, 1, 200, 17, 33, 1, None, False),
    (2, 2, 130, 1, 1, 2, None, True),
    (2, 2, 70, 3, 65, 2, None, True),
    (3, 1, 129, 128, 24, 3, None, True),
    (2, 2, 129, 31, 127, 2, None, False),
    (4, 1, 150, 33, 47, 2, [0, 1, 1, 64, 129, 150], True),
    (2, 2, 140, 64, 64, 2, [0, 70, 140], False),
    (1, 1, 70, 12, 100, 1, [0, 0, 70], True),
]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("nb,nbk,T,r,p,heads,off,st", SHAPES)
def test_scan_and_gradients(dtype, nb, nbk, T, r, p, heads, off, st):
    lead = None if not st else () if off is None else (len(off) - 1,)
    q, k, v, logA, S = inputs(nb, nbk, T, r, p, heads, dtype, seed=T + r, lead=lead)
    scale, ch = r ** -0.5, chunks_of(T, off)
    seg = None if off is None else A.Segments(off, DEV)
    o, So = A.head_decay_scan(q, k, v, logA, scale=scale, state=S, segments=seg,
                              return_state=True)
    g = torch.Generator().manual_seed(9)
    dO = torch.randn(o.shape, generator=g).to(dtype).to(DEV)
    dS = torch.randn(So.shape, generator=g).to(DEV)
    (ro, rS, rg), (bo, bS, bg) = oracle(q, k, v, logA, S, scale, off, dO, dS)
    assert o.dtype == dtype and So.dtype == FP32
    check("o", o, ro, bo, ch, r, p)
    check("S", So, rS, bS, ch, r, p)
    x = [t.clone().requires_grad_(True) for t in (q, k, v, logA)] + (
        [] if S is None else [S.clone().requires_grad_(True)])
    o2, S2 = A.head_decay_scan(*x[:4], scale=scale, state=x[4] if st else None, segments=seg,
                               return_state=True)
    assert torch.equal(o2.detach(), o) and torch.equal(S2.detach(), So)
    got = torch.autograd.grad((o2, S2), x, (dO, dS))
    for name, a, b, big, t in zip(("dq", "dk", "dv", "dlogA", "dS0"), got, rg, bg, x):
        assert a.dtype == t.dtype
        check(name, a, b, big, ch, r, p)
    # without the decays' gradient
    y = [t.detach().requires_grad_(i != 3) for i, t in enumerate(x)]
    o3, S3 = A.head_decay_scan(*y[:4], scale=scale, state=y[4] if st else None, segments=seg,
                               return_state=True)
    rest = torch.autograd.grad((o3, S3), y[:3] + y[4:], (dO, dS))
    for a, b in zip(rest, got[:3] + got[4:]):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_fp32_results_have_fp32_accuracy(dtype):
    """The state and the decays' gradient are fp32 whatever the inputs' type.  Each value is off
    by about sqrt(r + p + 128) independent roundings of 2^-24; twice that in the mean."""
    nb, T, r, p = 8, 640, 64, 64
    q, k, v, logA, S = inputs(nb, nb, T, r, p, 8, dtype, seed=21, lead=())
    dO = torch.randn(nb, T, p, generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
    x = [t.requires_grad_(True) for t in (q, k, v, logA, S)]
    o, So = A.head_decay_scan(*x[:4], state=S, return_state=True)
    y = [t.detach().double().requires_grad_(True) for t in x]
    ro, rS = O.head_decay_scan(*y[:4], state=y[4])
    got = (So, *torch.autograd.grad(o, x[3:], dO))
    ref = (rS, *torch.autograd.grad(ro, y[3:], dO.double()))
    for name, a, b in zip(("S", "dlogA", "dS0"), got, ref):
        off = ((a.detach().double() - b.detach()).norm() / b.detach().norm()).item()
        assert off <= 2 * math.sqrt(r + p + 128) * 2.0 ** -24, (name, off)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("nb,nbk,T,r,p,off,st", [
    (2, 2, 64 * 40 + 5, 64, 64, None, True),
    (2, 1, 64 * 33, 128, 48, None, False),
    (1, 1, 64 * 70 + 1, 40, 99, [0, 64 * 50 + 3, 64 * 50 + 3, 64 * 70 + 1], True),
    (1, 1, 64 * 40, 41, 99, None, True),
])
def test_split_along_the_sequence(dtype, nb, nbk, T, r, p, off, st):
    """Few long sequences are cut into runs joined through their decays."""
    lead = None if not st else () if off is None else (len(off) - 1,)
    q, k, v, logA, S = inputs(nb, nbk, T, r, p, nb, dtype, seed=3, lead=lead, slow=2.0 ** -12)
    seg = None if off is None else A.Segments(off, DEV)
    from smat_attention_amd.kernels.hip_decay import _Plan
    assert _Plan("test", q, v, nb, seg).nruns > (len(seg) if seg else 1)
    g = torch.Generator().manual_seed(1)
    dO = torch.randn(nb, T, p, generator=g).to(dtype).to(DEV)
    x = [t.requires_grad_(True) for t in (q, k, v, logA)] + (
        [] if S is None else [S.requires_grad_(True)])
    o, So = A.head_decay_scan(*x[:4], state=S, segments=seg, return_state=True)
    dS = torch.randn(So.shape, generator=g).to(DEV)
    got = torch.autograd.grad((o, So), x, (dO, dS))
    d = [None if t is None else t.detach() for t in (q, k, v, logA, S)]
    (ro, rS, rg), (bo, bS, bg) = oracle(*d, 1.0, off, dO, dS)
    ch = chunks_of(T, off)
    check("o", o.detach(), ro, bo, ch, r, p)
    check("S", So.detach(), rS, bS, ch, r, p)
    for name, a, b, big in zip(("dq", "dk", "dv", "dlogA", "dS0"), got, rg, bg):
        check(name, a, b, big, ch, r, p)


def test_a_state_at_any_address():
    """A state that does not begin at 16 bytes enters the runs as another does: every element goes
    the same way."""
    q, k, v, logA, S = inputs(2, 2, 64 * 40, 64, 64, 2, BF16, seed=23, lead=(), slow=2.0 ** -12)
    off = torch.empty(S.numel() + 1, device=DEV)[1:].view_as(S).copy_(S)
    assert off.data_ptr() % 16
    a, b = (A.head_decay_scan(q, k, v, logA, state=s, return_state=True) for s in (S, off))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("la", [0.0, -1e-7, -30.0, -200.0, -math.inf])
@pytest.mark.parametrize("T", [40, 64 * 30 + 7])
def test_extreme_decays(la, T):
    """No decay at all, one that fp32 cannot tell from none in a token, decays whose powers
    underflow within a chunk, and a state that is the last token's alone."""
    nb, r, p = 2, 32, 40
    q, k, v, _, S = inputs(nb, nb, T, r, p, 2, FP32, seed=5, lead=())
    logA = torch.tensor([la, -0.25], device=DEV)
    x = [t.requires_grad_(True) for t in (q, k, v, S)]
    o, So = A.head_decay_scan(*x[:3], logA, state=S, return_state=True)
    g = torch.Generator().manual_seed(2)
    dO, dS = torch.randn(o.shape, generator=g).to(DEV), torch.randn(S.shape, generator=g).to(DEV)
    got = torch.autograd.grad((o, So), x, (dO, dS))
    y = [t.detach() for t in (q, k, v)]
    (ro, rS, rg), (bo, bS, bg) = oracle(*y, logA, S.detach(), 1.0, None, dO, dS)
    ch = chunks_of(T, None)
    check("o", o.detach(), ro, bo, ch, r, p)
    check("S", So.detach(), rS, bS, ch, r, p)
    for name, a, b, big in zip(("dq", "dk", "dv", "dS0"), got, rg[:3] + rg[4:], bg[:3] + bg[4:]):
        check(name, a, b, big, ch, r, p)


def test_gradient_against_differences():
    """The directional derivative of <o, dO> + <S, dS>: central differences of the oracle in 64
    bits (truncation h^2, cancellation 2^-52 / h: both far below the fp32 gradients')."""
    nb, T, r, p = 4, 100, 24, 16
    q, k, v, logA, S = inputs(nb, nb, T, r, p, 2, FP32, seed=8, lead=())
    x = [t.requires_grad_(True) for t in (q, k, v, logA, S)]
    g = torch.Generator().manual_seed(2)
    dO, dS = torch.randn(nb, T, p, generator=g).to(DEV), torch.randn(nb, r, p, generator=g).to(DEV)
    o, So = A.head_decay_scan(*x[:4], state=x[4], return_state=True)
    grads = torch.autograd.grad((o, So), x, (dO, dS))
    _, (_, _, bg) = oracle(*[t.detach() for t in x], 1.0, None, dO, dS)
    h = 1e-5
    for i, t in enumerate(x):
        d = torch.randn(t.shape, generator=g).double().to(DEV)

        def f(s):
            y = [u.detach().double() + (s * d if j == i else 0) for j, u in enumerate(x)]
            ro, rS = O.head_decay_scan(*y[:4], state=y[4])
            return ((ro * dO).sum() + (rS * dS).sum()).item()
        want = (f(h) - f(-h)) / (2 * h)
        have = (grads[i].double() * d).sum().item()
        size = (bg[i] * d.abs()).sum().item()
        assert abs(have - want) <= (r + p + 128 + 144) * 2.0 ** -24 * size + 1e-7 * size, (i, have, want)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("T", [9, 77])
def test_layouts(dtype, T):
    """Transposed views, odd row strides, offset bases and stride-0 gradients give what
    contiguous copies give."""
    H, r, p = 3, 34, 21
    q, k, v, logA, _ = inputs(H, H, T, r, p, H, dtype, seed=6)
    want = A.head_decay_scan(q, k, v, logA)

    def packed(t):                                   # (T, H, cols) memory, rows padded by 3
        buf = torch.full((T + 1, H, t.shape[-1] + 3), float("nan"), device=DEV, dtype=t.dtype)
        view = buf[1:, :, 1:1 + t.shape[-1]]
        view.copy_(t.transpose(0, 1))
        return view.transpose(0, 1)
    args = [packed(t) for t in (q, k, v)] + [torch.stack([logA, logA], 1)[:, 0]]
    assert torch.equal(A.head_decay_scan(*args), want)
    x = [t.detach().requires_grad_(True) for t in args]
    y = [t.detach().requires_grad_(True) for t in (q, k, v, logA)]
    A.head_decay_scan(*x).sum().backward()
    A.head_decay_scan(*y).backward(torch.ones_like(want))
    for a, b in zip(x, y):
        assert torch.equal(a.grad, b.grad)


def test_shared_keys_and_broadcast_inputs():
    """Key heads shared by value heads, one key for all tokens: gradients are sums."""
    nbk, group, T, r, p = 2, 3, 70, 16, 24
    q, k, v, logA, _ = inputs(nbk * group, nbk, T, r, p, 6, FP32, seed=4)
    q.requires_grad_(True)
    k1 = k[:, :1].clone().requires_grad_(True)
    o = A.head_decay_scan(q, k1.expand(nbk, T, r), v, logA)
    ql, k2 = q.detach().clone().requires_grad_(True), k1.detach().clone().requires_grad_(True)
    o2 = A.head_decay_scan(ql.repeat_interleave(group, 0),
                           k2.repeat(1, T, 1).repeat_interleave(group, 0), v, logA)
    assert torch.equal(o, o2)
    dO = torch.randn(o.shape, generator=torch.Generator().manual_seed(1)).to(DEV)
    a, b = torch.autograd.grad(o, (q, k1), dO), torch.autograd.grad(o2, (ql, k2), dO)
    _, (_, _, bg) = oracle(ql.detach(), k2.detach().expand(nbk, T, r), v, logA, None, 1.0, None, dO,
                           torch.zeros(nbk * group, r, p, device=DEV))
    for x, y, big in zip(a, b, (bg[0], bg[1].sum(1, keepdim=True))):
        # both sums of `group` (and T) values round at most so often, of the magnitudes' sum
        assert ((x - y).abs() <= 2 * (group + T) * 2.0 ** -24 * big).all()


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_offsets_past_32_bits(dtype):
    """Rows further apart than 2^31 elements in all."""
    T, r, p, st = 66, 32, 32, 2 ** 25 + 32 + 3
    q, k, v, logA, _ = inputs(1, 1, T, r, p, 1, dtype, seed=7)
    far = torch.empty(T * st, device=DEV, dtype=dtype).view(1, T, st)[:, :, :p]
    far.copy_(v)
    assert torch.equal(A.head_decay_scan(q, k, far, logA), A.head_decay_scan(q, k, v, logA))
    far.copy_(k)
    x = [t.requires_grad_(True) for t in (q, far, v)]
    a = torch.autograd.grad(A.head_decay_scan(*x, logA).sum(), x)
    x = [q, k.requires_grad_(True), v]
    b = torch.autograd.grad(A.head_decay_scan(*x, logA).sum(), x)
    for s, t in zip(a, b):
        assert torch.equal(s, t)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_segments_and_sequences_keep_apart(dtype, bad):
    """What is not finite in one segment or sequence reaches no other one: outputs, states and
    gradients of the others stay the same bits."""
    nb, T, r, p, off = 3, 64 * 40, 64, 40, [0, 64 * 20 + 5, 64 * 20 + 35, 64 * 40]
    q, k, v, logA, S = inputs(nb, nb, T, r, p, 3, dtype, seed=15, lead=(3,))
    dO = torch.randn(nb, T, p, generator=torch.Generator().manual_seed(3)).to(dtype).to(DEV)
    seg = A.Segments(off, DEV)

    def run(x, dO):
        x = [t.clone().requires_grad_(True) for t in x]
        o, So = A.head_decay_scan(*x[:3], logA, state=x[3], segments=seg, return_state=True)
        return [o.detach(), So.detach(), *torch.autograd.grad(o, x, dO)]
    want = run((q, k, v, S), dO)
    for j, (lo, hi) in enumerate(zip(off, off[1:])):
        y, dO2 = [t.clone() for t in (q, k, v, S)], dO.clone()
        for t in (*y[:3], dO2):
            t[1, lo:hi] = bad
        y[3][j, 1] = bad
        got = run(y, dO2)
        for i, (a, b) in enumerate(zip(got, want)):
            a, b = a.clone(), b.clone()
            if i in (1, 5):                          # states: (segment, sequence)
                a[j, 1] = b[j, 1] = 0
            else:
                a[1, lo:hi] = b[1, lo:hi] = 0
            assert torch.equal(a, b), (i, j)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_far_apart_magnitudes(dtype):
    """Values at the ends of the type's range: subnormal ones beside the largest."""
    nb, T, r, p = 2, 100, 16, 24
    q, k, v, logA, S = inputs(nb, nb, T, r, p, 2, dtype, seed=11, lead=())
    info = torch.finfo(dtype)
    v = v * (info.smallest_normal * 0.3 if dtype != FP32 else 1e-30)
    v[:, ::5] = info.max / 2 if dtype == FP16 else 1e30
    k = k * 2.0 ** -6
    o, So = A.head_decay_scan(q, k, v, logA, scale=2.0 ** -8, state=S, return_state=True)
    (ro, rS, _), (bo, bS, _) = oracle(q, k, v, logA, S, 2.0 ** -8, None)
    check("S", So, rS, bS, 2, r, p)
    check("o", o, ro, bo, 2, r, p)
