"""The gated delta rule (gated_delta_scan, its gradient, gated_delta_step) and drafted trees
over the decode cache, against the token-by-token oracle in 64 bits.

Tolerances.  A result stored in type t is off by its rounding, eps(t) / 2 of its value, and by
the arithmetic before it.  That arithmetic is fp32 sums of products whose operands carry at
least 24 bits (two terms, 2^-17, for what ends in a 16-bit output): a chunk adds at most
(r + p + 128) roundings of 2^-24 of the largest magnitude involved, and the chunks' errors add
up at most linearly, since the state's map is no expansion for |k| <= 1 and 0 <= beta <= 2.  So
``_bound`` allows chunks * (r + p + 128) * 2^-24 of the largest value, plus 2^-15 (two operands
of 2^-17, twice over for the two sums) of the largest value where outputs are 16-bit.
"""
import math

import pytest
import torch

import oracle.delta_ref as O

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from smat_attention_amd import attention as A

DEV = "cuda:0"
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _bound(got, ref, chunks, r, p, sixteen):
    big = ref.abs().max().item() if ref.numel() else 0.0
    tol = chunks * (r + p + 128) * 2.0 ** -24 * big + (2.0 ** -15 * big if sixteen else 0.0)
    half = torch.finfo(got.dtype).eps / 2 * ref.abs()
    return half + tol + torch.finfo(got.dtype).tiny


def _check(name, got, ref, chunks, r, p):
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    if not ref.numel():
        return
    assert torch.isfinite(got).all(), name
    off = (got.double() - ref).abs()
    lim = _bound(got, ref, chunks, r, p, got.dtype != FP32)
    worst = (off - lim).max().item()
    assert worst <= 0, f"{name}: off by {off.max().item():.3e}, {worst:.3e} beyond the bound"


def _inputs(nb, nbk, T, r, p, dtype, seed=0, state=None, decay=1.0):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)
    unit = lambda *s: torch.nn.functional.normalize(rn(*s), dim=-1)
    q, k = unit(nbk, T, r).to(dtype), unit(nbk, T, r).to(dtype)
    # rounding can leave a norm a little above one; the bound above needs |k| <= 1
    k = (k.float() * (1 - 2.0 ** -6)).to(dtype)
    v = rn(nb, T, p).to(dtype)
    logA = -decay * torch.nn.functional.softplus(rn(nb, T) - 2.0)
    beta = torch.sigmoid(rn(nb, T))
    S = None if state is None else rn(*state, nb, r, p)
    return [None if t is None else t.to(DEV) for t in (q, k, v, logA, beta, S)]


SHAPES = [
    # nb, nbk, T, r, p, offsets, state
    (3, 3, 1, 64, 64, None, True),
    (3, 1, 7, 40, 50, None, False),
    (300, 150, 16, 128, 256, None, True),
    (2, 2, 17, 33, 9, None, True),
    (2, 2, 63, 128, 128, None, False),
    (2, 1, 64, 64, 64, None, True),
    (4, 2, 65, 96, 80, None, True),
    (1, 1, 200, 17, 33, None, False),
    (2, 2, 130, 1, 1, None, True),
    (2, 2, 129, 128, 256, None, True),
    (4, 1, 150, 33, 47, [0, 1, 1, 64, 129, 150], True),
    (2, 2, 140, 64, 64, [0, 70, 140], False),
    (1, 1, 70, 5, 129, [0, 0, 70], True),
]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("nb,nbk,T,r,p,off,st", SHAPES)
def test_scan_and_gradients(dtype, nb, nbk, T, r, p, off, st):
    nseg = 1 if off is None else len(off) - 1
    lead = () if off is None else (nseg,)
    q, k, v, logA, beta, S = _inputs(nb, nbk, T, r, p, dtype, seed=T + r,
                                     state=lead if st else None)
    scale = r ** -0.5
    seg = None if off is None else A.Segments(off, DEV)
    chunks = sum(-(-(b - a) // 64) for a, b in zip(off or [0], (off or [0, T])[1:])) or 1
    ref_in = [t.double().requires_grad_(True) for t in (q, k, v, logA, beta)]
    S64 = None if S is None else S.double().requires_grad_(True)
    ro, rS = O.delta_scan(*ref_in, scale=scale, state=S64, offsets=off)
    with torch.no_grad():
        o, So = A.gated_delta_scan(q, k, v, logA, beta, scale=scale, state=S, segments=seg,
                                   return_state=True)
    assert o.dtype == dtype and So.dtype == FP32
    _check("o", o, ro.detach(), chunks, r, p)
    _check("S", So, rS.detach(), chunks, r, p)

    g = torch.Generator().manual_seed(9)
    dO = torch.randn(o.shape, generator=g).to(dtype).to(DEV)
    dS = torch.randn(So.shape, generator=g).to(DEV)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v, logA, beta)]
    Sl = None if S is None else S.clone().requires_grad_(True)
    o2, S2 = A.gated_delta_scan(*leaves, scale=scale, state=Sl, segments=seg, return_state=True)
    if T > 16 or off is not None:                    # fewer are taken one by one without grad
        assert torch.equal(o2.detach(), o) and torch.equal(S2.detach(), So)
    _check("o with grad", o2.detach(), ro.detach(), chunks, r, p)
    _check("S with grad", S2.detach(), rS.detach(), chunks, r, p)
    wrt = leaves + ([Sl] if st else [])
    got = torch.autograd.grad((o2, S2), wrt, (dO, dS))
    ref = torch.autograd.grad((ro, rS), ref_in + ([S64] if st else []), (dO.double(), dS.double()))
    # dlogA sums the whole chunk's terms, each as large as max |S| |dS|
    for name, a, b, x in zip(("dq", "dk", "dv", "dlogA", "dbeta", "dS0"), got, ref, wrt):
        assert a.dtype == x.dtype
        if name == "dlogA":
            terms = (rS.detach().abs().max() * dS.abs().max()).item() * r * p
            off_by = (a.double() - b).abs().max().item()
            assert off_by <= chunks * (r + p + 128) * 2.0 ** -24 * max(terms, b.abs().max().item())
        else:
            _check(name, a, b, 2 * chunks, r, p)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_fp32_results_have_fp32_accuracy(dtype):
    """The state and the gates' gradients are fp32 whatever the inputs' type.  One chunk: each
    value is off by about sqrt(r + p + 128) independent roundings of 2^-24; twice that in the
    mean over the values."""
    nb, T, r, p = 4, 64, 64, 64
    q, k, v, logA, beta, S = _inputs(nb, nb, T, r, p, dtype, seed=21, state=())
    x = [t.requires_grad_(True) for t in (q, k, v, logA, beta, S)]
    o, So = A.gated_delta_scan(*x[:5], state=S, return_state=True)
    y = [t.detach().double().requires_grad_(True) for t in x]
    ro, rS = O.delta_scan(*y[:5], state=y[5])
    dO = torch.randn(o.shape, generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
    got = (So, *torch.autograd.grad(o, x[3:], dO))
    ref = (rS, *torch.autograd.grad(ro, y[3:], dO.double()))
    for name, a, b in zip(("S", "dlogA", "dbeta", "dS0"), got, ref):
        off = ((a.detach().double() - b.detach()).norm() / b.detach().norm()).item()
        assert off <= 2 * math.sqrt(r + p + 128) * 2.0 ** -24, (name, off)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("nb,nbk,T,r,p,off,st", [
    (2, 2, 64 * 40 + 5, 64, 64, None, True),
    (2, 1, 64 * 33, 128, 48, None, False),
    (1, 1, 64 * 70 + 1, 40, 33, [0, 64 * 50 + 3, 64 * 50 + 3, 64 * 70 + 1], True),
])
def test_split_along_the_sequence(dtype, nb, nbk, T, r, p, off, st):
    """Few long sequences are cut into runs joined through their transitions."""
    lead = () if off is None else (len(off) - 1,)
    q, k, v, logA, beta, S = _inputs(nb, nbk, T, r, p, dtype, seed=3, state=lead if st else None,
                                     decay=0.1)
    seg = None if off is None else A.Segments(off, DEV)
    from smat_attention_amd.kernels.hip_delta import _Plan
    assert _Plan("test", q, v, seg).nruns > (len(seg) if seg else 1)
    leaves = [t.requires_grad_(True) for t in (q, k, v, logA, beta)]
    o, So = A.gated_delta_scan(*leaves, state=S, segments=seg, return_state=True)
    ref_in = [t.detach().double().requires_grad_(True) for t in leaves]
    ro, rS = O.delta_scan(*ref_in, state=S, offsets=off)
    chunks = -(-T // 64)
    _check("o", o.detach(), ro.detach(), chunks, r, p)
    _check("S", So.detach(), rS.detach(), chunks, r, p)
    dO = torch.randn(o.shape, generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
    got = torch.autograd.grad(o, leaves, dO)
    ref = torch.autograd.grad(ro, ref_in, dO.double())
    for name, a, b in zip(("dq", "dk", "dv", "dlogA", "dbeta"), got, ref):
        _check(name, a, b, 2 * chunks, r, p)


@pytest.mark.parametrize("st,want", [(True, True), (False, True), (True, False), (False, False)])
@pytest.mark.parametrize("off", [None, [0, 64 * 20 + 3, 64 * 20 + 3, 64 * 20 + 40, 64 * 41 + 9]])
def test_split_gradients_of_the_states(off, st, want):
    """Runs' transitions are formed where a state enters, or where one leaves and a gradient may
    come back through it: each of the four, over one sequence and over packed ones."""
    nb, T, r, p = 2, 64 * 41 + 9, 48, 32
    lead = () if off is None else (len(off) - 1,)
    q, k, v, logA, beta, S = _inputs(nb, nb, T, r, p, FP32, seed=13, state=lead if st else None,
                                     decay=0.02)
    x = [t.requires_grad_(True) for t in (q, k, v, logA, beta)] + ([S.requires_grad_(True)] if st
                                                                   else [])
    seg = None if off is None else A.Segments(off, DEV)
    got = A.gated_delta_scan(*x[:5], state=S, segments=seg, return_state=want)
    y = [t.detach().double().requires_grad_(True) for t in x]
    ref = O.delta_scan(*y[:5], state=y[5] if st else None, offsets=off)
    got, ref = (got, ref) if want else ((got,), ref[:1])
    g = torch.Generator().manual_seed(14)
    d = [torch.randn(t.shape, generator=g).to(DEV) for t in got]
    got = torch.autograd.grad(got, x, d)
    ref = torch.autograd.grad(ref, y, [t.double() for t in d])
    for name, a, b in zip(("dq", "dk", "dv", "dlogA", "dbeta", "dS0"), got, ref):
        if name == "dlogA" and want:                 # sums terms as large as <dS, S>
            continue
        _check(name, a, b, 2 * -(-T // 64), r, p)


@pytest.mark.parametrize("kind", ["resets", "strong", "same_keys", "beta2", "beta0", "no_decay"])
def test_hard_gates(kind):
    """Decays to zero, writes that replace everything, keys that repeat, padding tokens."""
    nb, T, r, p = 2, 150, 32, 40
    q, k, v, logA, beta, S = _inputs(nb, nb, T, r, p, FP32, seed=5, state=())
    if kind == "resets":
        logA[:, ::7] = -math.inf
    if kind == "strong":
        logA = logA * 200
    if kind == "same_keys":
        k = k[:, :1].expand_as(k)
        beta = torch.ones_like(beta)
    if kind == "beta2":
        beta = torch.full_like(beta, 2.0)
    if kind == "beta0":
        beta[:, 20:] = 0
        logA[:, 20:] = 0
    if kind == "no_decay":
        logA = torch.zeros_like(logA)
    o, So = A.gated_delta_scan(q, k, v, logA, beta, state=S, return_state=True)
    ro, rS = O.delta_scan(q, k, v, logA, beta, state=S)
    _check("o", o, ro, 3, r, p)
    _check("S", So, rS, 3, r, p)
    if kind == "beta0":
        assert torch.allclose(So, O.delta_scan(*(t[:, :20] for t in (q, k, v, logA, beta)),
                                               state=S)[1].float(), rtol=1e-5, atol=1e-5)


def test_gradient_against_differences():
    """The directional derivative of <o, dO> + <S, dS>: central differences of the oracle in 64
    bits (truncation h^2, cancellation 2^-52 / h: both far below the fp32 gradients')."""
    nb, T, r, p = 2, 100, 24, 16
    q, k, v, logA, beta, S = _inputs(nb, nb, T, r, p, FP32, seed=8, state=())
    x = [t.requires_grad_(True) for t in (q, k, v, logA, beta, S)]
    g = torch.Generator().manual_seed(2)
    dO, dS = torch.randn(nb, T, p, generator=g).to(DEV), torch.randn(nb, r, p, generator=g).to(DEV)
    o, So = A.gated_delta_scan(*x[:5], state=x[5], return_state=True)
    grads = torch.autograd.grad((o, So), x, (dO, dS))
    h = 1e-5
    for i, t in enumerate(x):
        d = torch.randn(t.shape, generator=g).double().to(DEV)

        def f(s):
            y = [u.detach().double() + (s * d if j == i else 0) for j, u in enumerate(x)]
            ro, rS = O.delta_scan(*y[:5], state=y[5])
            return ((ro * dO).sum() + (rS * dS).sum()).item()
        want = (f(h) - f(-h)) / (2 * h)
        have = (grads[i].double() * d).sum().item()
        size = (grads[i].double() * d).abs().sum().item()
        assert abs(have - want) <= 4 * (r + p + 128) * 2.0 ** -24 * size + 1e-7 * size, (i, have, want)


def test_shared_keys_and_broadcast_inputs():
    """Key heads shared by value heads, gates broadcast over heads: gradients are sums."""
    nbk, group, T, r, p = 2, 3, 70, 16, 24
    q, k, v, logA, beta, _ = _inputs(nbk * group, nbk, T, r, p, FP32, seed=4)
    la1 = logA[:1].clone().requires_grad_(True)
    q.requires_grad_(True)
    o = A.gated_delta_scan(q, k, v, la1.expand(nbk * group, T), beta)
    ql, la2 = q.detach().clone().requires_grad_(True), la1.detach().clone().requires_grad_(True)
    o2 = A.gated_delta_scan(ql.repeat_interleave(group, 0), k.repeat_interleave(group, 0), v,
                            la2.repeat(nbk * group, 1), beta)
    assert torch.equal(o, o2)
    dO = torch.randn(o.shape, generator=torch.Generator().manual_seed(1)).to(DEV)
    a, b = torch.autograd.grad(o, (q, la1), dO), torch.autograd.grad(o2, (ql, la2), dO)
    for x, y in zip(a, b):
        assert (x - y).abs().max() <= group * 2.0 ** -22 * y.abs().max()


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_layouts(dtype):
    """Transposed views, odd row strides, offset bases and stride-0 gradients give what
    contiguous copies give."""
    _layouts(dtype, 77)
    _layouts(dtype, 9)


def _layouts(dtype, T):
    H, r, p = 3, 34, 21
    q, k, v, logA, beta, _ = _inputs(H, H, T, r, p, dtype, seed=6)
    want = A.gated_delta_scan(q, k, v, logA, beta)

    def packed(t):                                   # (T, H, cols) memory, rows padded by 3
        buf = torch.full((T + 1, H, t.shape[-1] + 3), float("nan"), device=DEV, dtype=t.dtype)
        view = buf[1:, :, 1:1 + t.shape[-1]]
        view.copy_(t.transpose(0, 1))
        return view.transpose(0, 1)
    args = [packed(t) for t in (q, k, v)] + [t.t().contiguous().t() for t in (logA, beta)]
    assert torch.equal(A.gated_delta_scan(*args), want)
    x = [t.detach().requires_grad_(True) for t in args]
    y = [t.detach().requires_grad_(True) for t in (q, k, v, logA, beta)]
    A.gated_delta_scan(*x).sum().backward()
    A.gated_delta_scan(*y).backward(torch.ones_like(want))
    for a, b in zip(x, y):
        assert torch.equal(a.grad, b.grad)


def test_offsets_past_32_bits():
    """Rows further apart than 2^31 elements."""
    T, r, p, st = 66, 32, 32, 2 ** 25 + 32
    q, k, v, logA, beta, _ = _inputs(1, 1, T, r, p, BF16, seed=7)
    far = torch.empty(T * st, device=DEV, dtype=BF16).view(1, T, st)[:, :, :p]
    far.copy_(v)
    assert torch.equal(A.gated_delta_scan(q, k, far, logA, beta),
                       A.gated_delta_scan(q, k, v, logA, beta))


def test_far_key_rows():
    """Queries and keys whose rows lie 2^24 elements and more apart."""
    T, r, p, st = 66, 32, 32, 2 ** 24 + 8
    q, k, v, logA, beta, _ = _inputs(1, 1, T, r, p, BF16, seed=7)
    buf = torch.empty(2 * T * st, device=DEV, dtype=BF16).view(2, 1, T, st)[..., :r]
    buf[0].copy_(q)
    buf[1].copy_(k)
    assert torch.equal(A.gated_delta_scan(buf[0], buf[1], v, logA, beta),
                       A.gated_delta_scan(q, k, v, logA, beta))


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_segments_and_sequences_keep_apart(dtype, bad):
    """What is not finite in one segment or sequence reaches no other one: outputs, states and
    gradients of the others stay the same bits."""
    nb, T, r, p, off = 3, 64 * 40, 64, 40, [0, 64 * 20 + 5, 64 * 20 + 35, 64 * 40]
    x = _inputs(nb, nb, T, r, p, dtype, seed=15, state=(3,), decay=0.1)
    dO = torch.randn(nb, T, p, generator=torch.Generator().manual_seed(3)).to(dtype).to(DEV)
    seg = A.Segments(off, DEV)

    def run(x, dO):
        x = [t.clone().requires_grad_(True) for t in x]
        o, S = A.gated_delta_scan(*x[:5], state=x[5], segments=seg, return_state=True)
        return [o.detach(), S.detach(), *torch.autograd.grad(o, x, dO)]
    want = run(x, dO)
    for lo, hi in ((off[0], off[1]), (off[1], off[2]), (off[2], off[3])):
        y, dO2 = [t.clone() for t in x], dO.clone()
        for t in (*y[:5], dO2):
            t[1, lo:hi] = bad
        got = run(y, dO2)
        keep = torch.ones(nb, T, dtype=torch.bool, device=DEV)
        keep[1, lo:hi] = False
        skeep = torch.ones(3, nb, dtype=torch.bool, device=DEV)
        skeep[off.index(lo), 1] = False
        for n, (a, b) in enumerate(zip(got, want)):
            m = skeep if n in (1, 7) else keep
            assert torch.equal(a[m], b[m]), (n, lo)


def test_gradient_with_resets():
    """Decays to zero inside chunks, at their borders and at both ends."""
    nb, T, r, p = 2, 150, 32, 40
    q, k, v, logA, beta, S = _inputs(nb, nb, T, r, p, FP32, seed=16, state=())
    logA[:, [0, 3, 4, 63, 64, 100, 149]] = -math.inf
    x = [t.requires_grad_(True) for t in (q, k, v, logA, beta, S)]
    o, So = A.gated_delta_scan(*x[:5], state=S, return_state=True)
    y = [t.detach().double().requires_grad_(True) for t in x]
    ro, rS = O.delta_scan(*y[:5], state=y[5])
    g = torch.Generator().manual_seed(17)
    d = [torch.randn(t.shape, generator=g).to(DEV) for t in (o, So)]
    got = torch.autograd.grad((o, So), x, d)
    ref = torch.autograd.grad((ro, rS), y, [t.double() for t in d])
    for name, a, b in zip(("dq", "dk", "dv", "dlogA", "dbeta", "dS0"), got, ref):
        assert torch.isfinite(a).all() and torch.isfinite(b).all(), name
        if name == "dlogA":                          # sums terms as large as <dS, S> (see above)
            lim = 3 * (r + p + 128) * 2.0 ** -24 * r * p * (rS.abs().max() * d[1].abs().max())
            assert (a.double() - b).abs().max() <= lim
        else:
            _check(name, a, b, 6, r, p)


def test_two_calls_at_once():
    """Calls on two streams, each with its own workspaces."""
    cases = [_inputs(2, 2, 64 * 36, 64, 64, BF16, seed=s) for s in (18, 19)]
    want = [A.gated_delta_scan(*c[:5]) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(A.gated_delta_scan(*cases[i][:5]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


def test_empty():
    q, k, v, logA, beta, S = _inputs(2, 2, 0, 8, 8, BF16, state=())
    o, So = A.gated_delta_scan(q, k, v, logA, beta, state=S, return_state=True)
    assert o.shape == (2, 0, 8) and torch.equal(So, S)
    x = [t.requires_grad_(True) for t in (q, S)]
    o, So = A.gated_delta_scan(x[0], k, v, logA, beta, state=x[1], return_state=True)
    gq, gS = torch.autograd.grad(So.sum(), x)
    assert gq.shape == q.shape and torch.equal(gS, torch.ones_like(S))
    o, So = A.gated_delta_scan(q.detach()[:0], k[:0], v[:0], logA[:0], beta[:0],
                               return_state=True)
    assert o.shape == (0, 0, 8) and So.shape == (0, 8, 8)


def test_only_the_state_has_a_gradient():
    q, k, v, logA, beta, S = _inputs(2, 2, 70, 16, 16, BF16, state=())
    S.requires_grad_(True)
    o, So = A.gated_delta_scan(q, k, v, logA, beta, state=S, return_state=True)
    (g,) = torch.autograd.grad(So.sum(), S)
    S64 = S.detach().double().requires_grad_(True)
    _, rS = O.delta_scan(q, k, v, logA, beta, state=S64)
    _check("dS0", g, torch.autograd.grad(rS.sum(), S64)[0], 4, 16, 16)


# ---------------------------------------------------------------------------
# one token
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("nb,nbk,r,p", [(1, 1, 64, 64), (6, 2, 128, 128), (3, 3, 1, 1),
                                        (5, 5, 33, 47), (2, 1, 96, 256), (600, 300, 64, 129),
                                        (520, 520, 40, 100)])
def test_step(dtype, nb, nbk, r, p):
    q, k, v, logA, beta, S = _inputs(nb, nbk, 1, r, p, dtype, seed=r, state=())
    ro, rS = O.delta_scan(q, k, v, logA, beta, scale=0.5, state=S)
    keep = S.clone()
    new = torch.empty_like(S)
    o = A.gated_delta_step(q[:, 0], k[:, 0], v[:, 0], logA[:, 0], beta[:, 0], S, scale=0.5,
                           out_state=new)
    assert torch.equal(S, keep) and o.dtype == dtype
    _check("o", o, ro[:, 0], 1, r, p)
    _check("S", new, rS, 1, r, p)
    out = torch.empty_like(o)
    got = A.gated_delta_step(q[:, 0], k[:, 0], v[:, 0], logA[:, 0], beta[:, 0], S, scale=0.5,
                             out=out)
    assert got is out and torch.equal(out, o) and torch.equal(S, new)


def test_decoder_runs_as_the_scan():
    """A prompt in two blocks, then tokens one by one: the whole scan's outputs and state."""
    nb, T, r, p = 4, 150, 48, 64
    q, k, v, logA, beta, _ = _inputs(nb, 2, T, r, p, FP32, seed=11)
    ro, rS = O.delta_scan(q, k, v, logA, beta, scale=0.2)
    dec = A.GatedDeltaDecoder(torch.zeros(nb, r, p, device=DEV), scale=0.2)
    o = [dec.prefill(*(t[:, a:b] for t in (q, k, v, logA, beta))) for a, b in ((0, 7), (7, 140))]
    o += [dec.step(*(t[:, t_] for t in (q, k, v, logA, beta)))[:, None] for t_ in range(140, T)]
    _check("o", torch.cat(o, 1), ro, 3 + 10, r, p)
    _check("S", dec.S, rS, 3 + 10, r, p)


def test_captured_and_replayed():
    """The scan with its gradient and the step in graphs, each replay against the eager call,
    with eager work and synchronisations between the replays."""
    nb, T, r, p = 2, 64 * 34, 32, 32
    x = [t.requires_grad_(True) for t in _inputs(nb, nb, T, r, p, BF16, seed=12)[:5]]
    dO = torch.randn(nb, T, p, device=DEV, dtype=BF16)
    st = torch.randn(nb, r, p, device=DEV)

    def train():
        o = A.gated_delta_scan(*x)
        return (o.detach(), *torch.autograd.grad(o, x, dO))

    def one():
        with torch.no_grad():
            o = A.gated_delta_step(*(t[:, 0] for t in x), st, out_state=nxt)
        return o, nxt
    nxt = torch.empty_like(st)
    for fn in (train, one):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            fn()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = fn()
        for rep in range(4):
            with torch.no_grad():
                for t in x[:3]:
                    t.copy_(torch.randn_like(t) * 0.1)
            graph.replay()
            torch.cuda.synchronize()
            have = [t.clone() for t in got]
            want = fn()
            for a, b in zip(have, want):
                assert torch.equal(a, b), rep


def test_on_another_stream():
    q, k, v, logA, beta, S = _inputs(2, 2, 300, 64, 64, BF16, seed=13, state=())
    want = A.gated_delta_scan(q, k, v, logA, beta, state=S)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = A.gated_delta_scan(q, k, v, logA, beta, state=S)
    side.synchronize()
    assert torch.equal(got, want)


# ---------------------------------------------------------------------------
# drafted trees
# ---------------------------------------------------------------------------

def _tree_case(R, H, M, B, r, p, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)
    Phi = (torch.nn.functional.elu(rn(R * H, M, r)) + 1).to(dtype)
    Psi = (torch.nn.functional.elu(rn(R * H, M, r)) + 1).to(dtype)
    Vb = rn(R * H, M, p)
    Vb[..., -1] = 1
    U, S = rn(R * H, B, r, p), rn(R * H, r, p)
    U[..., -1], S[..., -1] = 20 + U[..., -1].abs(), 20 + S[..., -1].abs()
    return [t.to(DEV) for t in (Phi, Psi, Vb.to(dtype), U, S)]


def _random_parents(M, seed, unused=0):
    g = torch.Generator().manual_seed(seed)
    par = []
    for j in range(M):
        if j >= M - unused:
            par.append(-2)
        else:
            par.append(int(torch.randint(-1, j, (1,), generator=g)) if j else -1)
    return par


def _tree_check(out, ref, r, M):
    """N and its normaliser are fp32 sums of r + r M terms of positive features: the relative
    error of each is (r + M + 8) 2^-24 of the sum of magnitudes, and so is the quotient's of
    the largest output, twice."""
    tol = 2 * (r + M + 8) * 2.0 ** -24 * max(ref.abs().max().item(), 1.0) * 4
    assert out.shape == ref.shape and (out.double() - ref).abs().max().item() <= tol


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("R,H,M,B,r,p", [(1, 1, 1, 1, 1, 2), (1, 4, 8, 5, 64, 65),
                                         (3, 2, 64, 7, 128, 129), (2, 3, 17, 2, 33, 40),
                                         (70, 4, 5, 3, 16, 17), (2, 1, 33, 130, 96, 144)])
def test_tree(dtype, R, H, M, B, r, p):
    Phi, Psi, Vb, U, S = _tree_case(R, H, M, B, r, p, dtype, seed=M)
    parents = [_random_parents(M, 10 * b + M, unused=(b % 3 if M > 5 else 0)) for b in range(R)]
    tree = A.DraftTree(parents, DEV)
    ahead = torch.arange(R, device=DEV, dtype=torch.int32)
    dec = A.SmatDecoder.from_cache(U, S.clone(), 3, ahead=ahead.clone())
    nodes = torch.tensor([(b * 7) % (M + 1) - 1 for b in range(R)], dtype=torch.int32)
    out = dec.tree_step(Phi, Psi, Vb, tree)
    state = dec.tree_state(Psi, Vb, tree, nodes.to(DEV))
    assert torch.equal(dec.S, S)
    for b in range(R):
        rows = slice(b * H, (b + 1) * H)
        ref, states = O.tree_nodes(Phi[rows], Psi[rows], Vb[rows], parents[b], S[rows], U[rows],
                                   3 + b)
        _tree_check(out[rows], ref, r, M)
        n = int(nodes[b])
        after = S[rows].double() if n < 0 or states[n] is None else states[n]
        assert (state[rows].double() - after).abs().max() <= \
            (M + 1) * 2.0 ** -24 * max(after.abs().max().item(), 1.0) * 4
    dec.commit(Psi, Vb, tree, nodes.to(DEV))
    assert torch.equal(dec.S, state)
    taken = [0 if n < 0 or parents[b][n] == -2 else tree.level[b, n] + 1
             for b, n in enumerate(nodes.tolist())]
    assert dec.ahead.tolist() == [b + t for b, t in enumerate(taken)]


def test_tree_is_the_steps_of_its_paths():
    """A chain committed is that many steps; the steps after it take up the new positions."""
    nb, M, B, r, p = 6, 5, 7, 32, 33
    Phi, Psi, Vb, U, S = _tree_case(1, nb, M + 1, B, r, p, BF16, seed=2)
    a = A.SmatDecoder.from_cache(U, S.clone(), 4)
    b = A.SmatDecoder.from_cache(U, S.clone(), 4)
    rows = [t[:, :M].contiguous() for t in (Phi, Psi, Vb)]
    tree = A.DraftTree([-1, 0, 1, 2, 3], DEV)
    got = b.tree_step(*rows, tree)
    want = torch.stack([a.step(Phi[:, j], Psi[:, j], Vb[:, j]) for j in range(M)], 1)
    _tree_check(got, want.double(), r, M)
    b.commit(rows[1], rows[2], tree, torch.full((3,), M - 1, device=DEV, dtype=torch.int32))
    assert (b.S - a.S).abs().max() <= 4 * M * 2.0 ** -24 * a.S.abs().max()
    x, y = (d.step(Phi[:, M], Psi[:, M], Vb[:, M]) for d in (a, b))
    _tree_check(y, x.double(), r, M)
    assert b.ahead.tolist() == [M] * 3 and b.i == 5


def test_tree_keeps_branches_apart():
    """Infinities and NaN in one branch, and in unused nodes, reach no other branch."""
    nb, M, B, r, p = 2, 6, 3, 40, 41
    Phi, Psi, Vb, U, S = _tree_case(1, nb, M, B, r, p, FP32, seed=3)
    parents = [-1, -1, 0, 1, -2, 2]
    tree = A.DraftTree(parents, DEV)
    dec = A.SmatDecoder.from_cache(U, S, 0)
    want = dec.tree_step(Phi, Psi, Vb, tree)
    for bad in (float("nan"), float("inf")):
        Psi2, Vb2, Phi2 = Psi.clone(), Vb.clone(), Phi.clone()
        for t in (Psi2, Vb2, Phi2):
            t[:, 1] = bad
            t[:, 4] = bad
        got = dec.tree_step(Phi2, Psi2, Vb2, tree)
        for j in (0, 2, 4, 5):
            assert torch.equal(got[:, j], want[:, j]), (bad, j)
        nodes = torch.tensor([5], device=DEV, dtype=torch.int32)
        assert torch.equal(dec.tree_state(Psi2, Vb2, tree, nodes),
                           dec.tree_state(Psi, Vb, tree, nodes))


def test_tree_layouts_and_graph():
    """Strided rows; a verification round (read, commit, step) captured and replayed."""
    R, H, M, B, r, p = 2, 3, 9, 4, 48, 49
    Phi, Psi, Vb, U, S = _tree_case(R, H, M, B, r, p, BF16, seed=5)
    tree = A.DraftTree(_random_parents(M, 1), DEV)
    dec = A.SmatDecoder.from_cache(U, S.clone(), 0)
    want = dec.tree_step(Phi, Psi, Vb, tree)

    def packed(t):
        buf = torch.full((M, R * H, t.shape[-1] + 5), float("nan"), device=DEV, dtype=t.dtype)
        buf[:, :, 3:3 + t.shape[-1]].copy_(t.transpose(0, 1))
        return buf[:, :, 3:3 + t.shape[-1]].transpose(0, 1)
    assert torch.equal(dec.tree_step(packed(Phi), packed(Psi), packed(Vb), tree), want)

    nodes = torch.tensor([4, -1], device=DEV, dtype=torch.int32)
    ahead = torch.zeros(R, device=DEV, dtype=torch.int32)
    dec = A.SmatDecoder.from_cache(U, S.clone(), 0, ahead=ahead)

    def round_():
        o = dec.tree_step(Phi, Psi, Vb, tree)
        dec.commit(Psi, Vb, tree, nodes)
        o2 = dec.tree_step(Phi, Psi, Vb, tree)
        dec.commit(Psi, Vb, tree, nodes)             # an even number: the first buffer again
        return o, o2
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        round_()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = round_()
    eager = A.SmatDecoder.from_cache(U, S.clone(), 0, ahead=torch.zeros_like(ahead))
    dec.S.copy_(S)
    ahead.zero_()
    for rep in range(4):
        graph.replay()
        torch.cuda.synchronize()
        want = []
        for _ in range(2):
            want.append(eager.tree_step(Phi, Psi, Vb, tree))
            eager.commit(Psi, Vb, tree, nodes)
        for a, b in zip(got, want):
            assert torch.equal(a, b), rep
        assert torch.equal(dec.S, eager.S) and torch.equal(ahead, eager.ahead)
