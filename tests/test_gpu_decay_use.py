"""Linear attention with a decay for each head and the block's end as programs use them: tokens
one by one, decoders, captured graphs, streams, large tensors, and a small model of both."""
import math

import pytest
import torch

import oracle.decay_ref as O
import oracle.join_ref as J
from test_gpu_decay import BF16, FP16, FP32, DEV, check, inputs, oracle

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from smat_attention_amd import attention as A


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("nb,nbk,r,p,heads", [(1, 1, 64, 64, 1), (6, 2, 128, 128, 3), (3, 3, 1, 1, 3),
                                              (5, 5, 33, 47, 1), (2, 1, 96, 7, 2),
                                              (600, 300, 64, 127, 4), (520, 520, 40, 100, 8)])
def test_step(dtype, nb, nbk, r, p, heads):
    q, k, v, logA, S = inputs(nb, nbk, 1, r, p, heads, dtype, seed=r, lead=())
    (ro, rS, _), (bo, bS, _) = oracle(q, k, v, logA, S, 0.5, None)
    keep, new = S.clone(), torch.empty_like(S)
    x = [t[:, 0] for t in (q, k, v)]
    o = A.head_decay_step(*x, logA, S, scale=0.5, out_state=new)
    assert torch.equal(S, keep) and o.dtype == dtype
    check("o", o, ro[:, 0], bo[:, 0], 1, r, p)
    check("S", new, rS, bS, 1, r, p)
    out = torch.empty_like(o)
    got = A.head_decay_step(*x, logA, S, scale=0.5, out=out)
    assert got is out and torch.equal(out, o) and torch.equal(S, new)
    # rows apart
    wide = [torch.full((t.shape[0], t.shape[1] + 3), math.nan, device=DEV, dtype=dtype) for t in x]
    for w, t in zip(wide, x):
        w[:, 1:1 + t.shape[1]] = t
    far = [w[:, 1:1 + t.shape[1]] for w, t in zip(wide, x)]
    new2 = torch.empty_like(keep)
    assert torch.equal(A.head_decay_step(*far, logA, keep, scale=0.5, out_state=new2), o)
    assert torch.equal(new2, new)


def test_step_without_sequences():
    z = torch.zeros
    o = A.head_decay_step(z(0, 8, device=DEV), z(0, 8, device=DEV), z(0, 9, device=DEV),
                          z(2, device=DEV), z(0, 8, 9, device=DEV))
    assert o.shape == (0, 9)


@pytest.mark.parametrize("la", [0.0, -math.inf])
def test_step_at_the_ends(la):
    q, k, v, _, S = inputs(2, 2, 1, 16, 24, 2, FP32, seed=4, lead=())
    logA = torch.tensor([la, -0.5], device=DEV)
    (ro, rS, _), (bo, bS, _) = oracle(q, k, v, logA, S, 1.0, None)
    o = A.head_decay_step(q[:, 0], k[:, 0], v[:, 0], logA, S)
    check("o", o, ro[:, 0], bo[:, 0], 1, 16, 24)
    check("S", S, rS, bS, 1, 16, 24)


def test_decoder_runs_as_the_scan():
    """A prompt in two blocks, then tokens one by one: the whole scan's outputs and state."""
    nb, T, r, p = 4, 150, 48, 64
    q, k, v, logA, _ = inputs(nb, 2, T, r, p, 2, FP32, seed=11)
    (ro, rS, _), (bo, bS, _) = oracle(q, k, v, logA, None, 0.2, None)
    dec = A.HeadDecayDecoder(torch.zeros(nb, r, p, device=DEV), logA, scale=0.2)
    o = [dec.prefill(*(t[:, a:b] for t in (q, k, v))) for a, b in ((0, 7), (7, 140))]
    o += [dec.step(*(t[:, t_] for t in (q, k, v)))[:, None] for t_ in range(140, T)]
    check("o", torch.cat(o, 1), ro, bo, 3 + 10, r, p)
    check("S", dec.S, rS, bS, 3 + 10, r, p)
    assert dec.cache_words() == nb * r * p


def test_a_prompt_in_pieces_is_the_prompt():
    """Cuts at chunk borders carry the state on, so outputs keep the scan's accuracy anywhere."""
    nb, T, r, p = 2, 300, 32, 72
    q, k, v, logA, S = inputs(nb, nb, T, r, p, 1, FP32, seed=2, lead=())
    (ro, rS, _), (bo, bS, _) = oracle(q, k, v, logA, S, 1.0, None)
    for cuts in ([64, 128], [1, 2, 65], [299]):
        st, o = S, []
        for a, b in zip([0] + cuts, cuts + [T]):
            x, st = A.head_decay_scan(*(t[:, a:b] for t in (q, k, v)), logA, state=st,
                                      return_state=True)
            o.append(x)
        ch = 5 + len(cuts)
        check("o", torch.cat(o, 1), ro, bo, ch, r, p)
        check("S", st, rS, bS, ch, r, p)


def test_empty():
    q, k, v, logA, S = inputs(2, 2, 0, 8, 8, 2, BF16, lead=())
    x = [t.requires_grad_(True) for t in (q, S, logA)]
    o, So = A.head_decay_scan(x[0], k, v, x[2], state=x[1], return_state=True)
    assert o.shape == (2, 0, 8) and torch.equal(So, S)
    gq, gS, gA = torch.autograd.grad(So.sum(), x)
    assert gq.shape == q.shape and torch.equal(gS, torch.ones_like(S)) and not gA.any()
    x = [t.detach()[:0].requires_grad_(True) for t in (q, k, v)]
    la = logA.detach().requires_grad_(True)
    o, So = A.head_decay_scan(*x, la, return_state=True)
    assert o.shape == (0, 0, 8) and So.shape == (0, 8, 8)
    assert not torch.autograd.grad(So.sum(), la)[0].any()


def test_only_the_state_or_the_decay_has_a_gradient():
    q, k, v, logA, S = inputs(2, 2, 70, 16, 16, 2, BF16, lead=())
    zero = torch.zeros(2, 70, 16, device=DEV, dtype=BF16)
    (_, _, rg), (_, _, bg) = oracle(q, k, v, logA, S, 1.0, None, zero, torch.ones_like(S))
    for i, t in ((3, logA), (4, S)):
        t.requires_grad_(True)
        _, So = A.head_decay_scan(q, k, v, logA, state=S, return_state=True)
        g, = torch.autograd.grad(So.sum(), t)
        check(str(i), g, rg[i], bg[i], 4, 16, 16)
        t.requires_grad_(False)


def test_two_calls_at_once():
    """Calls on two streams, each with its own workspaces."""
    cases = [inputs(2, 2, 64 * 36, 64, 64, 2, BF16, seed=s) for s in (18, 19)]
    dO = torch.randn(2, 64 * 36, 64, device=DEV, dtype=BF16)
    h = torch.randn(2, 64 * 36, 64, device=DEV)
    seed = torch.tensor([3], device=DEV)

    def one(c):
        x = [t.detach().requires_grad_(True) for t in c[:4]]
        o = A.head_decay_scan(*x)
        y = A.block_join(o.detach(), h, pre_weight=torch.ones(64, device=DEV), dropout=0.1, seed=seed)
        return [o.detach(), *torch.autograd.grad(o, x, dO), *y]
    want = [one(c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(one(cases[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[i]))


def _capture(fn):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fn()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = fn()
    return graph, got


def test_captured_and_replayed():
    """The scan with its gradient (packed too), the step, and the block's end with its seed
    stepped between replays, each replay against the eager call, with eager work and
    synchronisations between the replays."""
    nb, T, r, p = 2, 64 * 34, 32, 32
    x = [t.requires_grad_(True) for t in inputs(nb, nb, T, r, p, 2, BF16, seed=12)[:4]]
    dO = torch.randn(nb, T, p, device=DEV, dtype=BF16)
    st, nxt = torch.randn(nb, r, p, device=DEV), torch.empty(nb, r, p, device=DEV)
    seg = A.Segments([0, 700, 701, T], DEV)
    f, h = torch.randn(300, 200, device=DEV, dtype=BF16), torch.randn(300, 200, device=DEV)
    z, w = torch.randn_like(f), torch.ones(200, device=DEV)
    y = [t.requires_grad_(True) for t in (f, h, z, w)]
    seed = torch.tensor([5], device=DEV)

    def train():
        o = A.head_decay_scan(*x)
        return (o.detach(), *torch.autograd.grad(o, x, dO))

    def packed():
        o = A.head_decay_scan(*x, segments=seg)
        return (o.detach(), *torch.autograd.grad(o, x, dO))

    def one():
        with torch.no_grad():
            return A.head_decay_step(*(t[:, 0] for t in x[:3]), x[3], st, out_state=nxt), nxt

    def join():
        a, b = A.block_join(y[0], y[1], post_weight=y[3], gate=y[2], scale=y[3], pre_weight=y[3],
                            dropout=0.3, seed=seed, salt=2)
        return (a.detach(), b.detach(), *torch.autograd.grad(a.sum() + b.float().sum(), y))
    for fn in (train, packed, one, join):
        graph, got = _capture(fn)
        for rep in range(4):
            with torch.no_grad():
                for t in (*x[:3], *y[:3]):
                    t.copy_(torch.randn_like(t) * 0.1)
            seed += 1
            graph.replay()
            torch.cuda.synchronize()
            have = [t.clone() for t in got]
            want = fn()
            for a, b in zip(have, want):
                assert torch.equal(a, b), (fn.__name__, rep)


def test_two_graphs_of_the_same_inputs():
    """Graphs captured one after the other keep workspaces apart: replayed in turn, on one stream
    and on two, each gives the eager call's results."""
    x = inputs(2, 2, 64 * 36, 64, 64, 2, BF16, seed=30)
    v2 = torch.randn_like(x[2])
    want = [A.head_decay_scan(*x[:4]), A.head_decay_scan(x[0], x[1], v2, x[3])]
    graphs = [_capture(lambda v=v: A.head_decay_scan(x[0], x[1], v, x[3])) for v in (x[2], v2)]
    for rep in range(3):
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for (_, o), w in zip(graphs, want))
        streams = [torch.cuda.Stream() for _ in graphs]
        for (g, o), st in zip(graphs, streams):
            o.zero_()
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for (_, o), w in zip(graphs, want))


def test_on_another_stream():
    q, k, v, logA, S = inputs(2, 2, 300, 64, 64, 1, BF16, seed=13, lead=())
    want = A.head_decay_scan(q, k, v, logA, state=S)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = A.head_decay_scan(q, k, v, logA, state=S)
    side.synchronize()
    assert torch.equal(got, want)


def test_past_31_bits():
    """More than 2^31 elements of values and outputs: the last sequences are what they are in a
    call of their own; and of the block's end's rows."""
    nb, T, r, p = 264, 65536, 32, 128                # 2.2e9 values
    g = torch.Generator(device=DEV).manual_seed(55)
    v = torch.randn(nb, T, p, device=DEV, generator=g, dtype=BF16)
    q, k = (torch.nn.functional.normalize(torch.randn(nb // 2, T, r, device=DEV, generator=g),
                                          dim=-1).to(BF16) for _ in range(2))
    logA = torch.tensor([-0.05, -0.3], device=DEV)
    o, S = A.head_decay_scan(q, k, v, logA, return_state=True)
    own, oS = A.head_decay_scan(q[-1:], k[-1:], v[-2:], logA, return_state=True)
    # the same sums cut into other runs: fp32's roundings apart, then one bf16 rounding each
    assert ((o[-2:].float() - own.float()).abs() <= 2.0 ** -7 * own.float().abs() + 1e-4).all()
    assert (S[-2:] - oS).abs().max() <= 1e-4
    del q, k, S, oS
    w = torch.rand(128, device=DEV)
    h, x = A.block_join(v.view(-1, p), o.view(-1, p), post_weight=w, pre_weight=w)
    a, b = A.block_join(v[-1], o[-1], post_weight=w, pre_weight=w)
    assert torch.equal(h[-T:], a) and torch.equal(x[-T:], b)


def test_the_same_tensor_twice():
    """One tensor as queries, keys and values, and as a block's output and its residual: the
    gradients are the sums of the separate ones'."""
    q, _, _, logA, _ = inputs(2, 2, 200, 64, 64, 2, FP32, seed=40)
    dO = torch.randn(2, 200, 64, device=DEV)
    one = q.clone().requires_grad_(True)
    three = [q.clone().requires_grad_(True) for _ in range(3)]
    a, b = A.head_decay_scan(one, one, one, logA), A.head_decay_scan(*three, logA)
    assert torch.equal(a, b)
    got, = torch.autograd.grad(a, one, dO)
    dq, dk, dv = (t.double() for t in torch.autograd.grad(b, three, dO))
    # two fp32 additions, in whichever order
    lim = 2 * 2.0 ** -24 * (dq.abs() + dk.abs() + dv.abs())
    assert ((got.double() - (dq + dk + dv)).abs() <= lim).all()
    w = torch.rand(64, device=DEV)
    two = [q.clone().requires_grad_(True) for _ in range(2)]
    (h, x), (h2, x2) = (A.block_join(f, r, post_weight=w, pre_weight=w)
                        for f, r in ((one, one), two))
    assert torch.equal(h, h2) and torch.equal(x, x2)
    got, = torch.autograd.grad((h, x), one, (dO, dO))
    df, dh = (t.double() for t in torch.autograd.grad((h2, x2), two, (dO, dO)))
    assert ((got.double() - (df + dh)).abs() <= 2.0 ** -24 * (df.abs() + dh.abs())).all()


def test_an_input_changed_after_the_forward_is_refused():
    q, k, v, logA, _ = inputs(1, 1, 70, 16, 16, 1, FP32, seed=41)
    f = v.clone()
    x = [t.requires_grad_(True) for t in (q, k, v, logA)]
    o = A.head_decay_scan(*x)
    r = f.clone().requires_grad_(True)
    h, _ = A.block_join(f, r, gate=f)
    with torch.no_grad():
        x[2].zero_()
        f.zero_()
    for y in (o, h):
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            torch.autograd.grad(y.sum(), x if y is o else r)


def _layer(P, x, h, scan, join, mask):
    """One block over (B, T, D): projections, the scan over heads, the output's projection, and
    the block's end."""
    B, T, Dm = x.shape
    H, hd = 2, Dm // 2
    heads = lambda t: t.view(B, T, H, hd).transpose(1, 2).reshape(B * H, T, hd)
    q, k, v = (heads(x @ P[n]) for n in ("q", "k", "v"))
    o = scan(q, k, v, P["logA"], hd ** -0.5)
    f = o.view(B, H, T, hd).transpose(1, 2).reshape(B, T, Dm) @ P["o"]
    return join(f, h, P, x @ P["z"], mask)


def test_a_model_of_both():
    """Two blocks as a training program has them, with dropout: outputs and the gradients of every
    parameter against 64 bits.  A value passes, a block, products of 64 terms, the scan's r + p +
    128 + 72 chunks = 408 roundings and the block's end's 128, each way: some 2 * 2 * (4 * 64 + 408
    + 128) of 2^-24, which a norm's division by an rms near one keeps as they are; four times that
    of the largest value."""
    B, T, Dm, p = 2, 100, 64, 0.2
    g = torch.Generator().manual_seed(5)
    rn = lambda *s: torch.randn(*s, generator=g)
    names = ("q", "k", "v", "o", "z")
    layers = [{**{n: rn(Dm, Dm) * Dm ** -0.5 for n in names}, "logA": -0.02 - 0.3 * torch.rand(2),
               "post": 1 + 0.1 * rn(Dm), "s": 0.5 + 0.1 * rn(Dm), "pre": 1 + 0.1 * rn(Dm)}
              for _ in range(2)]
    x0, dx, dh = rn(B, T, Dm), rn(B, T, Dm), rn(B, T, Dm)
    seed = torch.tensor([77], device=DEV)

    def mine(f, h, P, z, salt):
        return A.block_join(f, h, post_weight=P["post"], gate=z, gate_kind="silu", scale=P["s"],
                            pre_weight=P["pre"], dropout=p, seed=seed, salt=salt)

    def theirs(f, h, P, z, salt):
        m = J.kept(range(B * T), Dm, p, 77, salt).view(B, T, Dm).double().to(DEV) / (1 - p)
        return J.block_join(f, h, P["post"], z, "silu", P["s"], P["pre"], 1e-6, m)

    def run(dtype, scan, join):
        Ps = [{n: t.to(DEV, dtype).requires_grad_(True) for n, t in P.items()} for P in layers]
        h = x = x0.to(DEV, dtype)
        for i, P in enumerate(Ps):
            h, x = _layer(P, x, h, scan, join, i)
        leaves = [t for P in Ps for t in P.values()]
        grads = torch.autograd.grad((h, x), leaves, (dh.to(DEV, dtype), dx.to(DEV, dtype)))
        return [h.detach(), x.detach(), *grads]
    got = run(FP32, lambda q, k, v, la, s: A.head_decay_scan(q, k, v, la, scale=s), mine)
    ref = run(torch.float64, lambda q, k, v, la, s: O.head_decay_scan(q, k, v, la, scale=s)[0],
              theirs)
    for i, (a, b) in enumerate(zip(got, ref)):
        lim = 4 * 2 * 2 * (4 * 64 + 408 + 128) * 2.0 ** -24 * b.abs().max().item()
        assert (a.double() - b).abs().max().item() <= lim, i


def test_a_model_trains():
    """A step of a captured training program: it runs, and every parameter has a finite gradient."""
    torch.manual_seed(0)
    B, T, Dm = 2, 130, 64
    P = {n: (torch.randn(Dm, Dm, device=DEV) * Dm ** -0.5).to(BF16).requires_grad_(True)
         for n in ("q", "k", "v", "o", "z")}
    P.update({n: torch.ones(Dm, device=DEV, requires_grad=True) for n in ("post", "s", "pre")})
    P["logA"] = torch.tensor([-0.1, -0.01], device=DEV, requires_grad=True)
    x, h = torch.randn(B, T, Dm, device=DEV, dtype=BF16), torch.randn(B, T, Dm, device=DEV)
    seed = torch.tensor([1], device=DEV)

    def fn():
        h2, x2 = _layer(P, x, h, lambda q, k, v, la, s: A.head_decay_scan(q, k, v, la, scale=s),
                        lambda f, h, P, z, salt: A.block_join(
                            f, h, post_weight=P["post"], gate=z, scale=P["s"],
                            pre_weight=P["pre"], dropout=0.1, seed=seed, salt=salt), 0)
        return torch.autograd.grad((h2, x2), list(P.values()),
                                   (torch.ones_like(h2), torch.ones_like(x2)))
    graph, got = _capture(fn)
    graph.replay()
    torch.cuda.synchronize()
    for t, g in zip(P.values(), got):
        assert g.shape == t.shape and g.dtype == t.dtype and torch.isfinite(g).all() and g.any()
