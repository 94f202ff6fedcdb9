"""The gated delta rule and drafted trees as programs use them: in graphs that share their
inputs, on streams of their own, over padded batches, and past 2^31 elements."""
import pytest
import torch

import oracle.delta_ref as O
from test_gpu_delta import (BF16, DEV, FP16, FP32, _check, _inputs, _random_parents, _tree_case,
                            _tree_check)

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from smat_attention_amd import attention as A


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


def test_two_graphs_over_the_same_inputs():
    """Packed training and a few tokens, captured apart and replayed in turn, with eager work and
    synchronisations between."""
    off = [0, 64 * 20 + 5, 64 * 20 + 5, 64 * 21, 64 * 45 + 1]
    nb, T, r, p = 2, off[-1], 96, 40
    x = [t.requires_grad_(True) for t in _inputs(nb, 1, T, r, p, FP16, seed=51,
                                                 state=(4,), decay=0.1)]
    seg = A.Segments(off, DEV)
    dO = torch.randn(nb, T, p, device=DEV, dtype=FP16)

    def train():
        o, S = A.gated_delta_scan(*x[:5], state=x[5], segments=seg, return_state=True)
        return [o.detach(), S.detach(), *torch.autograd.grad((o, S), x, (dO, S.detach()))]

    def few():
        with torch.no_grad():
            return A.gated_delta_scan(*(t[:, :7] for t in x[:5]), state=x[5][0],
                                      return_state=True)
    graphs = [_capture(f) for f in (train, few)]
    for rep in range(4):
        with torch.no_grad():
            x[2].copy_(torch.randn_like(x[2]))
            x[5].copy_(torch.randn_like(x[5]))
        for g, _ in graphs if rep % 2 else graphs[::-1]:
            g.replay()
        torch.cuda.synchronize()
        have = [[t.clone() for t in got] for _, got in graphs]
        for h, f in zip(have, (train, few)):
            for a, b in zip(h, f()):
                assert torch.equal(a, b), rep


def test_a_decoder_in_a_graph():
    """A prompt block and tokens of a layer, captured as one; the state goes on from replay to
    replay."""
    nb, r, p, L = 4, 64, 128, 100
    x = _inputs(nb, 2, L + 2, r, p, BF16, seed=52)[:5]
    decs = [A.GatedDeltaDecoder(torch.zeros(nb, r, p, device=DEV), scale=0.125) for _ in range(2)]

    def turn(dec):
        o = [dec.prefill(*(t[:, :L] for t in x))]
        return o + [dec.step(*(t[:, i] for t in x)) for i in (L, L + 1)]
    graph, got = _capture(lambda: turn(decs[0]))
    decs[0].S.zero_()
    for rep in range(4):
        graph.replay()
        torch.cuda.synchronize()
        have = [t.clone() for t in got]
        for a, b in zip(have, turn(decs[1])):
            assert torch.equal(a, b), rep
        assert torch.equal(decs[0].S, decs[1].S)


def test_training_on_another_stream():
    x = [t.requires_grad_(True) for t in _inputs(2, 2, 64 * 35, 48, 64, BF16, seed=53)[:5]]
    dO = torch.randn(2, 64 * 35, 64, device=DEV, dtype=BF16)

    def train():
        return torch.autograd.grad(A.gated_delta_scan(*x), x, dO)
    want = train()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = train()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("T,pad", [(5, 16), (70, 128), (64, 192)])
def test_padding_leaves_the_state(dtype, T, pad):
    """Tokens with beta = 0 and logA = 0 behind a sequence: its outputs, state and gradients are
    those without them, and the padding has none where the outputs' gradient is zero."""
    nb, r, p = 3, 32, 48
    x = _inputs(nb, nb, pad, r, p, dtype, seed=54, state=())
    x[3][:, T:] = 0
    x[4][:, T:] = 0
    x = [t.requires_grad_(True) for t in x]
    y = [t.detach()[:, :T].double().requires_grad_(True) for t in x[:5]]
    y.append(x[5].detach().double().requires_grad_(True))
    o, S = A.gated_delta_scan(*x[:5], state=x[5], return_state=True)
    ro, rS = O.delta_scan(*y[:5], state=y[5])
    chunks = -(-pad // 64)
    _check("o", o.detach()[:, :T], ro.detach(), chunks, r, p)
    _check("S", S.detach(), rS.detach(), chunks, r, p)
    dO = torch.randn(nb, pad, p, device=DEV).to(dtype)
    dO[:, T:] = 0
    dS = torch.randn(nb, r, p, device=DEV)
    got = torch.autograd.grad((o, S), x, (dO, dS))
    ref = torch.autograd.grad((ro, rS), y, (dO[:, :T].double(), dS.double()))
    for i in (0, 1, 2, 4):
        _check(str(i), got[i][:, :T], ref[i], 2 * chunks, r, p)
    assert (got[0][:, T:] == 0).all() and (got[2][:, T:] == 0).all()
    _check("dS0", got[5], ref[5], 2 * chunks, r, p)


def test_past_31_bits():
    """More than 2^31 elements of values, outputs and workspaces: the last sequences are what
    they are in a call of their own."""
    nb, T, r, p = 132, 65536, 32, 256                # 2.2e9 values
    g = torch.Generator(device=DEV).manual_seed(55)
    v = torch.randn(nb, T, p, device=DEV, generator=g, dtype=BF16)
    q, k = (torch.nn.functional.normalize(torch.randn(nb // 2, T, r, device=DEV, generator=g),
                                          dim=-1).to(BF16) for _ in range(2))
    logA = -torch.rand(nb, T, device=DEV, generator=g)
    beta = torch.rand(nb, T, device=DEV, generator=g)
    o, S = A.gated_delta_scan(q, k, v, logA, beta, return_state=True)
    own, oS = A.gated_delta_scan(q[-1:], k[-1:], v[-2:], logA[-2:], beta[-2:], return_state=True)
    assert ((o[-2:].float() - own.float()).abs() <= 2.0 ** -7 * own.float().abs() + 1e-5).all()
    assert (S[-2:] - oS).abs().max() <= 1e-4


def test_a_cache_past_31_bits():
    """A type table of more than 2^31 elements: the last sequences' rows."""
    H, R, M, B, r, p = 8, 17, 9, 970, 128, 129       # 2.2e9 elements of U
    g = torch.Generator(device=DEV).manual_seed(56)
    U = torch.rand(R * H, B, r, p, device=DEV, generator=g)
    S = torch.rand(R * H, r, p, device=DEV, generator=g)
    Phi, Psi, Vb, _, _ = _tree_case(R, H, M, 1, r, p, BF16, seed=57)
    parents = _random_parents(M, 5)
    ahead = torch.full((R,), B - 4, device=DEV, dtype=torch.int32)     # the last types, wrapping
    dec = A.SmatDecoder.from_cache(U, S.clone(), 1, ahead=ahead)
    out = dec.tree_step(Phi, Psi, Vb, A.DraftTree(parents, DEV))
    rows = slice((R - 1) * H, R * H)
    ref, _ = O.tree_nodes(Phi[rows], Psi[rows], Vb[rows], parents, S[rows], U[rows], B - 3)
    _tree_check(out[rows], ref, r, M)


def test_a_step_past_31_bits():
    nb, r, p = 131200, 128, 128
    S = torch.randn(nb, r, p, device=DEV)
    q, k, v, logA, beta, _ = _inputs(nb, nb // 16, 1, r, p, BF16, seed=58)
    x = [t[:, 0] for t in (q, k, v, logA, beta)]
    new = torch.empty_like(S)
    o = A.gated_delta_step(*x, S, out_state=new)
    n = slice(nb - 16, nb)
    ro, rS = O.delta_scan(q[-1:], k[-1:], v[n], logA[n], beta[n], state=S[n])
    _check("o", o[n], ro[:, 0], 1, r, p)
    _check("S", new[n], rS, 1, r, p)
