"""The gated delta rule and drafted trees at the ends of fp32's range: what is finite stays
finite, and reaches no other branch, token before it, segment or sequence."""
import pytest
import torch

import oracle.delta_ref as O
from test_gpu_delta import DEV, FP32, _inputs, _tree_case

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from smat_attention_amd import attention as A

ENDS = [torch.finfo(FP32).min, torch.finfo(FP32).max, 3.397e38]


@pytest.mark.parametrize("end", ENDS)
def test_tree_values_at_the_end_of_the_range(end):
    """A value of fp32's largest magnitudes in one branch and in an unused node: the other
    branches keep their bits, its own node and descendants are right.  Their numerator is this
    value times a score below one, and the other terms vanish beside it: 2^-20 of it covers the
    value's, the score's and the quotient's roundings (40 + 8 of 2^-24, twice)."""
    nb, M, B, r, p = 2, 6, 3, 40, 41
    Phi, Psi, Vb, U, S = _tree_case(1, nb, M, B, r, p, FP32, seed=3)
    Phi, Psi = Phi / r, Psi / r                      # scores below one
    parents = [-1, -1, 0, 1, -2, 2]
    tree = A.DraftTree(parents, DEV)
    dec = A.SmatDecoder.from_cache(U, S, 0)
    want = dec.tree_step(Phi, Psi, Vb, tree)
    Vb2 = Vb.clone()
    Vb2[:, 1, 3] = end
    Vb2[:, 4, 5] = end
    got = dec.tree_step(Phi, Psi, Vb2, tree)
    ref, states = O.tree_nodes(Phi, Psi, Vb2, parents, S, U, 0)
    for j in (0, 2, 4, 5):
        assert torch.equal(got[:, j], want[:, j]), j
    other = [c for c in range(p - 1) if c != 3]
    for j in (1, 3):
        assert torch.equal(got[:, j, other], want[:, j, other]), j
        off = (got[:, j, 3].double() - ref[:, j, 3]).abs()
        assert (off <= 2.0 ** -20 * ref[:, j, 3].abs()).all(), (j, got[:, j, 3], ref[:, j, 3])
    nodes = torch.tensor([3], device=DEV, dtype=torch.int32)
    state = dec.tree_state(Psi, Vb2, tree, nodes)
    assert ((state.double() - states[3]).abs() <= 2.0 ** -20 * states[3].abs() + 1e-5).all()


def test_tree_table_at_the_end_of_the_range():
    """The cache's own values: a column of S near the end."""
    nb, M, B, r, p = 2, 4, 2, 24, 25
    Phi, Psi, Vb, U, S = _tree_case(1, nb, M, B, r, p, FP32, seed=4)
    Phi = torch.zeros_like(Phi)
    Phi[..., 7] = 0.5
    S[:, 7, 2] = torch.finfo(FP32).max
    parents = [-1, 0, 0, 1]
    got = A.SmatDecoder.from_cache(U, S, 0).tree_step(Phi, Psi, Vb, A.DraftTree(parents, DEV))
    ref, _ = O.tree_nodes(Phi, Psi, Vb, parents, S, U, 0)
    assert ((got.double() - ref).abs() <= 2.0 ** -18 * ref.abs().clamp(min=1.0)).all()


@pytest.mark.parametrize("end", ENDS)
@pytest.mark.parametrize("T,off", [(9, None), (150, None), (150, [0, 70, 100, 150])])
def test_scan_values_at_the_end_of_the_range(T, off, end):
    """One value of fp32's largest magnitudes in one column: everything stays finite, the tokens
    before it, the other columns, segments and sequences keep their bits, and its own column is
    right to the largest magnitude's fp32 accuracy."""
    nb, r, p, at, col = 3, 33, 40, T // 2, 6
    lead = () if off is None else (len(off) - 1,)
    q, k, v, logA, beta, S = _inputs(nb, nb, T, r, p, FP32, seed=31, state=lead)
    beta[1, at] = 1.0                                # the whole value is written
    v2 = v.clone()
    v2[1, at, col] = end
    seg = None if off is None else A.Segments(off, DEV)
    want, wS = A.gated_delta_scan(q, k, v, logA, beta, state=S, segments=seg, return_state=True)
    got, gS = A.gated_delta_scan(q, k, v2, logA, beta, state=S, segments=seg, return_state=True)
    ro, rS = O.delta_scan(q, k, v2, logA, beta, state=S, offsets=off)
    assert torch.isfinite(got).all() and torch.isfinite(gS).all()
    after = torch.zeros(nb, T, p, dtype=torch.bool, device=DEV)
    stop = T if off is None else next(b for b in off if b > at)
    after[1, at:stop, col] = True
    assert torch.equal(got[~after], want[~after])
    lim = 3 * (r + p + 128) * 2.0 ** -24             # three chunks, see _bound of the scan's tests
    assert (got.double() - ro)[after].abs().max() <= lim * ro[after].abs().max()
    assert (gS.double() - rS).abs().max() <= lim * rS.abs().max()


@pytest.mark.parametrize("T", [40, 64 * 40 + 5])
def test_gradient_at_the_end_of_the_range(T):
    """An output gradient at the end of the range in one column: that column's dV is right, the
    others keep their bits, and so do later tokens."""
    nb, r, p, at, col = 2, 32, 32, T // 2, 5
    q, k, v, logA, beta, S = _inputs(nb, nb, T, r, p, FP32, seed=32, state=(), decay=0.1)
    v = v.requires_grad_(True)
    g = torch.Generator().manual_seed(4)
    dO = torch.randn(nb, T, p, generator=g).to(DEV)
    dO2 = dO.clone()
    dO2[1, at, col] = torch.finfo(FP32).min
    o = A.gated_delta_scan(q, k, v, logA, beta, scale=0.5, state=S)
    (want,), (got,) = (torch.autograd.grad(o, (v,), d, retain_graph=True) for d in (dO, dO2))
    assert torch.isfinite(got).all()
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[1, :at + 1, col] = True
    assert torch.equal(got[~hit], want[~hit])
    y = v.detach().double().requires_grad_(True)
    ro, _ = O.delta_scan(q, k, y, logA, beta, scale=0.5, state=S)
    (ref,) = torch.autograd.grad(ro, (y,), dO2.double())
    lim = 2 * -(-T // 64) * (r + p + 128) * 2.0 ** -24
    assert (got.double() - ref)[hit].abs().max() <= lim * ref[hit].abs().max()
