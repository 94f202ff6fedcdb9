"""Gradients of the gated delta rule that are zero, whatever rounds before them."""
import pytest
import torch

from test_gpu_delta import BF16, DEV, FP16, FP32, _inputs

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from smat_attention_amd import attention as A


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("nb,nbk,T,r,p,off", [(4, 4, 1, 64, 64, None), (4, 2, 1, 128, 100, None),
                                              (2, 2, 130, 40, 33, None), (3, 3, 1, 17, 24, None),
                                              (2, 1, 75, 96, 64, [0, 1, 2, 2, 67, 75])])
def test_a_decay_of_nothing_has_no_gradient(dtype, nb, nbk, T, r, p, off):
    """Where no state enters, the first token's decay multiplies zeros: dlogA is zero there, not
    the difference of two equal sums.  With a state of zeros too; with another one it is not."""
    q, k, v, logA, beta, S = _inputs(nb, nbk, T, r, p, dtype, seed=41,
                                     state=() if off is None else (len(off) - 1,))
    seg = None if off is None else A.Segments(off, DEV)
    first = [a for a, b in zip(off or [0], (off or [0, T])[1:]) if b > a]
    logA.requires_grad_(True)
    for state in (None, torch.zeros_like(S), S):
        o, So = A.gated_delta_scan(q, k, v, logA, beta, state=state, segments=seg,
                                   return_state=True)
        dO = torch.randn(o.shape, generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
        (g,) = torch.autograd.grad((o, So), (logA,), (dO, torch.ones_like(So)))
        if state is S:
            assert (g[:, first] != 0).all()
        else:
            assert (g[:, first] == 0).all(), g[:, first].abs().max()
