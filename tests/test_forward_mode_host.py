"""The kernels have no forward-mode derivatives: a call with a tangent is refused, not answered
without one.  On the CPU: the refusal comes before any launch."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from smat_attention_amd import attention as A
from smat_attention_amd.kernels import hip_delta, hip_fwd


@pytest.fixture
def anywhere(monkeypatch):
    """Lets the argument checks run on host tensors (nothing is launched)."""
    for m in (hip_delta, hip_fwd):
        monkeypatch.setattr(m, "_on_gpu", lambda who, *ts: None)


@pytest.mark.parametrize("grad", [True, False])
def test_tangents_are_refused(anywhere, grad):
    x, w = torch.zeros(2, 3, 8), torch.zeros(2)
    with torch.set_grad_enabled(grad), fwAD.dual_level():
        d = fwAD.make_dual(x, torch.ones_like(x))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            A.block_join(d, x)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            A.block_join(x, x, gate=d)
        for args in ((d, x, x), (x, x, d)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                A.head_decay_scan(*args, w)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            A.head_decay_scan(x, x, x, fwAD.make_dual(w, w))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            A.gated_delta_scan(d, x, x, torch.zeros(2, 3), torch.zeros(2, 3))


def test_other_tensors_pass():
    x = torch.zeros(3)
    assert not A._wants_grad(x, None) and A._wants_grad(x.clone().requires_grad_(True))
    with fwAD.dual_level():
        fwAD.make_dual(x, x)
        assert not A._wants_grad(x, None)
