"""Drafted trees: what the argument checks refuse, on the CPU."""
import pytest
import torch

from smat_attention_amd.kernels import hip_fwd


@pytest.mark.parametrize("lo", [0, 1, 3])
def test_positions_do_not_overlap_the_accepted_nodes(monkeypatch, lo):
    """Workgroups read nodes while one of them moves its request's position."""
    monkeypatch.setattr(hip_fwd, "_on_gpu", lambda who, *ts: None)
    buf = torch.zeros(8, dtype=torch.int32)
    S = torch.zeros(4, 8, 9)
    tree = hip_fwd.DraftTree([-1, 0], "cpu")
    with pytest.raises(ValueError, match="must not be nodes"):
        hip_fwd.tree_state(torch.zeros(4, 2, 8), torch.zeros(4, 2, 9), tree, buf[2:4] if lo == 1
                           else buf[:4], S, torch.empty_like(S),
                           ahead=buf[lo:lo + (2 if lo == 1 else 4)])
