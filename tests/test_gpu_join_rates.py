"""Dropout's rate: a place is kept with the probability whose inverse scales it."""
import pytest
import torch

from test_gpu_join import DEV, FP32

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from smat_attention_amd import attention as A


def test_the_scale_is_the_inverse_of_the_rate_in_use():
    """The generator's words tell rates apart by 2^-32.  4096.5 of 2^32 words would be kept; the
    threshold (ties to even) keeps 4096, so the scale is 2^20: then the mean of what is
    kept is the input's."""
    rows, D = 8192, 8192
    f = torch.ones(rows, D, device=DEV, dtype=torch.bfloat16)
    h = torch.zeros(rows, D, device=DEV, dtype=FP32)
    seed = torch.tensor([5], device=DEV)
    p = 1 - 4096.5 / 2 ** 32
    f.requires_grad_(True)
    y, _ = A.block_join(f, h, dropout=p, seed=seed)
    there = y.detach() != 0
    # 64 kept on average; five standard deviations
    assert abs(int(there.sum()) - 64) <= 40
    assert (y.detach()[there] == 2.0 ** 20).all()
    df, = torch.autograd.grad(y, f, torch.ones_like(y))
    assert torch.equal(df != 0, there) and (df[there] == 2.0 ** 20).all()
