"""Dropout's mask in late turns of the rows' walk, forward and gradient: the generator's counter is
the row, wherever it is worked on."""
import pytest
import torch

import oracle.join_ref as O
from test_gpu_join import DEV

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from smat_attention_amd import attention as A


@pytest.mark.parametrize("rows,D,some", [
    # the rows around each turn's end (workgroups times rows at a time) and the last ones
    (17000, 40, [0, 2047, 2048, 4095, 4096, 8191, 8192, 16383, 16384, 16998, 16999]),
    (5000, 520, [0, 1023, 1024, 2047, 2048, 4095, 4096, 4999]),
    (1100, 4100, [0, 255, 256, 511, 512, 513, 768, 1023, 1024, 1099]),
    (600, 8192, [0, 255, 256, 511, 512, 599]),
])
def test_the_mask_of_late_rows(rows, D, some):
    p, seed, salt = 0.25, 2 ** 40 + 3, 9
    f = torch.ones(rows, D, device=DEV, requires_grad=True)
    key = torch.tensor([seed], device=DEV)
    y, _ = A.block_join(f, torch.zeros(rows, D, device=DEV), dropout=p, seed=key, salt=salt)
    df, = torch.autograd.grad(y, f, torch.ones_like(y))
    want = O.kept(some, D, p, seed, salt)
    assert torch.equal((y[some] != 0).cpu(), want)
    assert torch.equal((df[some] != 0).cpu(), want)
