"""The limits of the gated delta rule's sizes and strides, on the CPU."""
import torch

from smat_attention_amd.kernels import hip_delta


def test_a_single_row_is_near():
    """torch ignores the stride of an axis of one row: it is no distance between rows."""
    far = torch.empty_strided((2, 1, 4), (4, 2 ** 23, 1))
    assert far.contiguous().stride(1) == 2 ** 23
    t, sb, st = hip_delta._near_rows(far)
    assert t.data_ptr() == far.data_ptr() and (sb, st) == (4, 4)
    assert hip_delta._near_rows(torch.empty(2, 0, 4))[2] == 4
