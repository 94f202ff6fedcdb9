"""The limits of the gated delta rule's sizes and strides, on the CPU."""
import os
import re

import pytest
import torch

from smat_attention_amd.kernels import _lib, hip_delta
from smat_attention_amd.kernels._lib import HipKernelError

FAKE = 1 << 20                         # never dereferenced: the refusal comes first


def test_a_single_row_is_near():
    """torch ignores the stride of an axis of one row: it is no distance between rows."""
    far = torch.empty_strided((2, 1, 4), (4, 2 ** 23, 1))
    assert far.contiguous().stride(1) == 2 ** 23
    t, sb, st = hip_delta._near_rows(far)
    assert t.data_ptr() == far.data_ptr() and (sb, st) == (4, 4)
    assert hip_delta._near_rows(torch.empty(2, 0, 4))[2] == 4


def test_sequences_beyond_a_grid_are_refused():
    """In chunks 65535 sequences; token by token, and trees, what a grid's first axis holds."""
    def scan(nb, T):
        _lib.call("smat_delta_scan", 0, FAKE, FAKE, FAKE, FAKE, FAKE, None, FAKE, None, None, None,
                  None, None, None, None, nb, nb, T, 1, 1, 1, 1, 8, 8, 1.0, *[64] * 10, FAKE,
                  1 << 50, None)
    with pytest.raises(HipKernelError, match="within 65535"):
        scan(65536, 17)
    with pytest.raises(HipKernelError, match="below 2\\^24"):
        scan(1 << 24, 16)
    with pytest.raises(HipKernelError, match="below 2\\^24"):
        _lib.call("smat_delta_step", 0, *[FAKE] * 8, 1 << 24, 1, 8, 8, 1.0, 8, 8, 8, 1, 1, None)
    with pytest.raises(HipKernelError, match="below 2\\^23"):
        _lib.call("smat_tree_step", 0, *[FAKE] * 9, None, 1 << 23, 1, 1, 2, 1, 1, 8, 9, 0,
                  *[0] * 6, None)
    with pytest.raises(HipKernelError, match="below 2\\^23"):
        _lib.call("smat_tree_state", 0, *[FAKE] * 3, FAKE + 64, FAKE, FAKE, None, 1 << 23, 1, 1, 2,
                  8, 9, *[0] * 4, None)


def test_run_lengths_keep_within_the_grid():
    """Many short segments and a long one: cut so that the runs stay within 65535, where a call
    without cuts does."""
    short = list(range(65501))
    for off in (short + [short[-1] + 64 * 4096], short + [short[-1] + 64 * 4096 + 1]):
        seg = hip_delta.Segments(off, "cpu")
        assert len(seg) == 65501
        for code in range(3):
            K = seg.run_chunks(code, 1, 64, 64)
            assert seg.runs(K)[0].shape[0] <= 65535, (code, K)


def test_few_tokens_are_the_same_number_on_both_sides():
    """Calls of up to FEW_TOKENS tokens bring no workspace, which kFewTokens says is needed."""
    src = os.path.join(os.path.dirname(hip_delta.__file__), "..", "csrc", "delta_common.hpp")
    with open(src) as f:
        (n,) = re.findall(r"constexpr int kFewTokens = (\d+);", f.read())
    assert int(n) == hip_delta.FEW_TOKENS
