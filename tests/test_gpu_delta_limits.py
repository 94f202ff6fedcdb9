"""The gated delta rule at the limits of its sizes and strides."""
import pytest
import torch

import oracle.delta_ref as O
from test_gpu_delta import BF16, DEV, FP32, _check, _inputs

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from smat_attention_amd import attention as A
    from smat_attention_amd.kernels import _lib
    from smat_attention_amd.kernels._lib import stream_of


def _one_row(t, far):
    """t (n, 1, cols) with a row stride of `far`, which nothing multiplies."""
    return torch.as_strided(t, t.shape, (t.stride(0), far, 1))


@pytest.mark.parametrize("far", [2 ** 23, 2 ** 31 + 1])
@pytest.mark.parametrize("packed", [False, True])
def test_a_single_token_with_a_far_stride(far, packed):
    """One token a call, as a slice of a long batch gives it: forward, gradient and packed."""
    q, k, v, logA, beta, S = _inputs(3, 3, 1, 24, 32, BF16, seed=1, state=(1,) if packed else ())
    dO = torch.randn(3, 1, 32, device=DEV).to(BF16)
    seg = A.Segments([0, 1], DEV) if packed else None

    def run(f):
        x = [f(t).detach().requires_grad_(True) for t in (q, k, v)]
        o = A.gated_delta_scan(*x, logA, beta, state=S, segments=seg)
        with torch.no_grad():
            o2 = A.gated_delta_scan(*x, logA, beta, state=S, segments=seg)
        return o.detach(), o2, *torch.autograd.grad(o, x, f(dO))
    for a, b in zip(run(lambda t: _one_row(t, far)), run(lambda t: t)):
        assert torch.equal(a, b)


def test_few_tokens_take_any_row_stride():
    """The C entry's token-by-token form has 64-bit strides."""
    q, k, v, logA, beta, S = _inputs(2, 2, 2, 16, 16, BF16, seed=2, state=())
    st = 2 ** 23 + 8
    far = torch.empty(2 * st, device=DEV, dtype=BF16)
    far = torch.as_strided(far, (2, 2, 16), (16, st, 1))
    far.copy_(v)
    out = torch.empty(2, 2, 16, device=DEV, dtype=BF16)
    _lib.call("smat_delta_scan", _lib_code(q), q.data_ptr(), k.data_ptr(), far.data_ptr(),
              logA.data_ptr(), beta.data_ptr(), S.data_ptr(), out.data_ptr(), None, None, None,
              None, None, None, None, 2, 2, 2, 1, 1, 1, 1, 16, 16, 1.0, *q.stride()[:2],
              *k.stride()[:2], 16, st, *logA.stride(), *beta.stride(), None, 0, stream_of(q))
    assert torch.equal(out, A.gated_delta_scan(q, k, v, logA, beta, state=S))


def _lib_code(t):
    from smat_attention_amd.kernels.hip_fwd import _code
    return _code(t, "test")


def test_few_tokens_of_many_sequences():
    """More sequences than a grid's second axis holds, for one and for a few tokens."""
    nb, r, p = 70000, 4, 5
    q, k, v, logA, beta, S = _inputs(nb, nb // 2, 3, r, p, FP32, seed=3, state=())
    ro, rS = O.delta_scan(q, k, v, logA, beta, state=S)
    o, So = A.gated_delta_scan(q, k, v, logA, beta, state=S, return_state=True)
    _check("o", o, ro, 1, r, p)
    _check("S", So, rS, 1, r, p)
    x = [t[:, :1] for t in (q, k, v, logA, beta)]
    o, So = A.gated_delta_scan(*x, state=S, return_state=True)
    new = torch.empty_like(S)
    o1 = A.gated_delta_step(*(t[:, 0] for t in x), S, out_state=new)
    assert torch.equal(o[:, 0], o1) and torch.equal(So, new)
