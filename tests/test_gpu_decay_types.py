"""Decays in 16 bits: those of an fp32 copy in every form, with gradients in their own type, and
a decoder that follows its layer's."""
import pytest
import torch

from test_gpu_decay import BF16, DEV, FP16, FP32, inputs

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from smat_attention_amd import attention as A


@pytest.mark.parametrize("a_type", [BF16, FP16])
@pytest.mark.parametrize("T", [5, 150, 64 * 40])
def test_decays_of_16_bits(a_type, T):
    q, k, v, logA, S = inputs(4, 2, T, 32, 48, 2, BF16, seed=T, lead=())
    low = logA.to(a_type)
    dO = torch.randn(4, T, 48, generator=torch.Generator().manual_seed(1)).to(BF16).to(DEV)

    def run(la):
        x = [t.clone().requires_grad_(True) for t in (q, k, v, la, S)]
        o, So = A.head_decay_scan(*x[:4], state=x[4], return_state=True)
        return [o.detach(), So.detach(), *torch.autograd.grad((o, So), x, (dO, S))]
    got, want = run(low), run(low.float())
    assert got[5].dtype == a_type and want[5].dtype == FP32
    for a, b in zip(got, want):
        assert torch.equal(a, b.to(a.dtype))
    a, b = S.clone(), S.clone()
    x = [t[:, 0] for t in (q, k, v)]
    assert torch.equal(A.head_decay_step(*x, low, a), A.head_decay_step(*x, low.float(), b))
    assert torch.equal(a, b)


@pytest.mark.parametrize("a_type", [FP32, BF16, FP16, torch.float64])
@pytest.mark.parametrize("apart", [False, True])
def test_a_decoder_follows_its_layers_decays(a_type, apart):
    """An update of the parameter in place reaches the decoder, whatever its type and stride."""
    q, k, v, logA, S = inputs(2, 2, 3, 16, 24, 2, BF16, seed=3, lead=())
    par = torch.zeros(2, 2 if apart else 1, device=DEV, dtype=a_type)[:, 0]
    par.copy_(logA)
    dec = A.HeadDecayDecoder(S.clone(), par)
    with torch.no_grad():
        par.mul_(4.0)
    want = S.clone()
    o, want = A.head_decay_scan(q, k, v, par.float(), state=want, return_state=True)
    assert torch.equal(dec.prefill(q, k, v), o) and torch.equal(dec.S, want)
    x = [t[:, 0] for t in (q, k, v)]
    o = A.head_decay_step(*x, par.float().contiguous(), want)
    assert torch.equal(dec.step(*x), o) and torch.equal(dec.S, want)
