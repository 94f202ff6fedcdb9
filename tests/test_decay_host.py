"""The checks of head_decay_scan's, head_decay_step's and block_join's arguments, on the CPU, and
their oracles against themselves."""
import math

import pytest
import torch

import oracle.decay_ref as D
import oracle.join_ref as J
from smat_attention_amd import attention as A
from smat_attention_amd.kernels import _lib, hip_decay, hip_delta, hip_fwd, hip_join
from smat_attention_amd.kernels._lib import HipKernelError

FAKE = 1 << 20                         # never dereferenced: the refusal comes first


def _args(nb=2, nbk=2, T=3, r=8, p=9, heads=2):
    return [torch.zeros(nbk, T, r), torch.zeros(nbk, T, r), torch.zeros(nb, T, p),
            torch.zeros(heads)]


@pytest.fixture
def anywhere(monkeypatch):
    """Lets the argument checks run on host tensors (nothing is launched)."""
    for m in (hip_delta, hip_fwd):
        monkeypatch.setattr(m, "_on_gpu", lambda who, *ts: None)


def test_host_tensors_are_refused():
    with pytest.raises(ValueError, match="GPU"):
        A.head_decay_scan(*_args())
    with pytest.raises(ValueError, match="GPU"):
        A.head_decay_step(*(t[:, 0] for t in _args()[:3]), torch.zeros(2), torch.zeros(2, 8, 9))
    with pytest.raises(ValueError, match="GPU"):
        A.HeadDecayDecoder(torch.zeros(2, 8, 9), torch.zeros(2))
    with pytest.raises(ValueError, match="GPU"):
        A.block_join(torch.zeros(2, 8), torch.zeros(2, 8))


def _scan(args, state=None, segments=None):
    hip_decay.check_scan("head_decay_scan", *args, state, segments)


def test_scan_refusals(anywhere):
    _scan(_args())
    _scan(_args(nb=4, nbk=2, heads=1), state=torch.zeros(4, 8, 9))
    seg = hip_delta.Segments([0, 1, 3], "cpu")
    _scan(_args(), state=torch.zeros(2, 2, 8, 9), segments=seg)
    for i, shape in ((1, (2, 3, 6)), (2, (2, 4, 9)), (3, (2, 3)), (3, (3,)), (3, (0,))):
        a = _args()
        a[i] = torch.zeros(shape)
        with pytest.raises(ValueError):
            _scan(a)
    for kw in (dict(nb=3, nbk=2, heads=1), dict(nb=2, nbk=0)):
        with pytest.raises(ValueError, match="divide"):
            _scan(_args(**kw))
    for state, s in ((torch.zeros(2, 2, 8, 9), None), (torch.zeros(2, 8, 9), seg)):
        with pytest.raises(ValueError, match="state"):
            _scan(_args(), state=state, segments=s)
    with pytest.raises(TypeError, match="float32"):
        _scan(_args(), state=torch.zeros(2, 8, 9, dtype=torch.bfloat16))
    for kw, match in ((dict(r=129), "key size 129"), (dict(p=129), "value size 129"),
                      (dict(r=0), "key size 0")):
        with pytest.raises(ValueError, match=match):
            _scan(_args(**kw))
    a = _args()
    a[1] = a[1].half()
    with pytest.raises(TypeError, match="share a dtype"):
        _scan(a)
    with pytest.raises(TypeError):
        _scan([t.double() for t in _args()])
    a = _args()
    a[3] = a[3].double()
    with pytest.raises(TypeError, match="logA"):
        _scan(a)
    with pytest.raises(ValueError, match="sequences, T, columns"):
        _scan([t[0] for t in _args()[:3]] + [torch.zeros(1)])
    a = _args()
    a[:3] = [t[:, :1].expand(2, 2 ** 31 - 63, t.shape[2]) for t in a[:3]]
    with pytest.raises(ValueError, match="at most 2\\^31 - 64"):
        _scan(a)
    q, _, v, la = _args(T=4)
    with pytest.raises(ValueError, match="segments end at 3"):
        hip_decay._Plan("head_decay_scan", q, v, 2, seg)


def _step(q=None, k=None, v=None, logA=None, state=None, out=None, out_state=None):
    pick = lambda x, y: y if x is None else x
    return hip_decay.step(pick(q, torch.zeros(2, 8)), pick(k, torch.zeros(2, 8)),
                          pick(v, torch.zeros(4, 9)), pick(logA, torch.zeros(2)),
                          pick(state, torch.zeros(4, 8, 9)), 1.0, out, out_state)


def test_step_refusals(anywhere):
    S = torch.zeros(4, 8, 9)
    big = torch.zeros(2 * S.numel())
    for kw in (dict(k=torch.zeros(2, 9)), dict(q=torch.zeros(3, 8), k=torch.zeros(3, 8)),
               dict(v=torch.zeros(3, 9)), dict(logA=torch.zeros(3)), dict(logA=torch.zeros(1, 2)),
               dict(state=torch.zeros(4, 9, 8)), dict(out_state=torch.zeros(4, 8, 8)),
               dict(out=torch.zeros(4, 8)), dict(q=torch.zeros(8)),
               dict(state=S.transpose(0, 1).contiguous().transpose(0, 1)),
               dict(logA=torch.zeros(4)[::2]),
               dict(q=torch.zeros(8, 2).t()),
               dict(state=big[:S.numel()].view_as(S), out_state=big[9:9 + S.numel()].view_as(S)),
               dict(q=torch.zeros(2, 129), k=torch.zeros(2, 129), state=torch.zeros(4, 129, 9))):
        with pytest.raises(ValueError):
            _step(**kw)
    for kw in (dict(k=torch.zeros(2, 8).half()), dict(state=S.half()),
               dict(out=torch.zeros(4, 9).half()), dict(out_state=S.half()),
               dict(logA=torch.zeros(2).double())):
        with pytest.raises(TypeError):
            _step(**kw)


def test_entry_refusals():
    """What the C entries themselves refuse, before any launch."""
    def scan(nb=1, nbk=1, heads=1, T=17, nch=1, r=8, p=8, st=8, ws=FAKE << 8, dtype=0, nseg=1,
             nruns=1, tables=(None,) * 3, save_s=None):
        _lib.call("smat_head_decay_scan", dtype, FAKE, FAKE, FAKE, FAKE, None, FAKE, None, None,
                  save_s, *tables, nb, nbk, heads, T, nseg, nch, nruns, 1, r, p, 1.0, 64, st, 64, 8, 64, 8,
                  ws, 1 << 50, None)
    for kw, match in ((dict(r=7), "must lie in 8..128"), (dict(p=129), "must lie in 8..128"),
                      (dict(nb=3, nbk=2), "must divide"), (dict(nb=3, heads=2), "must divide"),
                      (dict(nb=1 << 23), "below 2\\^23"), (dict(st=1 << 23), "elements apart"),
                      (dict(st=-8), "elements apart"), (dict(T=65), "1 chunks for T=65"),
                      (dict(T=65, nch=2), "runs of 1 chunks"), (dict(dtype=3), "unknown dtype"),
                      (dict(tables=(FAKE, None, None)), "need the chunk"),
                      (dict(save_s=FAKE + 4), "16-byte aligned"),
                      (dict(T=2 ** 31 - 1, nch=2 ** 25), "bad sizes")):
        with pytest.raises(HipKernelError, match=match):
            scan(**kw)
    with pytest.raises(HipKernelError, match="workspace"):
        _lib.call("smat_head_decay_scan", 0, FAKE, FAKE, FAKE, FAKE, None, FAKE, None, None, None,
                  None, None, None, 1, 1, 1, 128, 1, 2, 2, 1, 8, 8, 1.0, *[8] * 6, FAKE << 8, 64,
                  None)

    def join(rows=1, D=8, gate=0, p=0.0, seed=None, h=0, dtype=0, types=(2, 2, 2), eps=0.0, z=None):
        _lib.call("smat_block_join", dtype, h, FAKE, FAKE, z, None, None, None, *types, seed, FAKE,
                  None, None, rows, D, gate, eps, 1.0, p, 0, 8, 8, 8, None)
    for kw, match in ((dict(D=7), "7 columns"), (dict(D=8193), "8193 columns"),
                      (dict(rows=2 ** 31), "rows"), (dict(gate=4), "unknown gate"),
                      (dict(p=0.5), "needs a seed"), (dict(p=1.0, seed=FAKE), "dropout"),
                      (dict(h=1), "residual stream"), (dict(dtype=7, h=7), "unknown dtype"),
                      (dict(types=(2, 5, 2)), "weight dtype"), (dict(eps=-1.0), "eps"),
                      (dict(gate=2), "null pointer")):
        with pytest.raises(HipKernelError, match=match):
            join(**kw)
    assert _lib.query("smat_block_join_workspace_bytes", 0, 64) == 0
    assert _lib.query("smat_block_join_workspace_bytes", 10, 8193) == 0


def test_join_refusals(anywhere):
    f, w, seed = torch.zeros(3, 16), torch.zeros(16), torch.zeros(1, dtype=torch.int64)

    def check(f=f, h=f, gate=None, post=None, scale=1.0, pre=None, dropout=0.0, seed=None):
        hip_join.check(f, h, gate, post, scale, pre, dropout, seed)
    check()
    check(gate=f, post=w, scale=w, pre=w, dropout=0.5, seed=seed)
    check(f=f.half(), h=f, pre=w.bfloat16())
    for kw in (dict(h=f[:2]), dict(gate=f[:, :8]), dict(post=w[:8]), dict(scale=torch.zeros(1)),
               dict(pre=f), dict(f=f[:, :7], h=f[:, :7]), dict(dropout=0.5),
               dict(dropout=0.5, seed=7), dict(dropout=0.5, seed=torch.zeros(1)),
               dict(dropout=0.5, seed=torch.zeros(2, dtype=torch.int64)),
               dict(f=torch.zeros(()), h=torch.zeros(()))):
        with pytest.raises(ValueError):
            check(**kw)
    for kw in (dict(f=f.half(), h=f.bfloat16()), dict(gate=f.half()), dict(f=f.double()),
               dict(pre=w.double())):
        with pytest.raises(TypeError):
            check(**kw)
    for kw in (dict(gate_kind="tanh"), dict(eps=-1e-6), dict(eps=math.nan), dict(dropout=1.0),
               dict(dropout=-0.1), dict(salt=-1), dict(salt=2 ** 32)):
        opt = dict(gate=f, gate_kind="silu", scale=1.0, eps=1e-6, dropout=0.0, salt=0)
        opt.update(kw)
        with pytest.raises(ValueError):
            hip_join.Options(**opt)
    # a gate's kind is checked only as a name: without a gate there is none
    assert hip_join.Options(None, "silu", 1.0, 1e-6, 0.0, 0).gate == 0


def test_the_generator_is_philox():
    """Known answers of Philox 4x32 with ten rounds, published with it."""
    assert J.philox((0,) * 4, (0,) * 2) == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    assert J.philox((0xffffffff,) * 4, (0xffffffff,) * 2) == [0x408f276d, 0x41c83b0e, 0xa20bc7c6,
                                                             0x6d5451fd]


def test_the_oracle_is_the_sum_over_pairs():
    """The recurrence against o_i = scale sum_j a^(i-j) (q_i . k_j) v_j, and the state's part."""
    g = torch.Generator().manual_seed(0)
    q, k, v, S = (torch.randn(*s, generator=g, dtype=torch.float64)
                  for s in ((2, 9, 3), (2, 9, 3), (4, 9, 5), (4, 3, 5)))
    la = torch.tensor([-0.1, -math.inf], dtype=torch.float64)
    o, So = D.head_decay_scan(q, k, v, la, scale=0.5, state=S)
    for s in range(4):
        a, T = math.exp(la[s % 2]), 9
        W = torch.tensor([[a ** (i - j) if j <= i else 0.0 for j in range(T)] for i in range(T)],
                         dtype=torch.float64)
        e = torch.tensor([a ** (i + 1) for i in range(T)], dtype=torch.float64)[:, None]
        want = 0.5 * (((q[s // 2] @ k[s // 2].t()) * W) @ v[s] + e * (q[s // 2] @ S[s]))
        assert torch.allclose(o[s], want, rtol=1e-12, atol=1e-12)
    assert torch.allclose(So[1], k[0, -1, :, None] * v[1, -1, None], rtol=1e-12, atol=0)


def test_run_lengths_stay_within_a_grid():
    """Every size gets a run length, and runs that a launch can hold."""
    for dtype in (0, 1, 2):
        for nb in (1, 7, 300, 70000):
            for nch in (1, 2, 33, 5000, 1 << 20):
                K = _lib.query("smat_head_decay_run_chunks", dtype, nb, nch, None, None, 0, 64, 128)
                assert 1 <= K <= nch and -(-nch // K) <= 65535
    assert _lib.query("smat_head_decay_run_chunks", 0, 8, 100, None, None, 0, 129, 64) == 1
