"""The checks of the gated delta rule's and the drafted trees' arguments, on the CPU, and the
oracle against itself."""
import pytest
import torch

import oracle.delta_ref as O
from smat_attention_amd import attention as A
from smat_attention_amd.kernels import _lib, hip_delta, hip_fwd
from smat_attention_amd.kernels._lib import HipKernelError


def test_segments_tables():
    s = hip_delta.Segments([0, 1, 1, 130, 194], "cpu")
    assert len(s) == 4 and s.T == 194 and s.nch == 5
    assert s.chunks.tolist() == [[0, 1], [1, 64], [65, 64], [129, 1], [130, 64]]
    runs, segrun = s.runs(2)
    assert runs.tolist() == [[0, 1, 0, 2], [1, 1, 1, 0], [1, 3, 2, 3], [3, 4, 2, 4], [4, 5, 3, 1]]
    assert segrun.tolist() == [0, 1, 2, 4, 5]
    assert s.runs(2)[0] is runs
    assert hip_delta.Segments(torch.tensor([0, 0]), "cpu").nch == 0


@pytest.mark.parametrize("bad", [[0], [1, 5], [0, 5, 4], [0.0, 5.0], [[0, 5]], [0, 2 ** 31]])
def test_segments_refuses(bad):
    with pytest.raises(ValueError):
        hip_delta.Segments(bad, "cpu")


def test_tree_tables():
    t = hip_fwd.DraftTree([[-1, 0, -1, 1, -2], [-1, -1, -1, 0, 3]], "cpu")
    assert (t.trees, t.nodes, t.levels) == (2, 5, 3)
    assert t.anc.tolist() == [[1, 3, 4, 11, 0], [1, 2, 4, 9, 25]]
    assert t.order.tolist() == [[0, 2, 1, 3, 4], [0, 1, 2, 3, 4]]
    assert t.lstart.tolist() == [[0, 2, 3, 4, 4, 4], [0, 3, 4, 5, 5, 5]]
    full = hip_fwd.DraftTree([-1] + list(range(63)), "cpu")
    assert full.levels == 64 and full.anc.tolist()[0][63] == -1      # all 64 bits
    assert hip_fwd.DraftTree([-2], "cpu").levels == 0


@pytest.mark.parametrize("bad", [[], [0], [-1, 1], [-3], [-1, 5], [-2, 0], [0.5], [-1] * 65,
                                 [[[0]]]])
def test_tree_refuses(bad):
    with pytest.raises(ValueError):
        hip_fwd.DraftTree(bad, "cpu")


def _args(nb=2, nbk=2, T=3, r=4, p=5):
    return [torch.zeros(nbk, T, r), torch.zeros(nbk, T, r), torch.zeros(nb, T, p),
            torch.zeros(nb, T), torch.zeros(nb, T)]


def test_host_tensors_are_refused():
    with pytest.raises(ValueError, match="GPU"):
        A.gated_delta_scan(*_args())
    with pytest.raises(ValueError, match="GPU"):
        A.gated_delta_step(*(t[:, 0] for t in _args()), torch.zeros(2, 4, 5))
    with pytest.raises(ValueError, match="GPU"):
        A.GatedDeltaDecoder(torch.zeros(2, 4, 5))
    with pytest.raises(ValueError, match="GPU"):
        A.SmatDecoder.from_cache(torch.zeros(2, 3, 4, 5), torch.zeros(2, 4, 5))


@pytest.fixture
def anywhere(monkeypatch):
    """Lets the argument checks run on host tensors (nothing is launched)."""
    for m in (hip_delta, hip_fwd):
        monkeypatch.setattr(m, "_on_gpu", lambda who, *ts: None)


def _scan_check(args, state=None, segments=None):
    hip_delta.check_scan("gated_delta_scan", *args, state, segments)


def test_scan_refusals(anywhere):
    _scan_check(_args())
    _scan_check(_args(nb=4, nbk=2), state=torch.zeros(4, 4, 5))
    seg = hip_delta.Segments([0, 1, 3], "cpu")
    _scan_check(_args(), state=torch.zeros(2, 2, 4, 5), segments=seg)
    for i, shape in ((1, (2, 3, 6)), (2, (2, 4, 5)), (3, (2, 4)), (4, (3, 3))):
        a = _args()
        a[i] = torch.zeros(shape)
        with pytest.raises(ValueError):
            _scan_check(a)
    with pytest.raises(ValueError, match="divide"):
        _scan_check(_args(nb=3, nbk=2))
    with pytest.raises(ValueError, match="divide"):
        _scan_check(_args(nb=2, nbk=0))
    with pytest.raises(ValueError, match="state"):
        _scan_check(_args(), state=torch.zeros(2, 2, 4, 5))
    with pytest.raises(ValueError, match="state"):
        _scan_check(_args(), state=torch.zeros(2, 4, 5), segments=seg)
    with pytest.raises(TypeError, match="float32"):
        _scan_check(_args(), state=torch.zeros(2, 4, 5, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="key size 129"):
        _scan_check(_args(r=129))
    with pytest.raises(ValueError, match="value size 257"):
        _scan_check(_args(p=257))
    with pytest.raises(ValueError):
        _scan_check(_args(r=0))
    a = _args()
    a[1] = a[1].half()
    with pytest.raises(TypeError, match="share a dtype"):
        _scan_check(a)
    with pytest.raises(TypeError):
        _scan_check([t.double() for t in _args()])
    a = _args()
    a[3] = a[3].double()
    with pytest.raises(TypeError, match="logA"):
        _scan_check(a)
    with pytest.raises(ValueError, match="sequences, T, columns"):
        _scan_check([t[0] for t in _args()])
    long = [t[:, :1].expand(2, 2 ** 31, *t.shape[2:]) for t in _args()]
    with pytest.raises(ValueError, match="at most 2\\^31"):
        _scan_check(long)
    with pytest.raises(ValueError, match="segments end at 3"):
        hip_delta._Plan("gated_delta_scan", *[_args(T=4)[i] for i in (0, 2)], seg)


def test_tree_refusals(anywhere):
    S, U = torch.zeros(4, 8, 9), torch.zeros(4, 3, 8, 9)
    tree = hip_fwd.DraftTree([-1, 0], "cpu")
    Phi, Psi, Vb = torch.zeros(4, 2, 8), torch.zeros(4, 2, 8), torch.zeros(4, 2, 9)

    def step(Phi=Phi, Psi=Psi, Vb=Vb, tree=tree, S=S, U=U, **kw):
        return hip_fwd.tree_step(Phi, Psi, Vb, tree, S, U, 0, **kw)

    for kw in (dict(Phi=Phi[:, :1]), dict(Vb=Vb[..., :8]), dict(U=U[:3]), dict(U=U[..., :8]),
               dict(Psi=Psi[:2]), dict(S=S.transpose(0, 1).contiguous().transpose(0, 1)),
               dict(tree=hip_fwd.DraftTree([[-1, 0]] * 3, "cpu")),
               dict(ahead=torch.zeros(3, dtype=torch.int32)),
               dict(ahead=torch.zeros(2, dtype=torch.int64)),
               dict(out=torch.zeros(4, 2, 9))):
        with pytest.raises(ValueError):
            step(**kw)
    with pytest.raises(TypeError):
        step(Psi=Psi.half())
    with pytest.raises(TypeError):
        step(Phi=Phi.double(), Psi=Psi.double(), Vb=Vb.double())

    def state(nodes, tree=tree, out=None, **kw):
        return hip_fwd.tree_state(Psi, Vb, tree, nodes, S, torch.empty_like(S) if out is None
                                  else out, **kw)
    i32 = dict(dtype=torch.int32)
    for args, kw in (((torch.zeros(3, **i32),), {}), ((torch.zeros(2),), {}),
                     ((torch.zeros(0, **i32),), {}),
                     ((torch.zeros(2, **i32),), dict(ahead=torch.zeros(4, **i32))),
                     ((torch.zeros(2, **i32),), dict(out=S)),
                     ((torch.zeros(4, **i32),), dict(tree=hip_fwd.DraftTree([[-1, 0]] * 2, "cpu")))):
        with pytest.raises(ValueError):
            state(*args, **kw)
    same = torch.zeros(2, **i32)
    with pytest.raises(ValueError, match="must not be nodes"):
        state(same, ahead=same)


def test_run_tables_are_not_staged_in_a_capture(monkeypatch):
    seg = hip_delta.Segments([0, 100, 300], "cpu")
    kept = seg.runs(2)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    seg.device = torch.device("cuda", 0)
    assert seg.runs(2) is kept
    with pytest.raises(RuntimeError, match="cannot be captured"):
        seg.runs(3)


def test_first_commit_is_not_captured(anywhere, monkeypatch):
    """A captured first commit would clear the positions in every replay."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    dec = A.SmatDecoder.from_cache(torch.zeros(2, 3, 8, 9), torch.zeros(2, 8, 9))
    with pytest.raises(RuntimeError, match="cannot be captured"):
        dec.commit(torch.zeros(2, 2, 8), torch.zeros(2, 2, 9), hip_fwd.DraftTree([-1, 0], "cpu"),
                   torch.zeros(2, dtype=torch.int32))
    assert dec.ahead is None


def test_step_refusals(anywhere):
    def step(nb=2, nbk=2, r=4, p=5, state=None, **kw):
        x = dict(q=torch.zeros(nbk, r), k=torch.zeros(nbk, r), v=torch.zeros(nb, p),
                 logA=torch.zeros(nb), beta=torch.zeros(nb),
                 state=torch.zeros(nb, r, p) if state is None else state, out=None,
                 out_state=None)
        x.update(kw)
        return hip_delta.step(x["q"], x["k"], x["v"], x["logA"], x["beta"], x["state"], 1.0,
                              x["out"], x["out_state"])
    base = torch.zeros(2 * 2 * 4 * 5)
    overlapping = dict(state=base[:40].view(2, 4, 5), out_state=base[20:60].view(2, 4, 5))
    for kw in (dict(k=torch.zeros(2, 5)), dict(logA=torch.zeros(3)), dict(nb=3),
               dict(state=torch.zeros(2, 5, 4)), dict(out=torch.zeros(2, 6)),
               dict(out_state=torch.zeros(2, 4, 6)), dict(r=129), dict(p=257), overlapping,
               dict(q=torch.zeros(4, 2).t(), k=torch.zeros(4, 2).t()),
               dict(state=torch.zeros(2, 5, 4).transpose(1, 2)), dict(q=torch.zeros(2, 1, 4))):
        with pytest.raises(ValueError):
            step(**kw)
    for kw in (dict(k=torch.zeros(2, 4).half()), dict(state=torch.zeros(2, 4, 5).half()),
               dict(out=torch.zeros(2, 5).half()), dict(beta=torch.zeros(2).double())):
        with pytest.raises(TypeError):
            step(**kw)


def test_c_entry_points_refuse():
    fake = 1 << 20                     # never dereferenced: validation fails first

    def scan(dtype=0, nb=2, nbk=2, T=64, nseg=1, nch=1, nruns=1, K=1, r=64, p=64, q=fake, n=1 << 40,
             tables=(None, None, None), save=None):
        _lib.call("smat_delta_scan", dtype, q, fake, fake, fake, fake, None, fake, None, save,
                  save, None, *tables, nb, nbk, T, nseg, nch, nruns, K, r, p, 1.0, *[64] * 10, fake, n,
                  None)
    for kw, what in ((dict(dtype=9), "unknown dtype"), (dict(q=None), "null pointer"),
                     (dict(nbk=3), "does not divide"), (dict(r=129), "beyond"),
                     (dict(p=257), "beyond"), (dict(nch=2), "chunks for T"),
                     (dict(nruns=2), "runs"), (dict(n=16), "workspace"),
                     (dict(tables=(fake, None, None)), "tables"), (dict(K=0), "runs"),
                     (dict(T=128, nch=2, nruns=2, save=fake), "save_m")):
        with pytest.raises(HipKernelError, match=what):
            scan(**kw)
    with pytest.raises(HipKernelError, match="at most 64"):
        _lib.call("smat_tree_step", 0, fake, fake, fake, fake, fake, fake, fake, fake, fake, None,
                  1, 1, 1, 65, 1, 1, 8, 9, 0, *[0] * 6, None)
    with pytest.raises(HipKernelError, match="must differ"):
        _lib.call("smat_tree_state", 0, fake, fake, fake, fake, fake, fake, None, 1, 1, 1, 2, 8, 9,
                  *[0] * 4, None)
    with pytest.raises(HipKernelError, match="must divide"):
        _lib.call("smat_decode_step_at", 0, fake, fake, fake, fake, fake + 64, fake, fake, None,
                  fake, 3, 4, 2, 8, 9, 0, 8, 8, 9, None)
    with pytest.raises(HipKernelError, match="null pointer"):
        _lib.call("smat_delta_step", 0, None, fake, fake, fake, fake, fake, fake, fake, 1, 1, 8, 8,
                  1.0, 8, 8, 8, 1, 1, None)


def test_run_lengths():
    for code in range(3):
        def q(nb, nch, r, p):
            return _lib.query("smat_delta_run_chunks", code, nb, nch, None, None, 0, r, p)
        assert q(512, 1000, 64, 64) == 1000          # enough sequences: whole segments
        assert q(1, 3, 64, 64) == 3                  # too short to split
        assert q(1, 0, 64, 64) == 1
        assert 2 <= q(8, 2048, 128, 128) < 2048
        # one long segment among short ones and an empty one
        off = [0, 64, 64, 64 * 91, 64 * 93, 64 * 100]
        assert 2 <= hip_delta.Segments(off, "cpu").run_chunks(code, 1, 64, 64) < 90
        assert hip_delta.Segments([0, 5], "cpu").run_chunks(code, 1, 64, 64) == 1
        assert hip_delta.Segments([0, 0], "cpu").run_chunks(code, 1, 64, 64) == 1


def test_oracle_is_the_plain_rule():
    """One token by hand, and decays and writes of nothing."""
    torch.manual_seed(0)
    q, k, v, la, b = (torch.randn(s, dtype=torch.float64) for s in
                      ((1, 1, 3), (1, 1, 3), (1, 1, 2), (1, 1), (1, 1)))
    S = torch.randn(1, 3, 2, dtype=torch.float64)
    a = la.exp().item()
    S1 = a * S[0]
    want = S1 + torch.outer(k[0, 0], b.item() * (v[0, 0] - S1.T @ k[0, 0]))
    o, got = O.delta_scan(q, k, v, la, b, scale=2.0, state=S)
    assert torch.allclose(got[0], want) and torch.allclose(o[0, 0], 2 * want.T @ q[0, 0])
    o, got = O.delta_scan(q, k, v, la * 0, b * 0, state=S)
    assert torch.equal(got, S)
