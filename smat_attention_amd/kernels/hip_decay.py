"""The kernels of linear attention with a decay for each head (csrc/decay*) behind their
Python checks.

``scan`` runs a whole-sequence forward, ``scan_backward`` its gradient, ``step`` one token;
:class:`HeadDecayFunction` ties the first two into autograd.  As in :mod:`.hip_fwd`, inputs
are borrowed, outputs and workspaces come from torch's caching allocator, work goes to torch's
current stream of the inputs' device, and every failure raises.
:mod:`smat_attention_amd.attention` has the public entry points.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import DTYPE_CODE, ptr
from .hip_delta import CHUNK, _near_rows, same_device
from .hip_fwd import _call_on, _code, _shape

MAX_D = 128
MIN_D = 8                # rows are read eight values at a time (kMinD)
_RUNS = "smat_head_decay_run_chunks"


class _Plan:
    """One call's geometry: its sizes and table addresses in the C entry points' order."""

    def __init__(self, who, Q, V, heads, segments):
        self.nbk, self.T, self.r = Q.shape
        self.nb, _, self.p = V.shape
        self.heads = heads
        if segments is None:
            self.nseg, self.nch = 1, -(-self.T // CHUNK)
        else:
            if segments.T != self.T:
                raise ValueError(f"{who}: segments end at {segments.T}, the inputs at {self.T}")
            if segments.device != Q.device:
                raise ValueError(f"{who}: segments are on {segments.device}, the inputs on "
                                 f"{Q.device}")
            self.nseg, self.nch = len(segments), segments.nch
        code = _code(Q, who)
        if segments is not None:
            self.K = segments.run_chunks(code, self.nb, self.r, self.p, _RUNS)
            runs, segrun = segments.runs(self.K)
            self.tables = (segments.chunks.data_ptr(), runs.data_ptr(), segrun.data_ptr())
            self.nruns = runs.shape[0]
        else:
            self.K = 1 if self.nch <= 1 else _lib.query(_RUNS, code, self.nb, self.nch, None, None,
                                                        0, self.r, self.p)
            self.tables = (None, None, None)
            self.nruns = max(1, -(-self.nch // self.K))

    def sizes(self, scale):
        return (*self.tables, self.nb, max(self.nbk, 1), self.heads, self.T, self.nseg, self.nch,
                self.nruns, self.K, self.r, self.p, float(scale))

    def workspace(self, backward, learn, device):
        if not backward and self.nruns == self.nseg:   # a forward without cuts needs none
            return None, 0
        n = _lib.query("smat_head_decay_workspace_bytes", self.nb, max(self.nbk, 1), self.T,
                       self.nseg, self.nruns, self.r, self.p, backward, learn)
        return (torch.empty(n, device=device, dtype=torch.uint8) if n else None), n


def check_scan(who, Q, K, V, logA, state, segments):
    """The argument checks of the whole-sequence form (those that word the errors are called
    only when one fails: a short call is a launch of some ten microseconds)."""
    dt, dev = Q.dtype, Q.device
    if (segments is None and Q.is_cuda and dev == K.device and dev == V.device
            and dev == logA.device and K.dtype == dt and V.dtype == dt and dt in DTYPE_CODE
            and logA.dtype == torch.float32 and Q.dim() == 3 and V.dim() == 3 and logA.dim() == 1
            and K.shape == Q.shape):
        (nbk, T, r), (nb, Tv, p), heads = Q.shape, V.shape, logA.shape[0]
        if (T == Tv and T < 2 ** 30 and 0 < nbk <= nb < 2 ** 23 and nb % nbk == 0 and heads > 0
                and nb % heads == 0 and 1 <= r <= MAX_D and 1 <= p <= MAX_D
                and (state is None or state.device == dev and state.dtype == torch.float32
                     and state.shape == (nb, r, p))):
            return
    if Q.dim() != 3 or V.dim() != 3:
        raise ValueError(f"{who}: Q, K and V must be (sequences, T, columns)")
    same_device(who, Q, K, V, logA, state)
    nbk, T, r = Q.shape
    nb, _, p = V.shape
    _shape(who, "K", K, (nbk, T, r))
    _shape(who, "V", V, (nb, T, p))
    if T > 2 ** 31 - CHUNK or nb >= 2 ** 23:
        raise ValueError(f"{who}: {T} tokens of {nb} sequences, at most 2^31 - {CHUNK} and "
                         f"2^23 - 1")
    check_sizes(who, nbk, nb, logA, r, p)
    check_types(who, Q, K, V, logA, state)
    if state is not None:
        _shape(who, "state", state, (nb, r, p) if segments is None else
               (len(segments), nb, r, p))


def check_sizes(who, nbk, nb, logA, r, p):
    if (nbk == 0) != (nb == 0) or (nbk and nb % nbk):
        raise ValueError(f"{who}: {nbk} key sequences do not divide {nb} value sequences")
    if logA.dim() != 1 or not logA.shape[0] or nb % logA.shape[0]:
        raise ValueError(f"{who}: logA must be (heads,) with heads dividing the {nb} value "
                         f"sequences, got {tuple(logA.shape)}")
    if not (1 <= r <= MAX_D and 1 <= p <= MAX_D):
        raise ValueError(f"{who}: key size {r} and value size {p} must lie in 1..{MAX_D}")


def check_types(who, Q, K, V, logA, state):
    _code(Q, who)
    if K.dtype != Q.dtype or V.dtype != Q.dtype:
        raise TypeError(f"{who}: Q, K and V must share a dtype, got {Q.dtype}, {K.dtype} and "
                        f"{V.dtype}")
    if logA.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError(f"{who}: logA must be float32, bfloat16 or float16, got {logA.dtype}")
    if state is not None and state.dtype != torch.float32:
        raise TypeError(f"{who}: the state is held in float32, got {state.dtype}")


def scan(Q, K, V, logA, state, scale, segments, want_state: bool, save: bool, learn: bool):
    """``(o, state_out or None, kept, inputs)``: the forward over checked arguments; ``kept`` is
    what the backward takes from it (the states entering the runs and, to learn the decays,
    those entering the chunks), ``inputs`` are the tensors that the kernels read."""
    plan = _Plan("head_decay_scan", Q, V, logA.shape[0], segments)
    code, dev = _code(Q, "head_decay_scan"), Q.device
    (Q, q_sb, q_st), (K, k_sb, k_st), (V, v_sb, v_st) = map(_near_rows, (Q, K, V))
    logA = logA.float().contiguous()
    o = torch.empty(plan.nb, plan.T, plan.p, device=dev, dtype=V.dtype)
    lead = () if segments is None else (plan.nseg,)
    f32 = dict(device=dev, dtype=torch.float32)
    s_out = torch.empty(*lead, plan.nb, plan.r, plan.p, **f32) if want_state else None
    if state is not None:
        state = state.contiguous()
    start = chunk_states = None
    if save and plan.nruns > plan.nseg:
        start = torch.empty(plan.nruns, plan.nb, plan.r, plan.p, **f32)
    if save and learn:
        R, P = -(-plan.r // 32) * 32, 64 if plan.p <= 64 else 128
        chunk_states = torch.empty(plan.nb, plan.nch, P, R, **f32)
    ws, n = plan.workspace(0, 0, dev)
    _call_on(Q, "smat_head_decay_scan", code, Q.data_ptr(), K.data_ptr(), V.data_ptr(),
             logA.data_ptr(), ptr(state) or None, o.data_ptr(), ptr(s_out) or None,
             ptr(start) or None, ptr(chunk_states) or None, *plan.sizes(scale), q_sb, q_st, k_sb,
             k_st, v_sb, v_st, ptr(ws) or None, n)
    return o, s_out, (state if start is None else start, chunk_states), (Q, K, V, logA)


def scan_backward(inputs, kept, dO, dS, scale, segments, want_dstate: bool, learn: bool):
    """``(dQ, dK, dV, dlogA or None, dstate or None)`` of one forward."""
    Q, K, V, logA = inputs
    start, chunk_states = kept
    plan = _Plan("head_decay_scan", Q, V, logA.shape[0], segments)
    code, dev = _code(Q, "head_decay_scan"), Q.device
    (_, q_sb, q_st), (_, k_sb, k_st), (_, v_sb, v_st) = map(_near_rows, (Q, K, V))
    dO, d_sb, d_st = _near_rows(dO)
    dQ = torch.empty(plan.nbk, plan.T, plan.r, device=dev, dtype=Q.dtype)
    dK = torch.empty_like(dQ)
    dV = torch.empty(plan.nb, plan.T, plan.p, device=dev, dtype=V.dtype)
    lead = () if segments is None else (plan.nseg,)
    dstate = (torch.empty(*lead, plan.nb, plan.r, plan.p, device=dev, dtype=torch.float32)
              if want_dstate else None)
    dlogA = None
    if learn:
        dlogA = (torch.empty if plan.nb else torch.zeros)(logA.shape[0], device=dev,
                                                          dtype=torch.float32)
    ws, n = plan.workspace(1, int(learn), dev)
    if dS is not None:
        dS = dS.contiguous()
    _call_on(Q, "smat_head_decay_scan_backward", code, Q.data_ptr(), K.data_ptr(), V.data_ptr(),
             logA.data_ptr(), dO.data_ptr(), ptr(dS) or None, ptr(start) or None,
             ptr(chunk_states) or None, dQ.data_ptr(), dK.data_ptr(), dV.data_ptr(),
             ptr(dstate) or None, ptr(dlogA) or None, *plan.sizes(scale), q_sb, q_st, k_sb, k_st,
             v_sb, v_st, d_sb, d_st, ptr(ws) or None, n)
    return dQ, dK, dV, dlogA, dstate


class HeadDecayFunction(torch.autograd.Function):
    """The whole-sequence form with gradients of Q, K, V, logA and the state.

    The forward keeps its inputs and, where the sequences are split along T, the states
    entering the runs; the decays' gradient also needs those entering the chunks."""

    @staticmethod
    def forward(ctx, Q, K, V, logA, state, scale, segments, want_state):
        learn = ctx.needs_input_grad[3]
        o, s_out, kept, inputs = scan(Q, K, V, logA, state, scale, segments, want_state, True,
                                      learn)
        ctx.save_for_backward(*inputs, *kept)
        ctx.meta = (scale, segments, logA.dtype, learn)
        ctx.set_materialize_grads(False)
        return o, s_out

    @staticmethod
    @once_differentiable
    def backward(ctx, dO, dS):
        saved = ctx.saved_tensors
        inputs, kept = saved[:4], saved[4:]
        scale, segments, a_type, learn = ctx.meta
        if dO is None and dS is None:
            return (None,) * 8
        V = inputs[2]
        if dO is None:
            dO = torch.zeros(V.shape, device=V.device, dtype=V.dtype)
        dQ, dK, dV, dlogA, dstate = scan_backward(inputs, kept, dO.to(V.dtype), dS, scale,
                                                  segments, ctx.needs_input_grad[4], learn)
        return (dQ, dK, dV, None if dlogA is None else dlogA.to(a_type), dstate, None, None, None)


def step(q, k, v, logA, state, scale, out, out_state):
    """One token (the checks are in place and the helpers that word the errors are called only
    when one fails: a step is a launch of a few microseconds)."""
    who = "head_decay_step"
    if q.dim() != 2 or v.dim() != 2 or state.dim() != 3:
        raise ValueError(f"{who}: q, k and v must be (sequences, columns), the state "
                         f"(sequences, r, p)")
    nbk, r = q.shape
    nb, p = v.shape
    dev, dt = state.device, q.dtype
    if out_state is None:
        out_state = state
    if out is None:
        out = torch.empty(nb, p, device=dev, dtype=v.dtype)
    if not (q.is_cuda and dev == q.device == k.device == v.device == logA.device == out.device
            == out_state.device):
        same_device(who, q, k, v, logA, state, out, out_state)
    rows = (nb, r, p)
    if not (k.shape == q.shape and state.shape == rows and out_state.shape == rows
            and out.shape == v.shape):
        _shape(who, "k", k, (nbk, r))
        _shape(who, "state", state, rows)
        _shape(who, "out_state", out_state, rows)
        _shape(who, "out", out, (nb, p))
    if (nbk == 0 or nb % nbk or logA.dim() != 1 or not logA.shape[0] or nb % logA.shape[0]
            or r > MAX_D or p > MAX_D or r < 1 or p < 1):
        check_sizes(who, nbk, nb, logA, r, p)
    f32 = torch.float32
    if not (k.dtype == v.dtype == dt and logA.dtype == state.dtype == f32):
        check_types(who, q, k, v, logA, state)
        logA = logA.float()
    if out.dtype != dt or out_state.dtype != f32:
        raise TypeError(f"{who}: out must be {dt} and out_state float32, got {out.dtype} and "
                        f"{out_state.dtype}")
    if not (state.is_contiguous() and out_state.is_contiguous() and out.is_contiguous()
            and logA.is_contiguous()):
        raise ValueError(f"{who}: state, out_state, out and logA must be contiguous")
    if nb >= 2 ** 24:
        raise ValueError(f"{who}: {nb} sequences, at most 2^24 - 1")
    if out_state is not state and out_state.data_ptr() != state.data_ptr():
        lo, hi = sorted((state.data_ptr(), out_state.data_ptr()))
        if hi < lo + state.numel() * 4:
            raise ValueError(f"{who}: out_state must be state itself or lie apart from it")
    (q_sb, q_s1), (k_sb, k_s1), (v_sb, v_s1) = q.stride(), k.stride(), v.stride()
    if not ((q_s1 == 1 or r == 1) and (k_s1 == 1 or r == 1) and (v_s1 == 1 or p == 1)):
        raise ValueError(f"{who}: rows of q, k and v must be contiguous")
    _call_on(q, "smat_head_decay_step", _code(q, who), q.data_ptr(), k.data_ptr(), v.data_ptr(),
             logA.data_ptr(), state.data_ptr(), out_state.data_ptr(), out.data_ptr(), nb,
             max(nbk, 1), logA.shape[0], r, p, scale, q_sb, k_sb, v_sb)
    return out
