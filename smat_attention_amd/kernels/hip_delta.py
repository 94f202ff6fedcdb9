"""The gated delta rule's kernels (csrc/delta*.hip) behind their Python checks.

``scan`` runs a whole-sequence forward, ``scan_backward`` its gradient, ``step`` one
token; :class:`GatedDeltaFunction` ties the first two into autograd.  As in
:mod:`.hip_fwd`, inputs are borrowed, outputs and workspaces come from torch's caching
allocator, work goes to torch's current stream of the inputs' device, and every failure
raises.  :mod:`smat_attention_amd.attention` has the public entry points.
"""
from __future__ import annotations

import numpy as np
import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import ptr
from .hip_fwd import _call_on, _code, _on_gpu, _rows3, _shape

CHUNK = 64
MAX_R, MAX_P = 128, 256
FEW_TOKENS = 16          # calls of up to so many tokens, unpacked, need no workspace (kFewTokens)


def same_device(who: str, ref: torch.Tensor, *ts) -> None:
    _on_gpu(who, ref, *ts)
    for t in ts:
        if t is not None and t.device != ref.device:
            raise ValueError(f"{who}: tensors on {ref.device} and {t.device}")


class Segments:
    """Packed sequences: ``offsets`` = 0, ..., T are the borders of the segments along the
    token axis (as many as the list has entries, less one; empty ones are allowed).  Checked
    and staged on ``device`` once; a program keeps it as long as its batch keeps the layout.
    """

    def __init__(self, offsets, device):
        off = np.asarray(offsets.cpu() if isinstance(offsets, torch.Tensor) else offsets)
        if off.ndim != 1 or off.size < 2 or off.dtype.kind not in "iu":
            raise ValueError("Segments: offsets must be a list of at least two integers")
        off = off.astype(np.int64)
        if off[0] != 0 or np.any(np.diff(off) < 0):
            raise ValueError("Segments: offsets must start at 0 and not decrease")
        if off[-1] >= 2 ** 31:
            raise ValueError("Segments: at most 2^31 - 1 tokens")
        self.offsets = [int(x) for x in off]
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        counts = -(-np.diff(off) // CHUNK)                       # chunks of each segment
        first = np.concatenate([[0], np.cumsum(counts)])
        seg = np.repeat(np.arange(len(counts)), counts)
        t0 = off[:-1][seg] + (np.arange(first[-1]) - first[:-1][seg]) * CHUNK
        rows = np.stack([t0, np.minimum(CHUNK, off[1:][seg] - t0)], 1).astype(np.int32)
        self._first, self._counts = first, counts
        # one row at least, so that the table's address says that there is one
        self.chunks = torch.from_numpy(rows if len(rows) else
                                       np.zeros((1, 2), np.int32)).to(self.device)
        self.nch = int(first[-1])
        self._lengths, self._times = (np.ascontiguousarray(x, dtype=np.int32) for x in
                                      np.unique(counts, return_counts=True))
        self._runs, self._best = {}, {}

    def __len__(self):
        return len(self.offsets) - 1

    @property
    def T(self):
        return self.offsets[-1]

    def run_chunks(self, code: int, nb: int, r: int, p: int,
                   rule: str = "smat_delta_run_chunks") -> int:
        """The run length for inputs of these sizes, searched at the first call with them."""
        key = (rule, code, nb, r, p)
        if key not in self._best:
            self._best[key] = _lib.query(rule, code, nb, self.nch,
                                         self._lengths.ctypes.data, self._times.ctypes.data,
                                         len(self._lengths), r, p)
        return self._best[key]

    def runs(self, K: int):
        """``(runs, segrun)`` on the device for runs of ``K`` chunks; staged at the first call
        with that K (outside a graph capture)."""
        if K not in self._runs:
            if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("Segments: the first call with inputs of these sizes stages a "
                                   "table and cannot be captured; make one before")
            rows, segrun = [], [0]
            for s, n in enumerate(self._counts):
                c0 = int(self._first[s])
                for a in range(0, max(int(n), 1), K):
                    rows.append((c0 + a, c0 + min(a + K, int(n)), s))
                segrun.append(len(rows))
            rows = np.array(rows)
            turns = np.argsort(rows[:, 0] - rows[:, 1], kind="stable")    # the longest first
            rows = np.concatenate([rows, turns[:, None]], 1)
            self._runs[K] = tuple(torch.from_numpy(np.asarray(x, np.int32)).to(self.device)
                                  for x in (rows, segrun))
        return self._runs[K]


def _near_rows(t):
    """``_rows3``, with rows that lie 2^23 elements and more apart copied together: the kernels
    reach the rows of a chunk by 32-bit offsets.  A single row's stride is anything (torch
    ignores it, in ``contiguous`` too) and means nothing: it becomes the row's length."""
    if t.shape[1] <= 1:
        t, sb, _ = _rows3(t)
        return t, sb, t.shape[2]
    return _rows3(t if t.stride(1) < 2 ** 23 else t.contiguous())


class _Plan:
    """One call's geometry: its sizes and table addresses in the C entry points' order."""

    def __init__(self, who, Q, V, segments):
        self.nbk, self.T, self.r = Q.shape
        self.nb, _, self.p = V.shape
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
            self.K = segments.run_chunks(code, self.nb, self.r, self.p)
        elif self.nch <= 1:
            self.K = 1
        else:
            self.K = _lib.query("smat_delta_run_chunks", code, self.nb, self.nch, None, None, 0,
                                self.r, self.p)
        if segments is None:
            self.tables = (None, None, None)
            self.nruns = max(1, -(-self.nch // self.K))
        else:
            runs, segrun = segments.runs(self.K)
            self.tables = (segments.chunks.data_ptr(), runs.data_ptr(), segrun.data_ptr())
            self.nruns = runs.shape[0]
        self.R, self.P = -(-self.r // 32) * 32, -(-self.p // 32) * 32

    def sizes(self, scale):
        return (*self.tables, self.nb, max(self.nbk, 1), self.T, self.nseg, self.nch, self.nruns,
                self.K, self.r, self.p, float(scale))

    def workspace(self, code, backward, device):
        n = _lib.query("smat_delta_workspace_bytes", code, self.nb, self.nbk, self.nch, self.nseg,
                       self.nruns, self.r, self.p, backward)
        return torch.empty(max(n, 1), device=device, dtype=torch.uint8), n


def check_scan(who, Q, K, V, logA, beta, state, segments):
    """The argument checks of the whole-sequence form."""
    if Q.dim() != 3 or V.dim() != 3:
        raise ValueError(f"{who}: Q, K and V must be (sequences, T, columns)")
    dev = Q.device
    if not (Q.is_cuda and dev == K.device == V.device == logA.device == beta.device
            and (state is None or state.device == dev)):
        same_device(who, Q, K, V, logA, beta, state)
    nbk, T, r = Q.shape
    nb, _, p = V.shape
    if not (K.shape == Q.shape and V.shape[1] == T and logA.shape == beta.shape == (nb, T)):
        _shape(who, "K", K, (nbk, T, r))
        _shape(who, "V", V, (nb, T, p))
        _shape(who, "logA", logA, (nb, T))
        _shape(who, "beta", beta, (nb, T))
    if (nbk == 0) != (nb == 0) or (nbk and nb % nbk):
        raise ValueError(f"{who}: {nbk} key sequences do not divide {nb} value sequences")
    if T >= 2 ** 31 or nb >= 2 ** 31:
        raise ValueError(f"{who}: {T} tokens of {nb} sequences, at most 2^31 - 1 each")
    _check_types(who, Q, K, V, logA, beta, state)
    _check_widths(who, r, p)
    if state is not None:
        _shape(who, "state", state, (nb, r, p) if segments is None else
               (len(segments), nb, r, p))


def _check_types(who, Q, K, V, logA, beta, state):
    _code(Q, who)
    if K.dtype != Q.dtype or V.dtype != Q.dtype:
        raise TypeError(f"{who}: Q, K and V must share a dtype, got {Q.dtype}, {K.dtype} and "
                        f"{V.dtype}")
    for name, t in (("logA", logA), ("beta", beta)):
        if t.dtype not in (torch.float32, torch.bfloat16, torch.float16):
            raise TypeError(f"{who}: {name} must be float32, bfloat16 or float16, got {t.dtype}")
    if state is not None and state.dtype != torch.float32:
        raise TypeError(f"{who}: the state is held in float32, got {state.dtype}")


def _check_widths(who, r, p):
    if not (1 <= r <= MAX_R and 1 <= p <= MAX_P):
        raise ValueError(f"{who}: key size {r} and value size {p} must lie in 1..{MAX_R} and "
                         f"1..{MAX_P}")


def scan(Q, K, V, logA, beta, state, scale, segments, want_state: bool, save: bool):
    """``(o, state_out or None, saved, inputs)``: the forward over checked arguments; ``saved``
    is what the backward takes from it, ``inputs`` are the tensors that the kernels read (rows
    with unit column stride, fp32 gates)."""
    who = "gated_delta_scan"
    plan = _Plan(who, Q, V, segments)
    code, dev = _code(Q, who), Q.device
    (Q, q_sb, q_st), (K, k_sb, k_st), (V, v_sb, v_st) = _rows3(Q), _rows3(K), _near_rows(V)
    logA, beta = logA.float(), beta.float()
    o = torch.empty(plan.nb, plan.T, plan.p, device=dev, dtype=V.dtype)
    lead = () if segments is None else (plan.nseg,)
    s_out = (torch.empty(*lead, plan.nb, plan.r, plan.p, device=dev, dtype=torch.float32)
             if want_state else None)
    save_s = save_u = save_m = None
    if save:
        save_s = torch.empty(plan.nb, plan.nch, plan.R, plan.P, device=dev)
        save_u = torch.empty(plan.nb, plan.nch, CHUNK, plan.P, device=dev)
        if plan.nruns > plan.nseg:
            save_m = torch.empty(plan.nruns, plan.nb, plan.R, plan.R, 3, device=dev,
                                 dtype=torch.bfloat16)
    ws = n = 0
    if save or segments is not None or plan.T > FEW_TOKENS:
        buf, n = plan.workspace(code, 0, dev)
        ws = buf.data_ptr()
    if state is not None:
        state = state.contiguous()
    _call_on(Q, "smat_delta_scan", code, Q.data_ptr(), K.data_ptr(), V.data_ptr(),
             logA.data_ptr(), beta.data_ptr(), ptr(state) or None, o.data_ptr(),
             ptr(s_out) or None, ptr(save_s) or None, ptr(save_u) or None, ptr(save_m) or None,
             *plan.sizes(scale), q_sb, q_st, k_sb, k_st, v_sb, v_st, *logA.stride(),
             *beta.stride(), ws, n)
    return o, s_out, (save_s, save_u, save_m), (Q, K, V, logA, beta)


def scan_backward(inputs, saved, dO, dS, scale, segments, want_dstate: bool):
    """``(dQ, dK, dV, dlogA, dbeta, dstate or None)`` of one forward."""
    who = "gated_delta_scan"
    Q, K, V, logA, beta = inputs
    save_s, save_u, save_m = saved
    plan = _Plan(who, Q, V, segments)
    code, dev = _code(Q, who), Q.device
    (_, q_sb, q_st), (_, k_sb, k_st), (_, v_sb, v_st) = _rows3(Q), _rows3(K), _near_rows(V)
    dO, d_sb, d_st = _near_rows(dO)
    dQ = torch.empty(plan.nbk, plan.T, plan.r, device=dev, dtype=Q.dtype)
    dK = torch.empty_like(dQ)
    dV = torch.empty(plan.nb, plan.T, plan.p, device=dev, dtype=V.dtype)
    dlogA = torch.empty(plan.nb, plan.T, device=dev, dtype=torch.float32)
    dbeta = torch.empty_like(dlogA)
    lead = () if segments is None else (plan.nseg,)
    dstate = (torch.empty(*lead, plan.nb, plan.r, plan.p, device=dev, dtype=torch.float32)
              if want_dstate else None)
    ws, n = plan.workspace(code, 1, dev)
    if dS is not None:
        dS = dS.contiguous()
    _call_on(Q, "smat_delta_scan_backward", code, Q.data_ptr(), K.data_ptr(), V.data_ptr(),
             logA.data_ptr(), beta.data_ptr(), dO.data_ptr(), ptr(dS), save_s.data_ptr(),
             save_u.data_ptr(), ptr(save_m) or None, dQ.data_ptr(), dK.data_ptr(), dV.data_ptr(),
             dlogA.data_ptr(), dbeta.data_ptr(), ptr(dstate), *plan.sizes(scale), q_sb, q_st, k_sb, k_st, v_sb,
             v_st, *logA.stride(), *beta.stride(), d_sb, d_st, ws.data_ptr(), n)
    return dQ, dK, dV, dlogA, dbeta, dstate


class GatedDeltaFunction(torch.autograd.Function):
    """The whole-sequence form with gradients of Q, K, V, logA, beta and the state.

    The forward keeps, besides its inputs, the state entering every chunk of 64 tokens and
    the chunk's ``U`` in fp32, and the transitions of the runs where T is split; the backward
    forms the chunks' other operands again."""

    @staticmethod
    def forward(ctx, Q, K, V, logA, beta, state, scale, segments, want_state):
        o, s_out, saved, inputs = scan(
            Q.detach(), K.detach(), V.detach(), logA.detach(), beta.detach(),
            None if state is None else state.detach(), scale, segments, want_state, True)
        ctx.save_for_backward(*inputs, *saved)
        ctx.meta = (scale, segments, logA.dtype, beta.dtype)
        ctx.set_materialize_grads(False)
        return o, s_out

    @staticmethod
    @once_differentiable
    def backward(ctx, dO, dS):
        inputs, saved = ctx.saved_tensors[:5], ctx.saved_tensors[5:]
        scale, segments, a_type, b_type = ctx.meta
        if dO is None and dS is None:
            return (None,) * 9
        if dO is None:
            V = inputs[2]
            dO = torch.zeros(V.shape, device=V.device, dtype=V.dtype)
        dQ, dK, dV, dlogA, dbeta, dstate = scan_backward(
            inputs, saved, dO.to(inputs[2].dtype), dS, scale, segments, ctx.needs_input_grad[5])
        return (dQ, dK, dV, dlogA.to(a_type), dbeta.to(b_type), dstate, None, None, None)


def step(q, k, v, logA, beta, state, scale, out, out_state):
    """One token (the checks are in place and the helpers that word the errors are called only
    when one fails: a step is a launch of a few microseconds)."""
    who = "gated_delta_step"
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
    if not (q.is_cuda and dev == q.device == k.device == v.device == logA.device == beta.device
            == out.device == out_state.device):
        same_device(who, q, k, v, logA, beta, state, out, out_state)
    rows = (nb, r, p)
    if not (k.shape == q.shape and logA.shape == beta.shape == (nb,) and state.shape == rows
            and out_state.shape == rows and out.shape == v.shape):
        _shape(who, "k", k, (nbk, r))
        _shape(who, "logA", logA, (nb,))
        _shape(who, "beta", beta, (nb,))
        _shape(who, "state", state, rows)
        _shape(who, "out_state", out_state, rows)
        _shape(who, "out", out, (nb, p))
    if (nbk == 0) != (nb == 0) or (nbk and nb % nbk):
        raise ValueError(f"{who}: {nbk} key sequences do not divide {nb} value sequences")
    f32 = torch.float32
    if not (k.dtype == v.dtype == dt and logA.dtype == beta.dtype == state.dtype == f32):
        _check_types(who, q, k, v, logA, beta, state)
        logA, beta = logA.float(), beta.float()
    if out.dtype != dt or out_state.dtype != f32:
        raise TypeError(f"{who}: out must be {dt} and out_state float32, got {out.dtype} and "
                        f"{out_state.dtype}")
    if not (state.is_contiguous() and out_state.is_contiguous() and out.is_contiguous()):
        raise ValueError(f"{who}: state, out_state and out must be contiguous")
    if r > MAX_R or p > MAX_P or r < 1 or p < 1 or nb >= 2 ** 24:
        _check_widths(who, r, p)
        raise ValueError(f"{who}: {nb} sequences, at most 2^24 - 1")
    if out_state is not state and out_state.data_ptr() != state.data_ptr():
        lo, hi = sorted((state.data_ptr(), out_state.data_ptr()))
        if hi < lo + state.numel() * 4:
            raise ValueError(f"{who}: out_state must be state itself or lie apart from it")
    (q_sb, q_s1), (k_sb, k_s1), (v_sb, v_s1) = q.stride(), k.stride(), v.stride()
    if not ((q_s1 == 1 or r == 1) and (k_s1 == 1 or r == 1) and (v_s1 == 1 or p == 1)):
        raise ValueError(f"{who}: rows of q, k and v must be contiguous")
    args = (_code(q, who), q.data_ptr(), k.data_ptr(), v.data_ptr(), logA.data_ptr(),
            beta.data_ptr(), state.data_ptr(), out_state.data_ptr(), out.data_ptr(), nb,
            max(nbk, 1), r, p, scale, q_sb, k_sb, v_sb, logA.stride(0), beta.stride(0))
    _call_on(q, "smat_delta_step", *args)
    return out
