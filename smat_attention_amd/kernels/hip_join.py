"""The end of a block (csrc/join.hip) behind its Python checks: :class:`BlockJoinFunction` is
the forward with its gradient, ``forward`` the forward alone.
:mod:`smat_attention_amd.attention` has the public entry point.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import DTYPE_CODE, SMAT_F32, ptr
from .hip_delta import same_device
from .hip_fwd import _call_on, _code, _shape

MIN_D, MAX_D = 8, 8192
GATES = {"linear": 1, "sigmoid": 2, "silu": 3}
_WHO = "block_join"


class Options:
    """What a call has beside its tensors, in the C entry points' order."""

    def __init__(self, gate, gate_kind, scale, eps, dropout, salt):
        if gate_kind not in GATES:
            raise ValueError(f"{_WHO}: gate_kind must be one of {', '.join(GATES)}, got "
                             f"{gate_kind!r}")
        if not eps >= 0:
            raise ValueError(f"{_WHO}: eps must be >= 0, got {eps}")
        if not 0 <= dropout < 1:
            raise ValueError(f"{_WHO}: dropout must lie in [0, 1), got {dropout}")
        if not 0 <= salt < 2 ** 32:
            raise ValueError(f"{_WHO}: salt must lie in [0, 2^32), got {salt}")
        self.gate = 0 if gate is None else GATES[gate_kind]
        self.scale = 1.0 if isinstance(scale, torch.Tensor) else float(scale)
        self.eps, self.dropout, self.salt = float(eps), float(dropout), int(salt)

    def args(self):
        return self.gate, self.eps, self.scale, self.dropout, self.salt


def check(f, h, gate, post, scale, pre, dropout, seed):
    vector = scale if isinstance(scale, torch.Tensor) else None
    if dropout and not isinstance(seed, torch.Tensor):
        raise ValueError(f"{_WHO}: dropout needs a seed, an int64 tensor of one element on the GPU")
    same_device(_WHO, f, h, gate, post, vector, pre, seed if dropout else None)
    if f.dim() < 1:
        raise ValueError(f"{_WHO}: f must be (..., columns)")
    _shape(_WHO, "h", h, tuple(f.shape))
    D = f.shape[-1]
    if not MIN_D <= D <= MAX_D:
        raise ValueError(f"{_WHO}: {D} columns must lie in {MIN_D}..{MAX_D}")
    if f.numel() // D >= 2 ** 31:
        raise ValueError(f"{_WHO}: {f.numel() // D} rows, at most 2^31 - 1")
    _code(f, _WHO)
    if h.dtype not in (f.dtype, torch.float32):
        raise TypeError(f"{_WHO}: h must be {f.dtype} or float32, got {h.dtype}")
    if gate is not None:
        _shape(_WHO, "gate", gate, tuple(f.shape))
        if gate.dtype != f.dtype:
            raise TypeError(f"{_WHO}: gate is {gate.dtype}, expected {f.dtype} as f")
    for name, w in (("post_weight", post), ("scale", vector), ("pre_weight", pre)):
        if w is not None:
            _shape(_WHO, name, w, (D,))
            _code(w, _WHO)
    if dropout:
        if seed.dtype != torch.int64 or seed.numel() != 1:
            raise ValueError(f"{_WHO}: seed must be an int64 tensor of one element, got "
                             f"{seed.dtype} {tuple(seed.shape)}")


def _rows(t, D):
    """``t`` as (rows, D) with unit column stride, and its row stride."""
    if t is None:
        return None, 0
    t = t.reshape(-1, D)
    if t.stride(1) != 1:
        t = t.contiguous()
    return t, t.stride(0)


def _weights(*ws):
    ws = [None if w is None else w.contiguous() for w in ws]
    return ws, ([ptr(w) or None for w in ws],
                [SMAT_F32 if w is None else DTYPE_CODE[w.dtype] for w in ws])


def forward(f, h, gate, post, vector, pre, seed, opt, keep):
    """``(h', x or None, (f, h, gate) rows, factors or None)`` over checked arguments."""
    D, shape = f.shape[-1], f.shape
    (f2, f_st), (h2, h_st), (z2, z_st) = _rows(f, D), _rows(h, D), _rows(gate, D)
    _, (wp, wt) = _weights(post, vector, pre)
    rows = f2.shape[0]
    out = torch.empty(shape, device=f.device, dtype=h.dtype)
    x = None if pre is None else torch.empty(shape, device=f.device, dtype=f.dtype)
    factors = torch.empty(rows + 1, 2, device=f.device, dtype=torch.float32) if keep else None
    _call_on(f, "smat_block_join", _code(f, _WHO), DTYPE_CODE[h.dtype], f2.data_ptr(),
             h2.data_ptr(), ptr(z2) or None, *wp, *wt, ptr(seed) or None, out.data_ptr(),
             ptr(x) or None, ptr(factors) or None, rows, D, *opt.args(), f_st, h_st, z_st)
    return out, x, factors


class BlockJoinFunction(torch.autograd.Function):
    """The block's end with gradients of f, h, the gate and the three weights.  Keeps its inputs,
    two numbers a row and the seed's value (a program may step its seed before the backward)."""

    @staticmethod
    def forward(ctx, f, h, gate, post, vector, pre, seed, opt):
        out, x, factors = forward(f, h, gate, post, vector, pre, seed, opt, True)
        ctx.save_for_backward(f, h, gate, post, vector, pre, factors)
        ctx.opt = opt
        ctx.set_materialize_grads(False)
        return out, x

    @staticmethod
    @once_differentiable
    def backward(ctx, dh, dx):
        f, h, gate, post, vector, pre, factors = ctx.saved_tensors
        if dh is None and dx is None:
            return (None,) * 8
        D, shape, dev = f.shape[-1], f.shape, f.device
        (f2, f_st), (h2, h_st), (z2, z_st) = _rows(f, D), _rows(h, D), _rows(gate, D)
        (dh2, dh_st), (dx2, dx_st) = _rows(dh, D), _rows(dx, D)
        keep, (wp, wt) = _weights(post, vector, pre)
        df = torch.empty(shape, device=dev, dtype=f.dtype)
        dz = None if gate is None else torch.empty(shape, device=dev, dtype=f.dtype)
        dho = torch.empty(shape, device=dev, dtype=h.dtype)
        rows = f2.shape[0]
        make = torch.empty if rows else torch.zeros
        need = ctx.needs_input_grad
        sums = [make(D, device=dev, dtype=torch.float32) if w is not None and need[i] else None
                for i, w in ((3, post), (4, vector), (5, pre))]
        n = (_lib.query("smat_block_join_workspace_bytes", rows, D)
             if any(s is not None for s in sums) else 0)
        ws = torch.empty(n, device=dev, dtype=torch.uint8) if n else None
        _call_on(f, "smat_block_join_backward", _code(f, _WHO), DTYPE_CODE[h.dtype],
                 f2.data_ptr(), h2.data_ptr(), ptr(z2) or None, *wp, *wt, factors.data_ptr(),
                 ptr(dh2) or None, ptr(dx2) or None, df.data_ptr(),
                 dho.data_ptr(), ptr(dz) or None, *(ptr(s) or None for s in sums), rows, D,
                 *ctx.opt.args(), f_st, h_st, z_st, dh_st, dx_st, ptr(ws) or None, n)
        sums = [None if s is None else s.to(w.dtype) for s, w in zip(sums, keep)]
        return (df, dho, dz, *sums, None, None)
