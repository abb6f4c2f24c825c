"""Gated linear recurrence (SSRU): argument checks, the autograd wrapper of
the HIP kernels and the plain composite used off the GPU.

ref: src/rnn/cells.h SSRU (f = sigmoid(Wf x + bf), highway(cell, W x, f)).
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import hip_ext

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
_ACTS = ("none", "relu")


def check_scan(what, x, gate, state, lens, act, dims):
    """Shared refusals; dims is x's number of dimensions."""
    if x.dim() != dims:
        raise ValueError(f"{what}: x must have {dims} dimensions, got "
                         f"{tuple(x.shape)}")
    if gate.shape != x.shape:
        raise ValueError(f"{what}: gate {tuple(gate.shape)} must have x's "
                         f"shape {tuple(x.shape)}")
    if gate.dtype != x.dtype or gate.device != x.device:
        raise ValueError(f"{what}: x and gate must share dtype and device")
    if x.shape[-1] == 0:
        raise ValueError(f"{what}: the width must be positive")
    ok = _DTYPES if x.is_cuda else _DTYPES + (torch.float64,)
    if x.dtype not in ok:
        raise ValueError(f"{what}: unsupported dtype {x.dtype}")
    if act not in _ACTS:
        raise ValueError(f"{what}: act must be one of {_ACTS}, got {act!r}")
    sdt = torch.float64 if x.dtype == torch.float64 else torch.float32
    if state is not None and (
            state.shape != (x.shape[0], x.shape[-1]) or state.dtype != sdt
            or state.device != x.device):
        raise ValueError(f"{what}: state must be {sdt} "
                         f"{(x.shape[0], x.shape[-1])} on x's device")
    if lens is not None and (
            lens.shape != (x.shape[0],) or lens.dtype != torch.int32
            or lens.device != x.device):
        raise ValueError(f"{what}: lens must be int32 {(x.shape[0],)} on x's "
                         "device")


def dense_rows(t):
    """t, or a copy of it if its last dimension is not dense or its rows lie
    further apart than the kernels' offsets reach."""
    if t.stride(-1) != 1 and t.shape[-1] != 1:
        return t.contiguous()
    if t.dim() == 3 and t.shape[1] > 1 and t.stride(1) >= 1 << 26:
        return t.contiguous()
    return t


def gated_scan_torch(x, gate, state=None, lens=None, reverse=False,
                     act="none"):
    """The recurrence step by step in (at least) 32 bits."""
    B, T, D = x.shape
    acc = torch.float64 if x.dtype == torch.float64 else torch.float32
    xa, ga = x.to(acc), gate.to(acc)
    f, om = torch.sigmoid(ga), torch.sigmoid(-ga)
    c = state if state is not None else xa.new_zeros(B, D)
    ys = [None] * T
    for t in range(T - 1, -1, -1) if reverse else range(T):
        new = f[:, t] * c + om[:, t] * xa[:, t]
        out = torch.relu(new) if act == "relu" else new
        if lens is not None:
            on = (lens > t)[:, None]
            new = torch.where(on, new, c)
            out = torch.where(on, out, torch.zeros_like(out))
        c, ys[t] = new, out
    y = torch.stack(ys, dim=1) if T else om * xa
    return y.to(x.dtype), c


class GatedScanFn(torch.autograd.Function):
    """x and gate as two tensors."""

    @staticmethod
    def forward(ctx, x, gate, state, lens, reverse, act):
        return _forward(ctx, x, gate, (x, gate), state, lens, reverse, act)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dlast):
        x, gate = ctx.saved_tensors[:2]
        dx = torch.empty_like(x, memory_format=torch.contiguous_format)
        dg = torch.empty_like(gate, memory_format=torch.contiguous_format)
        ds = _backward(ctx, x, gate, dy, dlast, dx, dg, 2)
        return dx, dg, ds, None, None, None


class GatedScanXGFn(torch.autograd.Function):
    """x and gate as the halves of one fused projection: one buffer in, one
    gradient buffer out."""

    @staticmethod
    def forward(ctx, xg, state, lens, reverse, act):
        d = xg.shape[-1] // 2
        return _forward(ctx, xg[..., :d], xg[..., d:], (xg,), state, lens,
                        reverse, act)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dlast):
        xg = ctx.saved_tensors[0]
        d = xg.shape[-1] // 2
        dxg = torch.empty_like(xg, memory_format=torch.contiguous_format)
        ds = _backward(ctx, xg[..., :d], xg[..., d:], dy, dlast,
                       dxg[..., :d], dxg[..., d:], 1)
        return dxg, ds, None, None, None


def _forward(ctx, x, gate, saved, state, lens, reverse, act):
    want = any(ctx.needs_input_grad)
    y, last, bnd = hip_ext(required=True).gated_scan_fwd(
        x, gate, state, lens, reverse, act, want)
    if want:
        ctx.save_for_backward(*saved, state, lens, bnd)
        ctx.reverse, ctx.act = reverse, act
        ctx.want_dstate = state is not None and state.requires_grad
        ctx.set_materialize_grads(False)
    return y, last


def _backward(ctx, x, gate, dy, dlast, dx, dg, n):
    state, lens, bnd = ctx.saved_tensors[n:]
    ds = hip_ext(required=True).gated_scan_bwd(
        x, gate, state, lens, bnd, dy,
        None if dlast is None else dlast.contiguous(), ctx.reverse, ctx.act,
        dx, dg, ctx.want_dstate)
    return ds if ctx.want_dstate else None
