"""Gated linear recurrence (SSRU) off the GPU: argument checks and the plain
composite. On the GPU the extension checks the same and runs the kernels.

ref: src/rnn/cells.h SSRU (f = sigmoid(Wf x + bf), highway(cell, W x, f)).
"""
from __future__ import annotations

import torch

_DTYPES = (torch.float32, torch.bfloat16, torch.float16, torch.float64)
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
    if not 0 < x.shape[-1] < 1 << 25:
        raise ValueError(f"{what}: the width must be 1..2^25-1, got "
                         f"{x.shape[-1]}")
    if x.dtype not in _DTYPES:
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


def check_untraced(what):
    if torch.jit.is_tracing():
        raise NotImplementedError(f"{what} cannot be traced: the trace would "
                                  "hold the number of steps")


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
    if c is state:      # no step: its value in memory of its own
        c = c.clone()
    return y.to(x.dtype), c
