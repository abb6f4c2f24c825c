"""The join of two transformer blocks (norm, gate, residual, next norm) off
the GPU: argument checks and the plain composite. On the GPU the extension
checks the same and runs the kernels.

ref: models/transformer.h preProcess/postProcess ('n', 'a') and the highway
functor (out = sigmoid(t) in1 + (1 - sigmoid(t)) in2).
"""
from __future__ import annotations

import torch

MAX_WIDTH = 16384
_DTYPES = (torch.float32, torch.bfloat16, torch.float16, torch.float64)


def check_join(x, res, gate, gate_kind, params, norm):
    """params: {name: tensor or None} of the four norm parameters."""
    if x.dim() < 1 or x.dtype not in _DTYPES:
        raise ValueError(f"block_norm: x must be [..., D] of {_DTYPES}, got "
                         f"{x.dtype} {tuple(x.shape)}")
    D = x.shape[-1]
    if not 0 < D <= MAX_WIDTH:
        raise ValueError(f"block_norm: the width must be 1..{MAX_WIDTH}, "
                         f"got {D}")
    if res is not None and (res.shape != x.shape or res.dtype != x.dtype
                            or res.device != x.device):
        raise ValueError("block_norm: res must have x's shape, dtype and "
                         "device")
    if norm not in ("layer", "rms"):
        raise ValueError(f"block_norm: norm must be layer or rms, got "
                         f"{norm!r}")
    if gate_kind not in ("scale", "highway"):
        raise ValueError("block_norm: gate_kind must be scale or highway, "
                         f"got {gate_kind!r}")
    if res is None and gate_kind == "highway":
        raise ValueError("block_norm: a highway needs res")
    vecs = {k: v for k, v in params.items() if v is not None}
    if gate is not None:
        if gate.dim() == 1 and gate.shape == (D,) and x.dim() > 1:
            vecs["gate"] = gate
        elif gate.shape != x.shape or gate.dtype != x.dtype \
                or gate.device != x.device:
            raise ValueError("block_norm: gate must be [D] or of x's shape "
                             f"and dtype, got {gate.dtype} "
                             f"{tuple(gate.shape)}")
    for side in ("post", "pre"):
        if params[side + "_bias"] is not None \
                and params[side + "_scale"] is None:
            raise ValueError(f"block_norm: {side}_bias needs {side}_scale")
    pdt = {v.dtype for v in vecs.values()}
    if len(pdt) > 1 or not pdt <= {x.dtype, torch.float32}:
        raise ValueError("block_norm: parameters must share one dtype, "
                         f"x's or float32, got {sorted(map(str, pdt))}")
    for k, v in vecs.items():
        if v.shape != (D,) or v.device != x.device:
            raise ValueError(f"block_norm: {k} must be [{D}] on x's device")


def _highway(u, r, g):
    return torch.sigmoid(-g) * r + torch.sigmoid(g) * u


class _Highway(torch.autograd.Function):
    """(1 - k) r + k u, k = sigmoid(g), whose gate's gradient is made of u - r:
    the sums of u ds and of r ds, which differentiating the formula gives,
    cancel where u and r have a common mean."""
    generate_vmap_rule = True

    @staticmethod
    def forward(u, r, g):
        return _highway(u, r, g)

    @staticmethod
    def setup_context(ctx, inputs, output):
        ctx.save_for_backward(*inputs)
        ctx.save_for_forward(*inputs)

    @staticmethod
    def backward(ctx, d):
        u, r, g = ctx.saved_tensors
        k, k1 = torch.sigmoid(g), torch.sigmoid(-g)
        return k * d, k1 * d, (k * k1 * ((u - r) * d)).sum_to_size(g.shape)

    @staticmethod
    def jvp(ctx, du, dr, dg):
        u, r, g = ctx.saved_tensors
        k, k1 = torch.sigmoid(g), torch.sigmoid(-g)
        out = torch.zeros_like(u)
        for coef, t in ((k, du), (k1, dr), (k * k1 * (u - r), dg)):
            out = out if t is None else out + coef * t
        return out


def block_norm_torch(x, res, gate=None, gate_kind="scale", res_scale=1.0,
                     post_scale=None, post_bias=None, pre_scale=None,
                     pre_bias=None, norm="layer", eps=1e-9):
    """The formulas in (at least) 32 bits."""
    acc = torch.float64 if x.dtype == torch.float64 else torch.float32

    def normed(v, scale, bias):
        if norm == "layer":
            v = v - v.mean(-1, keepdim=True)
        v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + eps)
        v = v * scale.to(acc)
        return v if bias is None else v + bias.to(acc)

    u, r = x.to(acc), 0.0 if res is None else res.to(acc) * res_scale
    if post_scale is not None:
        u = normed(u, post_scale, post_bias)
    if gate is None:
        s = r + u
    elif gate_kind == "scale":
        s = r + gate.to(acc) * u
    else:
        # a trace (model export) takes the formula's own ops
        highway = _highway if torch.jit.is_tracing() else _Highway.apply
        s = highway(u, r, gate.to(acc))
    h = None if pre_scale is None else normed(s, pre_scale, pre_bias).to(
        x.dtype)
    return s.to(x.dtype), h
