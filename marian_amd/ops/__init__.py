"""Compute ops with MI355X HIP fast paths.

Every hot op has two implementations:

- a hand-written HIP/CDNA4 kernel (marian_amd/ops/hip/, built for gfx950),
  used whenever the tensor lives on a ROCm device;
- a plain PyTorch composite, used on CPU (tests, the reference path for
  numerics checks).

On a GPU machine the HIP extension is REQUIRED: if a tensor is on device and
the extension failed to build/load, ops raise rather than silently falling
back (per-op opt-outs exist for A/B testing via ``use_hip(False)``).

ref: src/tensors/gpu/tensor_operators.cu (softmax/LN/CE kernels),
     src/tensors/gpu/prod.cpp (GEMM), src/translator/nth_element.cu (top-k).
"""
from __future__ import annotations

import os
from typing import Optional

import torch

_HIP_EXT = None
_HIP_TRIED = False
_HIP_ENABLED = True


def use_hip(flag: bool) -> None:
    global _HIP_ENABLED
    _HIP_ENABLED = flag


def hip_ext(required: bool = False):
    """Load the in-tree HIP extension (built by setup.py / __graft_entry__.build)."""
    global _HIP_EXT, _HIP_TRIED
    if _HIP_EXT is None and not _HIP_TRIED:
        _HIP_TRIED = True
        try:
            from . import _load
            _HIP_EXT = _load.load_extension()
        except Exception as e:  # pragma: no cover - GPU box only
            _HIP_EXT = None
            if required:
                raise RuntimeError(
                    f"marian_amd HIP extension failed to load: {e}") from e
    if required and _HIP_EXT is None:
        raise RuntimeError(
            "marian_amd HIP extension is not available on this GPU machine; "
            "build it with `python setup.py build_ext --inplace` "
            "(PYTORCH_ROCM_ARCH=gfx950)")
    return _HIP_EXT


def _on_gpu(t: torch.Tensor) -> bool:
    return t.is_cuda and _HIP_ENABLED


# ---------------------------------------------------------------------------
# Linear (GEMM + bias): addmm -> hipBLASLt epilogue; fp8 path for config #5
# ---------------------------------------------------------------------------

# BGRADB fused bias-grad: opt-in. Measured on MI355X the BGRADB-capable
# NT solution pool loses more on the dW GEMM than the fused reduce saves
# (B1024 transformer-big 585k -> 508k tok/s with it on everywhere).
_LT_BGRAD_OK = os.environ.get("MAMD_LT_BGRAD", "") == "1"


class _LtLinearFn(torch.autograd.Function):
    """Linear through direct hipBLASLt (ops/hip/ltgemm.cpp): forward GEMM
    with fused bias+ReLU epilogue (a separate ReLU pass costs a full
    read+write of the FFN activation). Backward runs TunableOp-tuned mm;
    ReLU backward uses the post-activation output (relu'(x) == [y > 0]),
    so the pre-activation is never materialized."""

    @staticmethod
    def forward(ctx, x2, W, b, relu):
        ext = hip_ext(required=True)
        y = ext.lt_linear_act(x2, W, b, relu)
        if relu:
            ctx.save_for_backward(x2, W, y)
        else:
            ctx.save_for_backward(x2, W)
        ctx.relu = relu
        return y

    @staticmethod
    def backward(ctx, dy):
        ext = hip_ext(required=True)
        if ctx.relu:
            x2, W, y = ctx.saved_tensors
            dyc = torch.ops.aten.threshold_backward(dy.contiguous(), y, 0)
        else:
            x2, W = ctx.saved_tensors
            dyc = dy.contiguous()
        dx = torch.mm(dyc, W.t() if W.stride(1) == 1 else W.t().contiguous())
        if _LT_BGRAD_OK:
            try:
                dWt, db = ext.lt_dwt_bgrad(x2, dyc, True)
                return dx, dWt.t(), db.to(dyc.dtype), None
            except RuntimeError:
                pass  # epilogue unsupported on this shape: torch fallback
        dW = torch.mm(x2.t(), dyc)  # TunableOp-tuned TN
        return dx, dW, dyc.sum(0), None


def _lt_ok(x, W, b) -> bool:
    return (b is not None and "MAMD_NO_LT" not in os.environ
            and x.dtype == torch.bfloat16 and W.dtype == torch.bfloat16
            and W.stride(1) == 1 and x.is_cuda)


def linear_act(x: torch.Tensor, W: torch.Tensor,
               b: Optional[torch.Tensor], act: str) -> torch.Tensor:
    """act(x @ W + b) with the activation fused into the GEMM epilogue
    where hipBLASLt supports it (relu)."""
    if act == "relu" and _lt_ok(x, W, b) and torch.is_grad_enabled()             and (x.requires_grad or W.requires_grad):
        x2 = x.reshape(-1, W.shape[0])
        shp = x.shape[:-1] + (W.shape[1],)
        return _LtLinearFn.apply(x2.contiguous(), W, b, True).view(shp)
    if act == "relu" and _lt_ok(x, W, b) and not torch.is_grad_enabled():
        ext = hip_ext(required=True)
        x2 = x.reshape(-1, W.shape[0]).contiguous()
        shp = x.shape[:-1] + (W.shape[1],)
        return ext.lt_linear_act(x2, W, b, True).view(shp)
    from ..models.layers import _ACT
    return _ACT[act](linear(x, W, b))


def _use_hand_wgrad(K: int, N: int, M: int) -> bool:
    """The hand-MFMA split-K wgrad (ops/hip/wgrad.hip) wins on the
    SMALL-output dW shapes where hipBLASLt cannot parallelize the
    M=B*T reduction (measured r2: [65536,1024]^T@[65536,1024] 551 vs
    431 TF/s, x2048 573 vs 516); on >=3072-wide outputs the library's
    bigger tiles win — keep torch there."""
    tiles = ((K + 127) // 128) * ((N + 127) // 128)
    return (M >= 4096 and K % 8 == 0 and N % 8 == 0 and tiles <= 128
            and "MAMD_NO_HAND_WGRAD" not in os.environ)


class _LinearFn(torch.autograd.Function):
    """addmm forward; backward routes the weight gradient through the
    hand-MFMA split-K kernel on the shapes where it beats hipBLASLt
    (see _use_hand_wgrad). With MAMD_CUSTOM_LINEAR=1 the bias gradient
    additionally uses the HIP column-sum kernel (a wash at NMT widths,
    kept for wider models)."""

    @staticmethod
    def forward(ctx, x2, W, b):
        ctx.save_for_backward(x2, W)
        ctx.has_bias = b is not None
        if b is None:
            return torch.mm(x2, W)
        return torch.addmm(b, x2, W)

    @staticmethod
    def backward(ctx, dy):
        x2, W = ctx.saved_tensors
        dyc = dy.contiguous()
        dx = torch.mm(dyc, W.t())
        db = None
        if x2.dtype == torch.bfloat16 and dyc.dtype == torch.bfloat16 \
                and _use_hand_wgrad(x2.shape[1], dyc.shape[1], x2.shape[0]):
            # db rides the wgrad kernel's dy reads: zero extra traffic
            dW, dbf = hip_ext(required=True).wgrad_bias_bf16(
                x2, dyc, 0, ctx.has_bias)
            if ctx.has_bias:
                db = dbf.to(dyc.dtype)
        else:
            dW = torch.mm(x2.t(), dyc)
        if ctx.has_bias and db is None:
            if "MAMD_CUSTOM_LINEAR" in os.environ:
                db = hip_ext(required=True).col_sum(dyc).to(dyc.dtype)
            else:
                db = dyc.sum(0)
        return dx, dW, db


def linear(x: torch.Tensor, W: torch.Tensor, b: Optional[torch.Tensor] = None
           ) -> torch.Tensor:
    """x [..., K] @ W [K, M] (+ b). On GPU with fp8 enabled, forward runs
    e4m3 scaled-mm (~2x bf16 MFMA rate)."""
    from .fp8 import fp8_enabled, fp8_linear
    if fp8_enabled() and x.is_cuda and x.dtype == torch.bfloat16:
        return fp8_linear(x, W.to(x.dtype), b.to(x.dtype) if b is not None else None)
    if not x.is_cuda:
        from .cpu_int8 import int8_enabled, int8_linear
        # fp32 weights only: .float() on other dtypes would allocate a
        # fresh tensor per call and defeat the packed-weight cache
        if int8_enabled() and W.dtype == torch.float32:
            y = int8_linear(x.float(), W,
                            b.float() if b is not None else None)
            if y is not None:
                return y.to(x.dtype)
    W = W.to(x.dtype)
    shp = x.shape[:-1] + (W.shape[1],)
    if _on_gpu(x) and torch.is_grad_enabled() \
            and (x.requires_grad or W.requires_grad) \
            and (("MAMD_CUSTOM_LINEAR" in os.environ)
                 or (x.dtype == torch.bfloat16 and _use_hand_wgrad(
                     W.shape[0], W.shape[1], x.numel() // W.shape[0]))):
        x2 = x.reshape(-1, W.shape[0])
        return _LinearFn.apply(x2, W.contiguous() if not W.is_contiguous()
                               and W.stride(0) != 1 else W,
                               b.to(x.dtype) if b is not None else None
                               ).view(shp)
    if b is None:
        return torch.matmul(x, W)
    return torch.addmm(b.to(x.dtype), x.reshape(-1, W.shape[0]), W).view(shp)


# ---------------------------------------------------------------------------
# LayerNorm  (ref kernels: gLNormalization / gLayerNormalizationGrad)
# ---------------------------------------------------------------------------

def layer_norm(x: torch.Tensor, scale: torch.Tensor, bias: torch.Tensor,
               eps: float = 1e-9) -> torch.Tensor:
    if _on_gpu(x):
        from ._layernorm import LayerNormFn
        return LayerNormFn.apply(x, scale, bias, eps)
    # normalized_shape from the WEIGHT (static at ONNX-trace time; using
    # x.shape[-1] traces as a dynamic Gather the LN symbolic rejects)
    return torch.nn.functional.layer_norm(
        x.float(), (scale.shape[-1],), scale.float(), bias.float(),
        eps).to(x.dtype)


def layer_norm_residual(x: torch.Tensor, res: torch.Tensor,
                        scale: torch.Tensor, bias: torch.Tensor,
                        eps: float = 1e-9) -> torch.Tensor:
    """LN(x + res) with the add fused into the LN kernel (the marian 'dan'
    postprocess epilogue)."""
    if _on_gpu(x) and x.shape == res.shape:
        from ._layernorm import LayerNormResFn
        return LayerNormResFn.apply(x.contiguous(), res.contiguous(),
                                    scale, bias, eps)
    return layer_norm(x + res, scale, bias, eps)


# ---------------------------------------------------------------------------
# The join of two transformer blocks (ref: transformer.h pre/postProcess)
# ---------------------------------------------------------------------------

def block_norm(x: torch.Tensor, res: Optional[torch.Tensor],
               gate: Optional[torch.Tensor] = None, gate_kind: str = "scale",
               res_scale: float = 1.0,
               post_scale: Optional[torch.Tensor] = None,
               post_bias: Optional[torch.Tensor] = None,
               pre_scale: Optional[torch.Tensor] = None,
               pre_bias: Optional[torch.Tensor] = None,
               norm: str = "layer", eps: float = 1e-9):
    """A block's output norm, gate and residual sum, and the norm before the
    next block; returns (s, h), h None without pre_scale.

        u = norm(x; post_scale, post_bias)   or x without post_scale
        s = res_scale * res + u                                 no gate
        s = res_scale * res + gate * u                          "scale"
        s = res_scale * (1 - k) * res + k * u, k = sigmoid(gate)  "highway"
        h = norm(s; pre_scale, pre_bias)

    norm: "layer" ((v - mean) / sqrt(var + eps)) or "rms" (v / sqrt(mean v^2
    + eps)), times scale, plus bias if there is one. x, res: [..., D], fp32 /
    bf16 / fp16, D <= 16384; without res its term is left out. gate: [D] (per
    channel) or x's shape (per token). Parameters are [D], all of x's dtype or all float32. h is taken
    from the 32-bit s; s and h are rounded once. Differentiable once in every
    tensor; on the GPU neither forward-mode derivatives nor traces are taken.
    """
    if _on_gpu(x):
        return hip_ext(required=True).block_norm(
            x, res, gate, gate_kind, res_scale, post_scale, post_bias,
            pre_scale, pre_bias, norm, eps)
    from ._block_norm import block_norm_torch, check_join
    check_join(x, res, gate, gate_kind,
               {"post_scale": post_scale, "post_bias": post_bias,
                "pre_scale": pre_scale, "pre_bias": pre_bias}, norm)
    return block_norm_torch(x, res, gate, gate_kind, res_scale, post_scale,
                            post_bias, pre_scale, pre_bias, norm, eps)


# ---------------------------------------------------------------------------
# Gated linear recurrence (ref: rnn/cells.h SSRU)
# ---------------------------------------------------------------------------

def gated_scan(x: torch.Tensor, gate: torch.Tensor,
               state: Optional[torch.Tensor] = None,
               lens: Optional[torch.Tensor] = None, reverse: bool = False,
               act: str = "none"):
    """Gated linear recurrence over sequences; returns (y, last).

        f_t = sigmoid(gate_t);  c_t = f_t c_{t-1} + (1 - f_t) x_t
        y_t = act(c_t)          act: "none" | "relu"

    x, gate: [B, T, D], fp32 / bf16 / fp16, D < 2^25, any batch and time
    strides (copied if the last dimension is not dense). state: float32 [B, D], the
    state before the first step (default zeros). lens: int32 [B]; the steps
    of row b are its first lens[b] positions (clamped to 0..T); what lies
    behind them is ignored, y is 0 there and so are its gradients.
    reverse: the steps run from position lens[b]-1 down to 0.
    y: [B, T, D] in x's dtype; last: float32 [B, D], the state after the last
    step (`state` itself for a row of no steps). States are held in 32 bits.
    Differentiable once in x, gate and state; on the GPU forward-mode
    derivatives are refused. Traces are refused everywhere: they would hold
    the outputs, or the number of steps.
    """
    if _on_gpu(x):
        return hip_ext(required=True).gated_scan(x, gate, state, lens,
                                                 reverse, act)
    from ._gated_scan import check_scan, check_untraced, gated_scan_torch
    check_untraced("gated_scan")
    check_scan("gated_scan", x, gate, state, lens, act, 3)
    return gated_scan_torch(x, gate, state, lens, reverse, act)


def gated_scan_xg(xg: torch.Tensor, state: Optional[torch.Tensor] = None,
                  lens: Optional[torch.Tensor] = None, reverse: bool = False,
                  act: str = "none"):
    """gated_scan on a fused projection xg [B, T, 2D], values first, gates
    second: read in place, and one gradient buffer comes out."""
    if _on_gpu(xg):
        return hip_ext(required=True).gated_scan_xg(xg, state, lens, reverse,
                                                    act)
    from ._gated_scan import check_scan, check_untraced, gated_scan_torch
    check_untraced("gated_scan_xg")
    if xg.dim() != 3 or xg.shape[-1] % 2:
        raise ValueError("gated_scan_xg: xg must be [B, T, 2D], got "
                         f"{tuple(xg.shape)}")
    d = xg.shape[-1] // 2
    x, gate = xg[..., :d], xg[..., d:]
    check_scan("gated_scan_xg", x, gate, state, lens, act, 3)
    return gated_scan_torch(x, gate, state, lens, reverse, act)


def gated_step(x: torch.Tensor, gate: torch.Tensor, state: torch.Tensor,
               act: str = "none", inplace: bool = False):
    """One step of gated_scan for each row; returns (y, new_state).

    x, gate: [N, D] (rows may be strided); state: float32 [N, D]. inplace
    writes the new state over `state` (which must be dense and share no
    memory with x or gate) and returns it, as a captured decode step needs;
    that call has no gradient. Otherwise a
    call that needs gradients runs as gated_scan over one position. On the GPU
    neither forward-mode derivatives nor traces are taken.
    """
    if _on_gpu(x):
        return hip_ext(required=True).gated_step(x, gate, state, act, inplace)
    from ._gated_scan import check_scan, gated_scan_torch
    if state is None:
        raise ValueError("gated_step: state is required")
    check_scan("gated_step", x, gate, state, None, act, 2)
    if inplace:
        if torch.is_grad_enabled() and (x.requires_grad or gate.requires_grad
                                        or state.requires_grad):
            raise ValueError("gated_step: inplace has no gradient")
        if not state.is_contiguous():
            raise ValueError("gated_step: inplace needs a dense state")
        own = state.untyped_storage()._cdata    # empty ones share address 0
        if own in (x.untyped_storage()._cdata, gate.untyped_storage()._cdata):
            raise ValueError("gated_step: inplace needs a state of its own "
                             "memory")
    y, new = gated_scan_torch(x[:, None], gate[:, None], state, act=act)
    return y[:, 0], state.copy_(new) if inplace else new


# ---------------------------------------------------------------------------
# Attention  (ref: composite ProdBatched+mask+gSoftmax+ProdBatched;
#             rebuilt as a fused flash-style CDNA4 kernel)
# ---------------------------------------------------------------------------

def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
              mask: Optional[torch.Tensor] = None,
              causal: bool = False, dropout_p: float = 0.0,
              lens: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Scaled dot-product attention.

    q: [B, H, Tq, Dh]; k/v: [B, H, Tk, Dh] (H may be 1 on k/v for MQA).
    mask: [B, 1, 1, Tk] or [B, 1, Tq, Tk] additive log-mask (0 / -inf).
    lens: optional int32 [B] prefix key lengths equivalent to mask (NMT
    masks are prefix masks); lets the fused kernel skip mask analysis.
    The 1/sqrt(Dh) scale is applied here.
    """
    if _on_gpu(q) and dropout_p == 0.0:
        from ._attention import fused_attention
        out = fused_attention(q, k, v, mask, causal, lens=lens)
        if out is not None:
            return out
        _warn_composite_attention(q)
    return attention_torch(q, k, v, mask, causal, dropout_p)


_warned_composite = False


def _warn_composite_attention(q: torch.Tensor):
    """the fused CDNA4 attention covers bf16/Dh=64 — every
    GPU BASELINE config (base 512/8, big+deep 1024/16). Any other head
    geometry silently compositing would misreport 'hand-written hot
    path', so say it LOUDLY once."""
    global _warned_composite
    if not _warned_composite and q.is_cuda:
        _warned_composite = True
        from ..common.logging_utils import log_info
        log_info("attention: fused HIP kernel NOT engaged "
                 f"(dtype={q.dtype}, Dh={q.shape[-1]}; fused path is "
                 "bf16/Dh=64) - running torch composite")


def attention_qkv(qkv: torch.Tensor, heads: int, mask=None, causal=False,
                  dropout_p: float = 0.0,
                  lens: Optional[torch.Tensor] = None):
    """Self-attention on the fused [B,T,3d] QKV projection (one buffer in,
    one buffer out in both directions). Returns [B,H,T,dh] or None for
    the composite fallback."""
    if dropout_p != 0.0 or not _on_gpu(qkv):
        return None
    from ._attention import fused_qkv_attention
    return fused_qkv_attention(qkv, heads, mask, causal, lens=lens)


def attention_kv(q2: torch.Tensor, kv: torch.Tensor, heads: int, mask=None,
                 dropout_p: float = 0.0,
                 lens: Optional[torch.Tensor] = None):
    """Cross-attention on fused projections q2 [B,Tq,d] / kv [B,Tk,2d];
    returns [B,H,Tq,dh] or None for the composite fallback."""
    if dropout_p != 0.0 or not _on_gpu(q2):
        return None
    from ._attention import fused_kv_attention
    return fused_kv_attention(q2, kv, heads, mask, lens=lens)


def attention_torch(q, k, v, mask=None, causal=False, dropout_p=0.0):
    scale = q.shape[-1] ** -0.5
    scores = torch.matmul(q, k.transpose(-1, -2)) * scale  # [B,H,Tq,Tk]
    if causal:
        Tq, Tk = scores.shape[-2], scores.shape[-1]
        cm = torch.ones(Tq, Tk, device=scores.device, dtype=torch.bool).tril(Tk - Tq)
        scores = scores.masked_fill(~cm, float("-inf"))
    if mask is not None:
        scores = scores + mask
    probs = torch.softmax(scores.float(), dim=-1).to(q.dtype)
    if dropout_p > 0.0:
        probs = torch.nn.functional.dropout(probs, dropout_p, training=True)
    return torch.matmul(probs, v)


# ---------------------------------------------------------------------------
# Softmax (row softmax with optional additive mask; ref: gSoftmax)
# ---------------------------------------------------------------------------

def softmax(x: torch.Tensor, dim: int = -1) -> torch.Tensor:
    if _on_gpu(x) and dim in (-1, x.dim() - 1):
        from ._softmax import SoftmaxFn
        return SoftmaxFn.apply(x)
    return torch.softmax(x.float(), dim=dim).to(x.dtype)


def log_softmax(x: torch.Tensor, dim: int = -1) -> torch.Tensor:
    if _on_gpu(x) and dim in (-1, x.dim() - 1):
        from ._softmax import LogSoftmaxFn
        return LogSoftmaxFn.apply(x)
    return torch.log_softmax(x.float(), dim=dim).to(x.dtype)


# ---------------------------------------------------------------------------
# Label-smoothed cross-entropy (ref: gCrossEntropyPick/-Backward)
# ---------------------------------------------------------------------------

def cross_entropy(logits: torch.Tensor, labels: torch.Tensor,
                  label_smoothing: float = 0.0,
                  mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Per-position CE with label smoothing; returns [N] float32 losses.

    logits: [N, V]; labels: [N] long; mask: [N] float (0 drops position).
    Smoothed loss = (1-eps)*nll(label) + eps * mean_v nll(v), matching the
    reference's label-smoothing formulation (layers/loss.cpp).
    """
    if _on_gpu(logits):
        from ._cross_entropy import CrossEntropyFn
        return CrossEntropyFn.apply(logits, labels, label_smoothing, mask)
    return cross_entropy_torch(logits, labels, label_smoothing, mask)


def cross_entropy_torch(logits, labels, label_smoothing=0.0, mask=None):
    lsm = torch.log_softmax(logits.float(), dim=-1)
    nll = -lsm.gather(-1, labels.unsqueeze(-1)).squeeze(-1)
    if label_smoothing > 0.0:
        smooth = -lsm.mean(dim=-1)
        loss = (1.0 - label_smoothing) * nll + label_smoothing * smooth
    else:
        loss = nll
    if mask is not None:
        loss = loss * mask.float()
    return loss


# ---------------------------------------------------------------------------
# Top-k for beam search (ref: translator/nth_element.cu NthElementGPU)
# ---------------------------------------------------------------------------

def topk(scores: torch.Tensor, k: int):
    """Row-wise top-k; scores [R, C] -> (values [R,k], indices [R,k])."""
    if _on_gpu(scores):
        ext = hip_ext()
        if ext is not None and hasattr(ext, "topk"):
            return ext.topk(scores.contiguous(), k)
    return torch.topk(scores, k, dim=-1)


# ---------------------------------------------------------------------------
# Fused Adam step (ref: the Element(...) Adam functor + castOptimizerType)
# ---------------------------------------------------------------------------

def grad_sumsq_finite(g: torch.Tensor) -> torch.Tensor:
    """Returns [2] fp32: (sum of squares, count of non-finite values) in
    ONE pass over the flat gradient (no fp32 temp, no g*g temp)."""
    if _on_gpu(g):
        return hip_ext(required=True).sumsq_finite(g.contiguous())
    gf = g.float()
    return torch.stack([(gf * gf).sum(),
                        (~torch.isfinite(gf)).sum().float()])


def adam_step(param32, grad, m, v, lr, beta1, beta2, eps, wd, step,
              grad_scale=1.0, lr_t=None, step_t=None):
    """One fused Adam update; grad is multiplied by grad_scale first
    (1/loss-scale x clip factor, folded in to avoid an extra pass).
    grad_scale may be a float OR a 0-dim fp32 device tensor (the async
    update path computes scaling/clipping on device, no host sync).
    lr_t/step_t: device-resident LR + step counter for hipGraph-replayed
    steps (bias correction computed in-kernel)."""
    if _on_gpu(param32):
        ext = hip_ext(required=True)
        gs_t = None
        gs = grad_scale
        if isinstance(grad_scale, torch.Tensor):
            gs_t = grad_scale.float().reshape(1)
            gs = 1.0
        ext.adam_step(param32, grad, m, v, lr, beta1, beta2, eps, wd,
                      step, gs, gs_t, lr_t, step_t)
        return
    # torch reference
    if lr_t is not None:
        lr = float(lr_t.reshape(-1)[0])
    if step_t is not None:
        step = int(step_t.reshape(-1)[0])
    g = grad.float()
    if isinstance(grad_scale, torch.Tensor) or grad_scale != 1.0:
        g = g * grad_scale
    m.mul_(beta1).add_(g, alpha=1 - beta1)
    v.mul_(beta2).addcmul_(g, g, value=1 - beta2)
    mh = m / (1 - beta1 ** step)
    vh = v / (1 - beta2 ** step)
    if wd:
        param32.mul_(1 - lr * wd)
    param32.addcdiv_(mh, vh.sqrt().add_(eps), value=-lr)
