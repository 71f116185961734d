"""Layer norm over the last dimension (``csrc/ops/norm.hip``), forward and backward.

    mu = mean_c x,  r = 1 / sqrt(mean_c (x - mu)^2 + eps),  y = (x - mu) r weight + bias

``layer_norm`` runs the HIP kernels for CUDA tensors and :func:`layer_norm_reference` otherwise.  ``x`` is bf16 or fp32,
of any shape; ``weight`` and ``bias`` [C] are each fp32, bf16 or absent, whatever the type of ``x`` (bf16 activations
with the learner's fp32 masters need no cast).  Statistics and sums are fp32, ``y`` and the gradients have the types of
``x``, ``weight`` and ``bias``; the parameter gradients are summed in a fixed order (bitwise reproducible).  Second
derivatives, forward-mode derivatives and traces without gradients are refused on the GPU.
"""
from __future__ import annotations

from typing import Optional

import torch

from gsc_amd.native import load as load_native
from .launch import check_device, check_forward_mode, check_leaves, check_not_traced, check_types, dense, differentiable_once, is_bf16, launch, ptr, raw_stream, rows_of


def layer_norm_reference(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                         eps: float = 1e-5) -> torch.Tensor:
    """The same function in elementary PyTorch operations (fp32 inside, or fp64 for fp64 inputs), differentiable."""
    xf = x if x.dtype == torch.float64 else x.float()
    mu = xf.mean(-1, keepdim=True)
    d = xf - (mu + (xf - mu).mean(-1, keepdim=True))   # the sum's rounding taken out: 0 in a row of equal values
    y = d * torch.rsqrt((d * d).mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight.to(xf.dtype)
    if bias is not None:
        y = y + bias.to(xf.dtype)
    return y.to(x.dtype)


def _forward(x2, weight, bias, eps, stats: bool):
    M, C = x2.shape
    y = torch.empty(M, C, device=x2.device, dtype=x2.dtype)
    st = torch.empty(2, M, device=x2.device, dtype=torch.float32) if stats else None
    if M > 0:
        s0 = ptr(st)
        launch(load_native().layer_norm_forward, x2, x2.data_ptr(), x2.stride(0), is_bf16(x2), ptr(weight), is_bf16(weight),
               ptr(bias), is_bf16(bias), y.data_ptr(), s0, s0 + 4 * M if stats else 0, M, C, eps)
    return y, st


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        x2 = rows_of(x, x.shape[-1])
        weight, bias = dense(weight), dense(bias)
        y, st = _forward(x2, weight, bias, eps, True)
        ctx.save_for_backward(x2, weight)
        (M, C), need = x2.shape, ctx.needs_input_grad
        wt, bt = weight.dtype if need[1] else None, bias.dtype if need[2] else None
        ctx.stats, ctx.shape, ctx.types, ctx.dev, ctx.plan = st, x.shape, (wt, bt), x.get_device(), None
        if M:
            ctx.plan = load_native().LayerNormBackward(is_bf16(x2), is_bf16(weight), st.data_ptr(), M, C,
                                                       wt is torch.bfloat16, bt is torch.bfloat16)
        return y.view(x.shape)

    @staticmethod
    @differentiable_once
    def backward(ctx, dy):
        x2, weight = ctx.saved_tensors   # read here: a saved-tensor hook may have moved them
        plan, (wt, bt), shape, dev = ctx.plan, ctx.types, ctx.shape, x2.device
        C = shape[-1]
        dw = torch.empty(C, device=dev, dtype=wt) if wt is not None else None
        db = torch.empty(C, device=dev, dtype=bt) if bt is not None else None
        dx = torch.empty(shape, device=dev, dtype=x2.dtype) if ctx.needs_input_grad[0] else None
        if plan is None:   # no rows
            for t in (dw, db):
                if t is not None:
                    t.zero_()
            return dx, dw, db, None
        part = torch.empty(plan.space, device=dev) if dw is not None or db is not None else None
        ld = C
        if not dy.is_contiguous():
            dy = rows_of(dy, C)
            ld = dy.stride(0)
        plan(x2.data_ptr(), x2.stride(0), dy.data_ptr(), ld, ptr(weight), ptr(dx), ptr(dw), ptr(db), ptr(part),
             raw_stream(ctx.dev))
        return dx, dw, db, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """See the module docstring.  ``eps`` > 0 keeps rows of equal values finite (their ``y`` is ``bias``); the sum of a
    row has to stay in the range of fp32."""
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"layer_norm: x needs a last dimension of at least 1, got shape {tuple(x.shape)}")
    C = x.shape[-1]
    for k, t in (("weight", weight), ("bias", bias)):
        if t is not None and t.shape != (C,):
            raise ValueError(f"layer_norm: {k} must have shape ({C},), got {tuple(t.shape)}")
    if not eps >= 0.0:
        raise ValueError(f"layer_norm: eps must be >= 0, got {eps}")
    if not x.is_cuda:
        return layer_norm_reference(x, weight, bias, eps)
    check_types("layer_norm", x=x, weight=weight, bias=bias)
    check_device("layer_norm", x, weight=weight, bias=bias)
    check_forward_mode("layer_norm", x, weight, bias)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        check_leaves("layer_norm", x, weight, bias)
        return _LayerNorm.apply(x, weight, bias, float(eps))
    check_not_traced("layer_norm")
    return _forward(rows_of(x, C), dense(weight), dense(bias), float(eps), False)[0].view(x.shape)
