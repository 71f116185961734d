"""Layer norm over the last dimension (``csrc/ops/norm.hip``), forward and backward.

    mu = mean_c x,  r = 1 / sqrt(mean_c (x - mu)^2 + eps),  y = (x - mu) r weight + bias

``layer_norm`` runs the HIP kernels for CUDA tensors and :func:`layer_norm_reference` otherwise.  ``x`` is bf16 or fp32,
of any shape; ``weight`` and ``bias`` [C] are each fp32, bf16 or absent, whatever the type of ``x`` (bf16 activations
with the learner's fp32 masters need no cast).  Statistics and sums are fp32, ``y`` and the gradients have the types of
``x``, ``weight`` and ``bias``; the parameter gradients are summed in a fixed order (bitwise reproducible).
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from gsc_amd.native import load as load_native

_TYPES = (torch.bfloat16, torch.float32)


def device_guard(t: torch.Tensor):
    """Kernels are launched on the device of their tensors, whichever is current."""
    return torch.cuda.device(t.device)


def rows_of(t: torch.Tensor, C: int) -> torch.Tensor:
    """[rows, C] view of ``t`` with contiguous rows (a copy only where its strides allow no such view)."""
    t = t if t.dim() == 2 else t.reshape(-1, C)
    return t if C == 1 or t.stride(1) == 1 else t.contiguous()


def check_cuda(name: str, x: torch.Tensor, **others) -> None:
    for k, t in others.items():
        if t is not None and t.device != x.device:
            raise ValueError(f"{name}: {k} is on {t.device}, x on {x.device}")


_STREAM = "gsc_amd.stream"


def note_leaves(name: str, out: torch.Tensor, *inputs) -> torch.Tensor:
    """Refuses to capture an op on a leaf whose gradient node lives in a graph made on another stream.

    Autograd keeps one gradient node per leaf for as long as any graph holds it, bound to the stream it was made on.  A
    backward pass captured later would make that stream, outside the capture, wait for the captured one, which ends the
    process when the capture ends.  ``inputs``: the Function's tensor arguments in order (None: absent)."""
    stream = torch.cuda.current_stream(out.device).cuda_stream
    capturing = torch.cuda.is_current_stream_capturing()
    for t, (node, _) in zip((t for t in inputs if t is not None), out.grad_fn.next_functions):
        if node is None or not t.is_leaf:
            continue
        if node.metadata.setdefault(_STREAM, stream) != stream and capturing:
            raise RuntimeError(f"{name}: a graph of the same leaf tensor {tuple(t.shape)}, made on another stream, is still "
                               "alive; a captured backward pass cannot share its gradient node (drop the outputs of "
                               "earlier calls before the capture, or capture with leaves of its own)")
    return out


def layer_norm_reference(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                         eps: float = 1e-5) -> torch.Tensor:
    """The same function in elementary PyTorch operations (fp32 inside, or fp64 for fp64 inputs), differentiable."""
    xf = x if x.dtype == torch.float64 else x.float()
    d = xf - xf.mean(-1, keepdim=True)
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
        with device_guard(x2):
            load_native().layer_norm_forward(
                x2.data_ptr(), x2.stride(0), x2.dtype == torch.bfloat16, weight.data_ptr() if weight is not None else 0,
                weight is not None and weight.dtype == torch.bfloat16, bias.data_ptr() if bias is not None else 0,
                bias is not None and bias.dtype == torch.bfloat16, y.data_ptr(), st.data_ptr() if stats else 0,
                st[1].data_ptr() if stats else 0, M, C, eps, torch.cuda.current_stream(x2.device).cuda_stream)
    return y, st


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        x2 = rows_of(x, x.shape[-1])
        y, st = _forward(x2, weight, bias, eps, True)
        ctx.save_for_backward(x2, weight, st)
        ctx.shape, ctx.bias = x.shape, None if bias is None else bias.dtype
        return y.view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x2, weight, st = ctx.saved_tensors
        M, C = x2.shape
        need = ctx.needs_input_grad
        mk = lambda *s, dt: torch.empty(*s, device=x2.device, dtype=dt)
        dx = mk(M, C, dt=x2.dtype) if need[0] else None
        dw = mk(C, dt=weight.dtype) if need[1] else None
        db = mk(C, dt=ctx.bias) if need[2] else None
        if M == 0:
            for t in (dw, db):
                if t is not None:
                    t.zero_()
        elif any(need[:3]):
            nat = load_native()
            dy2 = rows_of(dy, C)
            part = mk(nat.layer_norm_workspace(M, C), dt=torch.float32) if dw is not None or db is not None else None
            p = lambda t: t.data_ptr() if t is not None else 0
            bf = lambda t: t is not None and t.dtype == torch.bfloat16
            with device_guard(x2):
                nat.layer_norm_backward(x2.data_ptr(), x2.stride(0), dy2.data_ptr(), dy2.stride(0), bf(x2), p(weight),
                                        bf(weight), st.data_ptr(), st[1].data_ptr(), p(dx), p(dw), bf(dw), p(db), bf(db),
                                        p(part), M, C, torch.cuda.current_stream(x2.device).cuda_stream)
        return dx.view(ctx.shape) if dx is not None else None, dw, db, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """See the module docstring.  ``eps`` > 0 keeps rows of equal values finite (their ``y`` is ``bias``)."""
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"layer_norm: x needs a last dimension of at least 1, got shape {tuple(x.shape)}")
    C = x.shape[-1]
    for k, t in (("weight", weight), ("bias", bias)):
        if t is not None and t.shape != (C,):
            raise ValueError(f"layer_norm: {k} must have shape ({C},), got {tuple(t.shape)}")
    if not (eps >= 0.0):
        raise ValueError(f"layer_norm: eps must be >= 0, got {eps}")
    if not x.is_cuda:
        return layer_norm_reference(x, weight, bias, eps)
    for k, t in (("x", x), ("weight", weight), ("bias", bias)):
        if t is not None and t.dtype not in _TYPES:
            raise TypeError(f"layer_norm: {k} must be bfloat16 or float32 on the GPU, got {t.dtype}")
    check_cuda("layer_norm", x, weight=weight, bias=bias)
    weight = weight.contiguous() if weight is not None else None
    bias = bias.contiguous() if bias is not None else None
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return note_leaves("layer_norm", _LayerNorm.apply(x, weight, bias, float(eps)), x, weight, bias)
    return _forward(rows_of(x, C), weight, bias, float(eps), False)[0].view(x.shape)
