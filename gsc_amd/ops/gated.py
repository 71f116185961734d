"""Gated linear layer (``csrc/ops/gated.hip``), forward and backward.

    h = act(x Wg^T + bg) * (x Wu^T + bu)        weight [2F, D]: Wg rows over Wu rows, bias [2F]: bg, bu

``gated_linear`` runs both projections, the activation and the product in one HIP kernel for CUDA tensors, and
:func:`gated_linear_reference` otherwise.  Operands are bf16 or fp32 with fp32 accumulation.  The backward pass takes every
derivative from the fp32 values of both projections: it computes them again from ``x``, or, from ``D`` = 1,024 (bf16) or 128
(fp32) on, where that costs more than memory, reads what the forward pass kept (8 bytes for each element of ``h``; a caller
short of memory between the passes recomputes the layer with ``torch.utils.checkpoint``).  Second derivatives, forward-mode derivatives and
traces without gradients are refused on the GPU.

* bf16 ``x`` with fp32 masters: the weight operand is the masters' bf16 shadow (``FlatParams``) or a cast; their gradients
  come back in fp32.  Under autocast fp32 ``x`` is cast the same way, like :func:`gsc_amd.ops.linear.linear`.
* fp32 ``x`` and weight outside autocast: fp32 matrix instructions.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn.functional as F

from gsc_amd.native import load as load_native
from .launch import check_device, check_forward_mode, check_leaves, check_not_traced, check_types, dense, differentiable_once, is_bf16, launch, ptr, raw_stream, rows_of, size
from .linear import shadow

ACTIVATIONS = {"silu": 0, "gelu": 1, "sigmoid": 2}


def gated_linear_reference(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                           activation: str = "silu") -> torch.Tensor:
    """The same function in PyTorch operations (fp32 inside, fp64 for fp64 inputs), differentiable."""
    dt = torch.float64 if x.dtype == torch.float64 else torch.float32
    g, u = F.linear(x.to(dt), weight.to(dt), bias.to(dt) if bias is not None else None).chunk(2, -1)
    a = {"silu": F.silu, "gelu": F.gelu, "sigmoid": torch.sigmoid}[activation](g)
    return (a * u).to(x.dtype)


def _operands(x: torch.Tensor, w: torch.Tensor):
    """Both matrices as the kernels read them: rows start on 16 bytes, at most 2,000,000 elements apart, and end on a multiple
    of 8 elements (copies with zeros behind each row where they do not; of both in one launch)."""
    M, D = x.shape
    bad = []
    if M:
        for t in (x, w):
            ld = t.stride(0)
            if D % 8 or ld % 8 or t.data_ptr() % 16 or not D <= ld <= 2_000_000:
                bad.append(t)
    if not bad:
        return x, w
    a, b = bad[0], bad[1] if len(bad) == 2 else None
    rows = a.shape[0]
    rows2, ld2 = (0, 0) if b is None else (b.shape[0], b.stride(0))
    out = torch.empty(rows + rows2, -(-D // 8) * 8, device=x.device, dtype=x.dtype)
    launch(load_native().gated_pad, a, a.data_ptr(), a.stride(0), rows, ptr(b), ld2, rows2, out.data_ptr(), out.stride(0),
           is_bf16(x), D)
    if b is not None:
        return out[:rows], out[rows:]
    return (out, w) if a is x else (x, out)


def _forward(x2, w, bias, act, D, saved=None):
    M, Fo, bf, nat = x2.shape[0], w.shape[0] // 2, is_bf16(x2), load_native()
    h = torch.empty(M, Fo, device=x2.device, dtype=x2.dtype)
    if M > 0:
        n = nat.gated_forward_space(bf, M, D, Fo)
        args = (x2.data_ptr(), x2.stride(0), w.data_ptr(), w.stride(0), bf, ptr(bias), is_bf16(bias), h.data_ptr(), ptr(saved))
        if saved is None and not n:
            launch(nat.gated_forward, x2, *args, M, D, Fo, act)
        else:
            work = torch.empty(n, device=x2.device) if n else None
            launch(nat.gated_forward_split, x2, *args, size(saved), ptr(work), n, M, D, Fo, act)
    return h


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, w, act, dtype):
        D, bias = x.shape[-1], dense(bias)
        x2, w = _operands(rows_of(x, D, dtype), w)
        nat, M, Fo, bf = load_native(), x2.shape[0], w.shape[0] // 2, is_bf16(x2)
        n = nat.gated_saved_elements(bf, M, D, Fo) if M else 0
        saved = torch.empty(n, device=x2.device) if n else None
        h = _forward(x2, w, bias, act, D, saved)
        ctx.save_for_backward(x2, w, bias, saved)
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        ctx.run, ctx.dev = nat.gated_backward, x.get_device()
        ctx.sizes, ctx.flags = (M, D, Fo, x.shape), (bf, is_bf16(bias), act)
        ctx.types = (x.dtype if need_x else None, weight.dtype if need_w else None, bias.dtype if need_b else None)
        ctx.space = nat.gated_workspace(bf, M, D, Fo, need_x, need_w, need_b) if M else 0
        return h.view(*x.shape[:-1], Fo)

    @staticmethod
    @differentiable_once
    def backward(ctx, dh):
        x2, w, bias, saved = ctx.saved_tensors
        (M, D, Fo, shape), (bf, b_bf, act), (xt, wt, bt) = ctx.sizes, ctx.flags, ctx.types
        dev = x2.device
        dx = torch.empty(M, D, device=dev, dtype=xt) if xt is not None else None
        dw = torch.empty(2 * Fo, D, device=dev, dtype=wt) if wt is not None else None
        db = torch.empty(2 * Fo, device=dev, dtype=bt) if bt is not None else None
        if M == 0:
            for t in (dw, db):
                if t is not None:
                    t.zero_()
        else:
            dh2 = rows_of(dh, Fo)
            work = torch.empty(ctx.space, device=dev, dtype=torch.uint8)
            ctx.run(x2.data_ptr(), x2.stride(0), w.data_ptr(), w.stride(0), bf, ptr(bias), b_bf, dh2.data_ptr(), dh2.stride(0),
                    ptr(saved), size(saved), ptr(dx), xt is torch.bfloat16, ptr(dw), wt is torch.bfloat16, ptr(db),
                    bt is torch.bfloat16, work.data_ptr(), ctx.space, M, D, Fo, act, raw_stream(ctx.dev))
        return dx.view(shape) if dx is not None else None, dw, db, None, None, None


def gated_linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: str = "silu",
                 w16: Optional[torch.Tensor] = None) -> torch.Tensor:
    """See the module docstring.  ``x`` [.., D] -> [.., F]; ``activation``: silu, gelu (exact, erf) or sigmoid.  ``w16``:
    the bf16 weight operand of fp32 masters (default: their ``FlatParams`` shadow, else a cast)."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"gated_linear: activation must be one of {', '.join(ACTIVATIONS)}, got {activation!r}")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"gated_linear: x needs a last dimension of at least 1, got shape {tuple(x.shape)}")
    D = x.shape[-1]
    if weight.dim() != 2 or weight.shape[1] != D or weight.shape[0] % 2 or weight.shape[0] == 0:
        raise ValueError(f"gated_linear: weight must be [2F, {D}], got {tuple(weight.shape)}")
    if bias is not None and bias.shape != (weight.shape[0],):
        raise ValueError(f"gated_linear: bias must have shape ({weight.shape[0]},), got {tuple(bias.shape)}")
    if w16 is not None and (w16.shape != weight.shape or w16.dtype != torch.bfloat16):
        raise ValueError(f"gated_linear: w16 must be bfloat16 {tuple(weight.shape)}, got {w16.dtype} {tuple(w16.shape)}")
    if not x.is_cuda:
        return gated_linear_reference(x, weight, bias, activation)
    check_types("gated_linear", x=x, weight=weight, bias=bias)
    check_device("gated_linear", x, weight=weight, bias=bias, w16=w16)
    check_forward_mode("gated_linear", x, weight, bias, w16)
    dtype = x.dtype
    if torch.is_autocast_enabled("cuda"):
        dtype = torch.get_autocast_dtype("cuda")
        if dtype != torch.bfloat16:
            raise TypeError(f"gated_linear: autocast to {dtype} is not supported (bfloat16)")
    if dtype == torch.float32 and weight.dtype != torch.float32:
        raise TypeError("gated_linear: float32 x needs a float32 weight")
    w = weight
    if weight.dtype != dtype:
        w = w16 if w16 is not None else shadow(weight)
        w = w if w is not None else weight.detach().to(dtype)
    w = rows_of(w.detach(), D)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)):
        check_leaves("gated_linear", x, weight, bias)
        return _GatedLinear.apply(x, weight, bias, w, ACTIVATIONS[activation], dtype)
    check_not_traced("gated_linear")
    h = _forward(*_operands(rows_of(x, D, dtype), w), dense(bias), ACTIVATIONS[activation], D)
    return h.view(*x.shape[:-1], h.shape[1])
