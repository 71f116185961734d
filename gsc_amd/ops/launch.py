"""What the wrappers of the feed-forward operators share: argument checks, row views, launches, autograd rules."""
from __future__ import annotations

import functools
from typing import Optional

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable as _once_differentiable
from torch.autograd.graph import get_gradient_edge

TYPES = (torch.bfloat16, torch.float32)
raw_stream = torch._C._cuda_getCurrentRawStream


def launch(fn, t: torch.Tensor, *args) -> None:
    """``fn(*args, stream)`` on the device of ``t`` (made current if it is not) and its current stream."""
    dev = t.get_device()
    if dev == torch.cuda.current_device():
        fn(*args, raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            fn(*args, raw_stream(dev))


def ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


def size(t) -> int:
    return 0 if t is None else t.numel()


def is_bf16(t) -> bool:
    return t is not None and t.dtype is torch.bfloat16


def rows_of(t: torch.Tensor, C: int, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """[rows, C] view of ``t`` with contiguous rows (a copy only where its strides allow no such view).  ``dtype``: cast
    first, since a cast chooses strides of its own (overlapping rows of unit stride come back with others)."""
    if dtype is not None:
        t = t.to(dtype)
    t = t if t.dim() == 2 else t.reshape(-1, C)
    return t if C == 1 or t.stride(1) == 1 else t.contiguous()


def dense(t):
    """``t`` with contiguous elements, None as it is."""
    return t if t is None or t.is_contiguous() else t.contiguous()


def check_device(name: str, x: torch.Tensor, **others) -> None:
    for k, t in others.items():
        if t is not None and t.device != x.device:
            raise ValueError(f"{name}: {k} is on {t.device}, x on {x.device}")


def check_types(name: str, **tensors) -> None:
    for k, t in tensors.items():
        if t is not None and t.dtype not in TYPES:
            raise TypeError(f"{name}: {k} must be bfloat16 or float32 on the GPU, got {t.dtype}")


def check_forward_mode(name: str, *tensors) -> None:
    """Refuses inputs with a tangent: a kernel reads the primal alone, and its result would have none."""
    if forward_ad._current_level < 0:   # no dual level is open
        return
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{name}: forward-mode derivatives are not supported on the GPU")


def check_not_traced(name: str) -> None:
    """Refuses a launch under torch.jit.trace: the trace would hold the empty result and not the kernel that fills it."""
    if torch._C._is_tracing():
        raise RuntimeError(f"{name}: cannot be traced on the GPU without gradients (the kernel launch is not recorded)")


def differentiable_once(backward):
    """``once_differentiable`` at little cost to a plain backward pass: its wrapper is used under ``create_graph`` only.

    (What a backward pass does in Python runs on autograd's own thread, two to three times slower than the same lines of
    the forward pass, so the Functions prepare their launches in ``forward``.  Autograd makes the device of the forward
    call current there.)"""
    checked = _once_differentiable(backward)

    @functools.wraps(backward)
    def run(ctx, grad, enabled=torch.is_grad_enabled):
        return checked(ctx, grad) if enabled() else backward(ctx, grad)

    return run


class _Seen(Exception):
    pass


class _NoGradient(torch.autograd.Function):
    """The identity, whose backward pass hands on no gradient."""

    @staticmethod
    def forward(ctx, t):
        return t.view_as(t)

    @staticmethod
    def backward(ctx, g):
        return None


def _held(t: torch.Tensor) -> bool:
    """Whether any graph holds the gradient node of leaf ``t``: a mark on it outlives this function's own reference."""
    get_gradient_edge(t).node.metadata["gsc_amd.held"] = True
    return get_gradient_edge(t).node.metadata.pop("gsc_amd.held", False)


def _node_stream(t: torch.Tensor):
    """The stream of leaf ``t``'s gradient node (None: not found).  The engine makes it current before a node's hooks run; the
    hook ends the pass there.  Without a gradient to hand on, the pass touches no stream, so a capture is left as it was."""
    if t._backward_hooks:   # they would be called without a gradient
        return None
    seen = []

    def look(grads):
        seen.append(raw_stream(t.get_device()))
        raise _Seen

    hook = get_gradient_edge(t).node.register_prehook(look)
    try:
        torch.autograd.backward([_NoGradient.apply(t)], [t.detach()])
    except _Seen:
        pass
    finally:
        hook.remove()
    return seen[0] if seen else None


def check_leaves(name: str, *inputs) -> None:
    """Refuses to capture an op on a leaf whose gradient node lives in a graph made on another stream, by whatever operator.

    Autograd keeps one gradient node per leaf for as long as any graph holds it, bound to the stream it was made on.  A
    backward pass captured later would make that stream, outside the capture, wait for the captured one, which ends the
    process when the capture ends."""
    if not torch.cuda.is_current_stream_capturing():
        return
    for t in inputs:
        if t is not None and t.requires_grad and t.is_leaf and _held(t) and _node_stream(t) != raw_stream(t.get_device()):
            raise RuntimeError(f"{name}: a graph of the same leaf tensor {tuple(t.shape)}, made on another stream, is still "
                               "alive; a captured backward pass cannot share its gradient node (drop the outputs of "
                               "earlier calls before the capture, or capture with leaves of its own)")
