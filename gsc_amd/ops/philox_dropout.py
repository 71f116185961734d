"""Dropout from a counter-based generator (``csrc/ops/dropout.hip``): the mask is never stored.

Element ``i`` (row-major) stays when its 32-bit uniform, a function of ``(seed, offset, i)`` alone, is at least
``round(p 2^32)``; the backward pass draws the same mask again.  The same ``(seed, offset)`` gives the same mask on the
GPU, on the CPU and for any strides: callers give every call site its own ``seed`` and every step its own ``offset``.

``offset`` is an int, or a one-element int64 CUDA tensor read when the kernel runs: in a captured HIP graph each replay
draws a new mask once something in (or between) the replays has advanced that tensor.  The forward call keeps the value
it read for its own backward pass, so the tensor may be advanced between the two.  Second derivatives, forward-mode
derivatives and traces without gradients are refused on the GPU.
"""
from __future__ import annotations

from typing import Optional, Union

import numpy as np
import torch

from gsc_amd.native import load as load_native
from .launch import check_device, check_forward_mode, check_leaves, check_not_traced, check_types, differentiable_once, is_bf16, launch, ptr, raw_stream

_M32 = np.uint64(0xFFFFFFFF)


def _philox(groups: int, seed: int, offset: int) -> np.ndarray:
    """Philox4x32-10 blocks of groups 0 .. groups - 1 (key ``seed``, counter ``(group, offset)``): uint32 [groups, 4]."""
    i = np.arange(groups, dtype=np.uint64)
    c = [i & _M32, i >> np.uint64(32), np.full(groups, offset & 0xFFFFFFFF, np.uint64),
         np.full(groups, offset >> 32, np.uint64)]
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), p1 & _M32, (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(k1),
             p0 & _M32]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(c, 1).astype(np.uint32)


def threshold(p: float) -> int:
    """Uniforms below this (of 2^32) are dropped."""
    return min(round(p * 2.0 ** 32), 2 ** 32 - 1)


def dropout_mask(shape, p: float, seed: int, offset: int = 0) -> torch.Tensor:
    """The keep mask of :func:`dropout` as a CPU bool tensor."""
    n = int(np.prod(shape, dtype=np.int64))
    groups = -(-n // 8)
    a, b = _philox(groups, seed, offset), _philox(groups, seed, offset | (1 << 63))
    halves = lambda w: np.stack((w & 0xFFFF, w >> 16), -1).reshape(-1)[:n].astype(np.uint32)
    u = (halves(a) << np.uint32(16)) | halves(b)
    return torch.from_numpy(u >= np.uint32(threshold(p))).view(shape)


def dropout_reference(x: torch.Tensor, p: float, seed: int, offset: int = 0,
                      residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The same function in elementary PyTorch operations (fp32 inside, fp64 for fp64 inputs), differentiable."""
    keep = dropout_mask(x.shape, p, seed, offset).to(x.device)
    xf = x if x.dtype == torch.float64 else x.float()
    y = torch.where(keep, xf * (1.0 / (1.0 - p)), torch.zeros((), dtype=xf.dtype, device=x.device))
    if residual is not None:
        y = y + residual.to(xf.dtype)
    return y.to(x.dtype)


def _launch(x, res, p, seed, offset, at, keep_at):
    y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    n = x.numel()
    if n > 0:
        launch(load_native().dropout, x, x.data_ptr(), ptr(res), y.data_ptr(), is_bf16(x), n, seed, offset, ptr(at),
               ptr(keep_at), p)
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, offset, at):
        used = torch.empty(1, device=x.device, dtype=torch.int64) if at is not None else None
        ctx.used = used   # the offset this call read
        ctx.args = (is_bf16(x), x.numel(), seed, offset, ptr(used), 0, p)
        ctx.run, ctx.dev = load_native().dropout, x.get_device()
        return _launch(x.contiguous(), residual.contiguous() if residual is not None else None, p, seed, offset, at, used)

    @staticmethod
    @differentiable_once
    def backward(ctx, dy):
        need_x, need_res = ctx.needs_input_grad[:2]
        dx = None
        if need_x:
            dy = dy.contiguous()
            dx = torch.empty_like(dy)
            if ctx.args[1]:
                ctx.run(dy.data_ptr(), 0, dx.data_ptr(), *ctx.args, raw_stream(ctx.dev))
        return dx, dy if need_res else None, None, None, None, None


def dropout(x: torch.Tensor, p: float, seed: int, offset: Union[int, torch.Tensor] = 0,
            residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x / (1 - p)`` where the mask keeps an element and 0 elsewhere (whatever ``x`` holds there), plus ``residual``.

    ``p`` in [0, 1), ``seed`` in [0, 2^64), ``offset`` in [0, 2^63) (an int or a one-element int64 tensor on ``x``'s
    device, see above).  ``x`` and ``residual`` are bf16 or fp32, of the same shape and type; the sum is rounded once."""
    if not 0.0 <= p < 1.0:
        raise ValueError(f"dropout: p must be in [0, 1), got {p}")
    if not 0 <= seed < 1 << 64:
        raise ValueError(f"dropout: seed must be in [0, 2^64), got {seed}")
    at = None
    if isinstance(offset, torch.Tensor):
        if offset.dtype != torch.int64 or offset.numel() != 1:
            raise TypeError(f"dropout: an offset tensor is one int64 element, got {tuple(offset.shape)} {offset.dtype}")
        if offset.is_cuda != x.is_cuda or (x.is_cuda and offset.device != x.device):
            raise ValueError(f"dropout: the offset tensor is on {offset.device}, x on {x.device}")
        offset, at = (0, offset) if x.is_cuda else (int(offset), None)
    if not 0 <= offset < 1 << 63:
        raise ValueError(f"dropout: offset must be in [0, 2^63), got {offset}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"dropout: residual must match x ({tuple(x.shape)}, {x.dtype}), got {tuple(residual.shape)}, "
                         f"{residual.dtype}")
    if not x.is_cuda:
        return dropout_reference(x, p, seed, offset, residual)
    check_types("dropout", x=x)
    check_device("dropout", x, residual=residual)
    check_forward_mode("dropout", x, residual)
    if torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad)):
        check_leaves("dropout", x, residual)
        return _Dropout.apply(x, residual, float(p), int(seed), int(offset), at)
    check_not_traced("dropout")
    return _launch(x.contiguous(), residual.contiguous() if residual is not None else None, float(p), int(seed),
                   int(offset), at, None)
