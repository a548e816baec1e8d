"""Softmax cross entropy of a linear head over a large vocabulary (``kans_linear_xent_*``).

``linear_cross_entropy(hidden, weight, target)`` is ``cross_entropy(hidden @ weight.T, target)`` with its
gradients, without the logits ever being in memory: the forward keeps a sum of exponentials per row and
tile, the backward computes the logits again, a piece of the vocabulary at a time.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import device
from ._engine import DT_BF16, DT_F16, DT_F32
from .torch_module import _current_stream

_DT = {torch.float32: DT_F32, torch.float16: DT_F16, torch.bfloat16: DT_BF16}
_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


def _workspace(lib, h, n, d, v, backward):
    size = lib.kans_linear_xent_workspace(_DT[h.dtype], n, d, v, backward)
    device.check(min(size, 0), "kans_linear_xent_workspace")
    return torch.empty(size, dtype=torch.uint8, device=h.device), size


def _forward(h, w, target, ignore, reduction):
    n, d = h.shape
    v = w.shape[0]
    loss = torch.empty(n if reduction == 0 else (), dtype=torch.float32, device=h.device)
    state = torch.empty(4 + 3 * n, dtype=torch.int32, device=h.device)
    if n == 0:
        return loss if reduction == 0 else loss.fill_(float("nan") if reduction == 1 else 0.0), state
    lib = device.get_metal_bridge()
    ws, size = _workspace(lib, h, n, d, v, 0)
    device.check(lib.kans_linear_xent_forward(
        _DT[h.dtype], h.data_ptr(), w.data_ptr(), target.data_ptr(), n, d, v, ignore, reduction, loss.data_ptr(),
        state.data_ptr(), ws.data_ptr(), size, _current_stream(h.device)), "kans_linear_xent_forward")
    return loss, state


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, w, target, ignore, reduction):
        loss, state = _forward(h, w, target, ignore, reduction)
        ctx.save_for_backward(h, w, target, state)
        ctx.rest = (ignore, reduction)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        h, w, target, state = ctx.saved_tensors
        ignore, reduction = ctx.rest
        n, d = h.shape
        v = w.shape[0]
        dh = torch.empty_like(h) if ctx.needs_input_grad[0] else None
        dw = torch.empty_like(w) if ctx.needs_input_grad[1] else None
        if n == 0:
            return dh, None if dw is None else dw.zero_(), None, None, None
        lib = device.get_metal_bridge()
        grad = grad.contiguous()
        ws, size = _workspace(lib, h, n, d, v, 1)
        device.check(lib.kans_linear_xent_backward(
            _DT[h.dtype], h.data_ptr(), w.data_ptr(), target.data_ptr(), n, d, v, ignore, reduction, state.data_ptr(),
            grad.data_ptr(), None if dh is None else dh.data_ptr(), None if dw is None else dw.data_ptr(), ws.data_ptr(),
            size, _current_stream(h.device)), "kans_linear_xent_backward")
        return dh, dw, None, None, None


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, ignore_index: int = -100,
                         reduction: str = "mean") -> torch.Tensor:
    """Cross entropy of the logits hidden @ weight.T, in fp32, with gradients of hidden and weight.

    Args:
        hidden: [..., D], fp32, fp16 or bf16, on the GPU
        weight: the head [V, D], of hidden's type
        target: [...] int64, classes in [0, V) or ``ignore_index`` (rows that take part in nothing, whatever
            hidden holds there); any other value makes its row's loss NaN
        reduction: "mean" over the rows that are not ignored (NaN if there are none), "sum", or "none"
            (target's shape, 0 in ignored rows)

    The sums of the softmax and all products accumulate in fp32; fp32 inputs are multiplied as three
    bf16 terms each, to fp32's accuracy.  Results are the same on every run.
    """
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be 'mean', 'sum' or 'none', got {reduction!r}")
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1] or 0 in weight.shape:
        raise ValueError(f"hidden {tuple(hidden.shape)} and weight {tuple(weight.shape)} must be [..., D] and [V, D]")
    if target.shape != hidden.shape[:-1]:
        raise ValueError(f"target is {tuple(target.shape)}, expected {tuple(hidden.shape[:-1])}")
    if hidden.dtype not in _DT or weight.dtype != hidden.dtype:
        raise TypeError(f"hidden is {hidden.dtype} and weight {weight.dtype}; both must be fp32, fp16 or bf16")
    if target.dtype != torch.int64:
        raise TypeError(f"target is {target.dtype}, expected torch.int64")
    gpu = hidden.get_device()
    if gpu < 0 or weight.get_device() != gpu or target.get_device() != gpu:
        raise ValueError("linear_cross_entropy takes tensors on one GPU")
    h = hidden.reshape(-1, hidden.shape[-1]).contiguous()
    w, t = weight.contiguous(), target.reshape(-1).contiguous()
    args = (h, w, t, int(ignore_index), _REDUCTIONS[reduction])
    if torch.is_grad_enabled() and (h.requires_grad or w.requires_grad):
        loss = _LinearCrossEntropy.apply(*args)
    else:
        loss, _ = _forward(*args)
    return loss.reshape(target.shape) if reduction == "none" else loss
