"""Softmax cross entropy of a linear head over a large vocabulary (``kans_linear_xent_*``).

``linear_cross_entropy(hidden, weight, target)`` is ``cross_entropy(hidden @ weight.T, target)`` with its
gradients, without the logits ever being in memory: the forward keeps a sum of exponentials per row and
tile, the backward computes the logits again, a piece of the vocabulary at a time.
"""
from __future__ import annotations

import torch

from ._torch_ops import load

_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


def _refuse(hidden, weight, target, reduction):
    """What is wrong with the arguments of a call."""
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be 'mean', 'sum' or 'none', got {reduction!r}")
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1] or 0 in weight.shape:
        raise ValueError(f"hidden {tuple(hidden.shape)} and weight {tuple(weight.shape)} must be [..., D] and [V, D]")
    if target.shape != hidden.shape[:-1]:
        raise ValueError(f"target is {tuple(target.shape)}, expected {tuple(hidden.shape[:-1])}")
    if hidden.dtype not in (torch.float32, torch.float16, torch.bfloat16) or weight.dtype != hidden.dtype:
        raise TypeError(f"hidden is {hidden.dtype} and weight {weight.dtype}; both must be fp32, fp16 or bf16")
    if target.dtype != torch.int64:
        raise TypeError(f"target is {target.dtype}, expected torch.int64")
    raise ValueError("linear_cross_entropy takes tensors on one GPU")


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
    loss = load().linear_cross_entropy(hidden, weight, target, ignore_index, _REDUCTIONS.get(reduction, -1))
    if loss is None:
        _refuse(hidden, weight, target, reduction)
    return loss
