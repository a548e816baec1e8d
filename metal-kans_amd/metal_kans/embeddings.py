"""Rows of a table for the tokens of a batch, and the table's gradient (``kans_embedding_*``).

The gradient sorts the tokens and adds up the rows of equal ones in the order of their positions, in fp32: no
atomics, the same result on every run.
"""
from __future__ import annotations

import torch

from ._torch_ops import load

_LEAST, _MOST = 2.0 ** -126, (2.0 - 2.0 ** -23) * 2.0 ** 127  # of fp32's normal numbers


def _refuse(tokens, weight, scale):
    """What is wrong with the arguments of a call."""
    if weight.dim() != 2 or 0 in weight.shape:
        raise ValueError(f"weight {tuple(weight.shape)} must be [V, D]")
    if scale != 0 and not _LEAST <= abs(scale) <= _MOST:
        raise ValueError(f"scale must be zero or a normal number of fp32, got {scale}")
    if weight.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise TypeError(f"weight is {weight.dtype}, must be fp32, fp16 or bf16")
    if tokens.dtype != torch.int64:
        raise TypeError(f"tokens are {tokens.dtype}, expected torch.int64")
    raise ValueError("embedding takes tensors on one GPU")


def embedding(tokens: torch.Tensor, weight: torch.Tensor, scale: float = 1.0, ignore_index: int = -100) -> torch.Tensor:
    """scale * weight[tokens], with the gradient of weight.

    Args:
        tokens: [...] int64 on the GPU, rows in [0, V) or ``ignore_index`` (padding: a row of zeros, whose
            gradient is not looked at); any other value gives a row of NaN and takes no part in the gradient
        weight: the table [V, D], fp32, fp16 or bf16
        scale: a number that every row is multiplied with, in fp32 (zero, or from 2^-126 to below 2^128)

    Returns [..., D] in weight's type.  weight's gradient is dense: rows of tokens that are not there are zeros.
    """
    out = load().embedding(tokens, weight, scale, ignore_index)
    if out is None:
        _refuse(tokens, weight, scale)
    return out
