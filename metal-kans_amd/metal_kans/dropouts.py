"""Dropout from a counter-based generator, whose mask is never stored (``kans_dropout``)."""
from __future__ import annotations

from typing import Union

import torch

from ._torch_ops import load

_WORD = 1 << 64


def _refuse(x, p, seed):
    """What is wrong with the arguments of a call."""
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p must be in [0, 1], got {p}")
    if x.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise TypeError(f"x is {x.dtype}, must be fp32, fp16 or bf16")
    if isinstance(seed, torch.Tensor) and (seed.numel() != 1 or seed.dtype != torch.int64):
        raise TypeError("a tensor seed is one int64 element")
    raise ValueError("dropout takes tensors on one GPU")


def _signed(word: int, name: str) -> int:
    """A 64-bit word as a signed number."""
    if not -_WORD // 2 <= word < _WORD:
        raise ValueError(f"{name} must fit 64 bits, got {word}")
    return word - _WORD if word >= _WORD // 2 else word


def dropout(x: torch.Tensor, p: float, seed: Union[int, torch.Tensor], offset: int = 0) -> torch.Tensor:
    """x with a share p of its elements set to zero and the others divided by 1 - p, with x's gradient.

    Args:
        x: any shape, fp32, fp16 or bf16, on the GPU
        p: in [0, 1]; an element is dropped where its random number of 32 bits is below p 2^32
        seed: 64 bits that choose the random numbers: an int, or an int64 tensor of one element on x's device,
            which is read when the kernel runs (a captured graph drops others on every replay if the program
            changes it in between; the backward uses the value that its forward had, but a checkpoint, which runs the
            forward again in the backward, reads the seed again)
        offset: 64 bits more, for calls that share a seed (layers, steps)

    The random number of element i (counted in row-major order) is word i % 4 of Philox4x32-10 with key ``seed``
    at the counter (i // 4, offset), on every run and device alike.  Dropped elements are zero, also
    where x is infinite or NaN.
    """
    dev = isinstance(seed, torch.Tensor)
    out = load().dropout(x, p, 0 if dev else _signed(seed, "seed"), seed if dev else None, _signed(offset, "offset"))
    if out is None:
        _refuse(x, p, seed)
    return out
