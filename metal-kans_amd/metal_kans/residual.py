"""Norms before and after a block, fused with its gate and residual scale (``kans_residual_norm_*``).

``residual_norm`` is what stands between two blocks of a residual network (``TorchMetalKANLinear``
stacks, a feed-forward block)::

    y = x + scale * gate * norm(block) * post_weight      # the residual stream
    h = norm(y) * pre_weight                              # the next block's input

in one pass over the rows, with gradients for every input.  Everything is computed in fp32 and
rounded once, h from the y before its rounding; sums over rows are added up in a fixed order, so
results are the same on every run.
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from ._torch_ops import load

_DT = (torch.float32, torch.float16, torch.bfloat16)
_KINDS = {"rms": 0, "layer": 1}


def _refuse(x, block, gate, scale, post_weight, pre_weight, kind, eps):
    """What is wrong with the arguments of a call."""
    if kind not in _KINDS:
        raise ValueError(f"kind must be 'rms' or 'layer', got {kind!r}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x of shape {tuple(x.shape)} has no last dimension to normalize")
    if block is None and (gate is not None or post_weight is not None):
        raise ValueError("gate and post_weight need a block")
    if not 0.0 <= eps < float("inf"):
        raise ValueError(f"eps must be finite and >= 0, got {eps}")
    d = x.shape[-1]
    dt = block.dtype if block is not None else pre_weight.dtype if pre_weight is not None else x.dtype
    if dt not in _DT or x.dtype not in (dt, torch.float32):
        raise TypeError(f"x is {x.dtype} and the block {dt}; x must be fp32 or the block's fp32, fp16 or bf16")
    for name, t in (("block", block), ("gate", gate), ("post_weight", post_weight), ("pre_weight", pre_weight)):
        if t is not None and t.dtype != dt:
            raise TypeError(f"{name} is {t.dtype}, expected {dt}")
    if isinstance(scale, torch.Tensor) and (scale.numel() != 1 or scale.dtype != torch.float32):
        raise TypeError("a tensor scale is one fp32 element")
    for name, t in (("x", x), ("block", block), ("gate", gate), ("post_weight", post_weight), ("pre_weight", pre_weight),
                    ("scale", scale)):
        if isinstance(t, torch.Tensor) and (not t.is_cuda or t.device != x.device):
            raise ValueError(f"{name} is on {t.device}; residual_norm takes tensors on one GPU")
    if block is not None and block.shape != x.shape:
        raise ValueError(f"block is {tuple(block.shape)}, x {tuple(x.shape)}")
    for name, w in (("post_weight", post_weight), ("pre_weight", pre_weight)):
        if w is not None and tuple(w.shape) != (d,):
            raise ValueError(f"{name} is {tuple(w.shape)}, expected ({d},)")
    raise ValueError(f"gate of shape {tuple(gate.shape)} does not broadcast to {tuple(x.shape)}")


def residual_norm(x: torch.Tensor, block: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
                  scale: Union[float, torch.Tensor] = 1.0, post_weight: Optional[torch.Tensor] = None,
                  pre_weight: Optional[torch.Tensor] = None, kind: str = "rms", eps: float = 1e-6):
    """The residual stream behind a block and the normalized input of the next one.

    Args:
        x: residual stream [..., D]; fp32, or the block's dtype
        block: the block's output, of x's shape; None before the first block (y is x then)
        gate: broadcasts to x's shape: [D] for each channel, [B, 1, D] for each sequence, full, ...
        scale: residual scale, a number or an fp32 tensor of one element
        post_weight, pre_weight: [D], of the norms behind and before a block (None: ones)
        kind: "rms" (a / sqrt(mean(a^2) + eps)) or "layer" ((a - mean) / sqrt(var + eps))

    Returns (y, h): y = x + scale * gate * norm(block) * post_weight in x's dtype and
    h = norm(y) * pre_weight in the block's (without a block: pre_weight's or x's).  Tensors live on one
    GPU; block, gate and weights share one dtype.  Gradients of both outputs reach every input.
    """
    learned = isinstance(scale, torch.Tensor)
    out = load().residual_norm(x, block, gate, scale if learned else None, 0.0 if learned else scale, post_weight, pre_weight,
                               _KINDS.get(kind, -1), eps)
    if out is None:
        _refuse(x, block, gate, scale, post_weight, pre_weight, kind, eps)
    y, h = out
    return (x if block is None else y), h
