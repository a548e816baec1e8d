"""Mixing along the sequence: a short causal convolution and a selective state space scan (``kans_causal_conv_*``,
``kans_selective_scan_*``).

Both take whole sequences, with gradients, or carry a state: called with the state that the call before left, a
prompt in pieces and then single tokens give what the whole sequence would.  Everything is computed in fp32
and rounded once; sums are added up in a fixed order, the same on every run.
"""
from __future__ import annotations

from typing import Optional

import torch

from ._torch_ops import load

_DT = (torch.float32, torch.float16, torch.bfloat16)
_ACTIVATIONS = {None: 0, "silu": 1}


def _refuse_common(x, state, shape, dtype, lengths):
    if x.dim() != 3 or x.shape[-1] == 0:
        raise ValueError(f"x {tuple(x.shape)} must be [B, L, D]")
    if x.dtype not in _DT:
        raise TypeError(f"x is {x.dtype}, must be fp32, fp16 or bf16")
    if state is not None:
        if state.dtype != dtype:
            raise TypeError(f"state is {state.dtype}, expected {dtype}")
        if tuple(state.shape) != shape or not state.is_contiguous():
            raise ValueError(f"state {tuple(state.shape)} must be {shape} and contiguous")
    if lengths is not None:
        if lengths.dtype != torch.int64:
            raise TypeError(f"lengths are {lengths.dtype}, expected torch.int64")
        if tuple(lengths.shape) != (x.shape[0],):
            raise ValueError(f"lengths {tuple(lengths.shape)} must be ({x.shape[0]},)")


def _refuse_conv(x, weight, bias, activation, state, lengths):
    """What is wrong with the arguments of a call."""
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation must be 'silu' or None, got {activation!r}")
    if weight.dim() != 2 or not 1 <= weight.shape[1] <= 8 or x.dim() != 3 or weight.shape[0] != x.shape[-1]:
        raise ValueError(f"x {tuple(x.shape)} and weight {tuple(weight.shape)} must be [B, L, D] and [D, W], W from 1 to 8")
    if bias is not None and tuple(bias.shape) != (x.shape[-1],):
        raise ValueError(f"bias {tuple(bias.shape)} must be ({x.shape[-1]},)")
    _refuse_common(x, state, (x.shape[0], weight.shape[1] - 1, x.shape[-1]), x.dtype, lengths)
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and t.dtype != x.dtype:
            raise TypeError(f"{name} is {t.dtype}, expected {x.dtype}")
    raise ValueError("causal_conv takes tensors on one GPU")


def causal_conv(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: Optional[str] = "silu",
                state: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Each channel convolved with its own few taps along the sequence, up to and including the step itself.

    Args:
        x: [B, L, D], fp32, fp16 or bf16, on the GPU (any view whose channels lie side by side is read as it is)
        weight: [D, W], W from 1 to 8; the last tap is the step's own
        bias: [D]
        activation: "silu" (u sigmoid(u)) or None
        state: [B, W - 1, D], contiguous, apart from x: the inputs before the first step (None: zeros).  Afterwards it holds the last
            W - 1 inputs of each sequence, for the next call.  Without gradients only.
        lengths: [B] int64 on the GPU, the steps of each sequence that count: the others give zeros (as do gradients
            there) and are not looked at, nor kept in the state

    Returns [B, L, D] in x's type, which all tensors share; gradients reach x, weight and bias.
    """
    out = load().causal_conv(x, weight, bias, _ACTIVATIONS.get(activation, -1), state, lengths)
    if out is None:
        _refuse_conv(x, weight, bias, activation, state, lengths)
    return out


def _refuse_scan(x, dt, A, B, C, D, z, dt_bias, state, lengths):
    """What is wrong with the arguments of a call."""
    if x.dim() != 3 or A.dim() != 2 or A.shape[0] != x.shape[-1] or not 1 <= A.shape[1] <= 64:
        raise ValueError(f"x {tuple(x.shape)} and A {tuple(A.shape)} must be [B, L, D] and [D, N], N from 1 to 64")
    _refuse_common(x, state, (x.shape[0], x.shape[-1], A.shape[1]), torch.float32, lengths)
    for name, t, last in (("dt", dt, x.shape[-1]), ("B", B, A.shape[1]), ("C", C, A.shape[1]), ("z", z, x.shape[-1])):
        if t is None:
            continue
        if tuple(t.shape) != (*x.shape[:2], last):
            raise ValueError(f"{name} {tuple(t.shape)} must be {(*x.shape[:2], last)}")
        if t.dtype != x.dtype:
            raise TypeError(f"{name} is {t.dtype}, expected {x.dtype}")
    for name, t in (("A", A), ("D", D), ("dt_bias", dt_bias)):
        if t is None:
            continue
        if t.dtype != torch.float32:
            raise TypeError(f"{name} is {t.dtype}, expected torch.float32")
        if name != "A" and tuple(t.shape) != (x.shape[-1],):
            raise ValueError(f"{name} {tuple(t.shape)} must be ({x.shape[-1]},)")
    raise ValueError("selective_scan takes tensors on one GPU")


def selective_scan(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                   D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None, dt_bias: Optional[torch.Tensor] = None,
                   softplus: bool = True, state: Optional[torch.Tensor] = None,
                   lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
    """A linear recurrence of N states a channel, whose step sizes, inputs and outputs depend on the token::

        s = softplus(dt + dt_bias)
        h[t] = exp(s[t] A) h[t - 1] + s[t] x[t] B[t]
        out[t] = (C[t] . h[t] + D x[t]) * silu(z[t])

    Args:
        x, dt, z: [batch, L, channels], fp32, fp16 or bf16, on the GPU; z (None: no gate) multiplies the result
        A: [channels, N] fp32, N up to 64, negative for states that decay
        B, C: [batch, L, N] of x's type, shared by the channels
        D, dt_bias: [channels] fp32 (None: zeros)
        softplus: False takes dt + dt_bias as it is
        state: [batch, channels, N] fp32, contiguous, apart from the others: the states before the first step (None: zeros).  Afterwards it
            holds those behind each sequence's last step, for the next call.  Without gradients only.
        lengths: [batch] int64 on the GPU, the steps of each sequence that count: the others give zeros (as do
            gradients there), are not looked at and leave the state

    Views whose channels (states) lie side by side and whose steps do not overlap are read as they are.  Returns [batch, L, channels] in x's
    type; gradients reach x, dt, A, B, C, D, z and dt_bias, those of A, D and dt_bias in fp32.
    """
    out = load().selective_scan(x, dt, A, B, C, D, z, dt_bias, softplus, state, lengths)
    if out is None:
        _refuse_scan(x, dt, A, B, C, D, z, dt_bias, state, lengths)
    return out
