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
from torch.autograd.function import once_differentiable

from . import device
from ._engine import DT_BF16, DT_F16, DT_F32
from .torch_module import _current_stream

_DT = {torch.float32: DT_F32, torch.float16: DT_F16, torch.bfloat16: DT_BF16}
_KINDS = {"rms": 0, "layer": 1}


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _forward(x, block, gate, post, pre, scale, group, kind, eps, dt, want_stats):
    d = x.shape[-1]
    rows = x.numel() // d
    y = x if block is None else torch.empty_like(x)
    h = torch.empty(x.shape, dtype=dt, device=x.device)
    stats = torch.empty((rows, 2 + 2 * kind), dtype=torch.float32, device=x.device) if want_stats else None
    dev = scale if isinstance(scale, torch.Tensor) else None
    device.check(device.get_metal_bridge().kans_residual_norm_forward(
        _DT[x.dtype], _DT[dt], kind, x.data_ptr(), _ptr(block), _ptr(gate), group, _ptr(post), _ptr(pre), _ptr(dev),
        0.0 if dev is not None else scale, eps, _ptr(y if block is not None else None), h.data_ptr(), _ptr(stats), rows, d,
        _current_stream(x.device)), "kans_residual_norm_forward")
    return y, h, stats


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, block, gate, post, pre, scale, group, kind, eps, dt):
        ctx.gate_shape = None
        if gate is not None and group == 0:  # repeats within a row or over leading dimensions
            ctx.gate_shape = gate.shape
            gate, group = gate.expand(x.shape).contiguous(), 1
        y, h, stats = _forward(x, block, gate, post, pre, scale, group, kind, eps, dt, True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, block, gate, post, pre, scale if isinstance(scale, torch.Tensor) else None, stats)
        ctx.rest = (0.0 if isinstance(scale, torch.Tensor) else scale, group, kind, eps, dt)
        return (y if block is not None else None), h

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh):
        x, block, gate, post, pre, dev, stats = ctx.saved_tensors
        scale, group, kind, eps, dt = ctx.rest
        if dy is None and dh is None:
            return (None,) * 10
        need = ctx.needs_input_grad
        d = x.shape[-1]
        rows = x.numel() // d
        dy = None if dy is None else dy.contiguous()
        dh = None if dh is None else dh.contiguous()
        like = lambda t, on: torch.empty_like(t) if t is not None and on else None  # noqa: E731
        dx, db, dg, dpost, dpre = (like(t, n) for t, n in zip((x, block, gate, post, pre), need))
        ds = like(dev, need[5])
        wide = ctx.gate_shape is not None and dg is not None
        if wide:  # summed below: in fp32
            dg = torch.empty(x.shape, dtype=torch.float32, device=x.device)
        if rows == 0:
            for t in (dg, dpost, dpre, ds):
                if t is not None:
                    t.zero_()
            if wide:
                dg = torch.zeros(ctx.gate_shape, dtype=dt, device=x.device)
            return dx, db, dg, dpost, dpre, ds, None, None, None, None
        lib = device.get_metal_bridge()
        size = lib.kans_residual_norm_workspace(rows, d, group if gate is not None else 0)
        ws = torch.empty(size, dtype=torch.uint8, device=x.device)
        device.check(lib.kans_residual_norm_backward(
            _DT[x.dtype], _DT[dt], kind, x.data_ptr(), _ptr(block), _ptr(gate), group, _ptr(post), _ptr(pre), _ptr(dev),
            scale, eps, stats.data_ptr(), _ptr(dy), _ptr(dh), _ptr(dx), _ptr(db), _ptr(dg),
            int(wide), _ptr(dpost), _ptr(dpre), _ptr(ds), rows, d, ws.data_ptr(), size,
            _current_stream(x.device)), "kans_residual_norm_backward")
        if wide:
            dg = dg.sum_to_size(ctx.gate_shape).to(dt)
        return dx, db, dg, dpost, dpre, ds, None, None, None, None


def _gate_rows(gate: torch.Tensor, x: torch.Tensor):
    """The gate as rows that each serve ``group`` consecutive rows of x: (gate, group).  Group 0: it
    repeats in another way (over a leading dimension, or within a row)."""
    lead, d = x.shape[:-1], x.shape[-1]
    g = (1,) * (x.dim() - gate.dim()) + tuple(gate.shape)
    if gate.dim() > x.dim() or any(a not in (1, b) for a, b in zip(g, x.shape)):
        raise ValueError(f"gate of shape {tuple(gate.shape)} does not broadcast to {tuple(x.shape)}")
    if g[-1] == d:
        n = len(lead)
        while n > 0 and g[n - 1] == 1:
            n -= 1
        if g[:n] == tuple(lead[:n]):
            group = 1
            for size in lead[n:]:
                group *= size
            return gate.contiguous(), group
    return gate, 0


def _refuse(x, block, gate, scale, post_weight, pre_weight, dt) -> None:
    d = x.shape[-1]
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
    if not isinstance(scale, torch.Tensor):
        scale = float(scale)
    # (the tests of a call that passes, quickly; a call that does not is told why)
    gpu, vec = x.get_device(), x.shape[-1:]
    if not (dt in _DT and gpu >= 0 and (x.dtype is dt or x.dtype is torch.float32)
            and (block is None or (block.shape == x.shape and block.dtype is dt and block.get_device() == gpu))
            and (gate is None or (gate.dtype is dt and gate.get_device() == gpu))
            and (post_weight is None or (post_weight.shape == vec and post_weight.dtype is dt and post_weight.get_device() == gpu))
            and (pre_weight is None or (pre_weight.shape == vec and pre_weight.dtype is dt and pre_weight.get_device() == gpu))
            and (type(scale) is float or (scale.numel() == 1 and scale.dtype is torch.float32 and scale.get_device() == gpu))):
        _refuse(x, block, gate, scale, post_weight, pre_weight, dt)
    rows = x.numel() // d
    group = max(rows, 1)
    if gate is not None:
        gate, group = _gate_rows(gate, x)
    xc = x.contiguous()
    block = block.contiguous() if block is not None else None
    post = post_weight.contiguous() if post_weight is not None else None
    pre = pre_weight.contiguous() if pre_weight is not None else None
    inputs = (xc, block, gate, post, pre, scale)
    if torch.is_grad_enabled() and any(t.requires_grad for t in inputs if isinstance(t, torch.Tensor)):
        y, h = _ResidualNorm.apply(*inputs, group, _KINDS[kind], float(eps), dt)
    else:
        if group == 0:
            gate, group = gate.expand(x.shape).contiguous(), 1
            inputs = (xc, block, gate, post, pre, scale)
        y, h, _ = _forward(*inputs, group, _KINDS[kind], float(eps), dt, False)
    return (x if block is None else y), h
