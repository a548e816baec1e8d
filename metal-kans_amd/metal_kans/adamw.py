"""AdamW over all tensors of a model at once, on the gfx950 kernel of ``kans_adamw_step``.

``TorchAdamW`` is a ``torch.optim.Optimizer`` for parameters on the GPU: fp32, fp16 or bf16 (16-bit ones
with an fp32 master in the state), the two moments in 32 bits or, with ``state_bits=8``, in 8.  One launch
updates up to 96 tensors; the step is enqueued on torch's current stream.

The states of a group's parameters of one dtype lie in one buffer per kind, each parameter's at a
multiple of 256 elements in the order of the group; ``state[p]`` holds views of them, ``flat_state()`` the
buffers.  Per parameter:

* ``step`` (int) and ``exp_avg``, ``exp_avg_sq`` in the parameter's shape: fp32, or with ``state_bits=8``
  int8 / uint8 codes with ``exp_avg_scale``, ``exp_avg_sq_scale`` (one fp32 each per 256 elements);
  the values that codes stand for are ``scale * (q / 127) * |q / 127|`` and ``scale * (q / 255) ** 4``;
* ``master`` (16-bit parameters): the fp32 value that the parameter is the rounding of.

A tensor that a program puts in one's place is copied into the buffer by the next step.

Gradients that are None leave their parameter alone.  Parameters are dense in memory, in any order of their dimensions;
fp32 states follow a parameter into another order, 8-bit ones refuse it (``state.clear()`` starts anew).  A 16-bit
parameter that was changed between steps (a loaded model; by its version or address, which an edit through ``.data`` moves
neither) gives its master its value where it is not the master's rounding any more.  A step on a
capturing stream is refused (its bias corrections belong to that one step).
"""
from __future__ import annotations

from array import array
from typing import Dict, List

import torch

from . import device
from ._engine import DT_BF16, DT_F16, DT_F32
from ._torch_ops import load
from .torch_module import _current_stream

_DT = {torch.float32: DT_F32, torch.float16: DT_F16, torch.bfloat16: DT_BF16}
BLOCK = 256  # elements that share a scale of the 8-bit states


class _Arena:
    """The states of one group's parameters of one dtype."""

    def __init__(self, params: List[torch.Tensor], bits: int):
        p0 = params[0]
        self.params = params
        self.bits = bits
        self.dtype, self.device = p0.dtype, p0.device
        self.numel = [p.numel() for p in params]
        self.blocks = []
        total = 0
        for n in self.numel:
            self.blocks.append(total)
            total += (n + BLOCK - 1) // BLOCK
        self.total = total
        zeros = lambda n, dt: torch.zeros(n, dtype=dt, device=self.device)  # noqa: E731
        f32 = torch.float32
        self.flat: Dict[str, torch.Tensor] = {
            "exp_avg": zeros(total * BLOCK, torch.int8 if bits == 8 else f32),
            "exp_avg_sq": zeros(total * BLOCK, torch.uint8 if bits == 8 else f32)}
        if bits == 8:
            self.flat["exp_avg_scale"] = zeros(total, f32)
            self.flat["exp_avg_sq_scale"] = zeros(total, f32)
        if self.dtype != f32:
            self.flat["master"] = zeros(total * BLOCK, f32)
        self.numel_q, self.blocks_q = array("q", self.numel), array("q", self.blocks)
        self.seen = array("q", [-1] * (2 * len(params)))  # address and version behind the last step

    def views(self, i: int) -> Dict[str, torch.Tensor]:
        b, n, shape = self.blocks[i], self.numel[i], self.params[i].shape
        out = {}
        for name, t in self.flat.items():
            if name.endswith("_scale"):
                out[name] = t[b:b + (n + BLOCK - 1) // BLOCK]
            else:
                # in the parameter's own order of memory
                out[name] = t[b * BLOCK:b * BLOCK + n].as_strided(shape, self.params[i].stride(), b * BLOCK)
        return out

    def start(self, i: int, state: dict) -> dict:
        """The state of parameter i in its present order of memory: zeros and its value, or what ``state`` holds."""
        p = self.params[i]
        if not _dense(p):
            raise ValueError(_NOT_DENSE)
        views = self.views(i)
        given = {name: state.get(name) for name in views}
        for name, v in views.items():
            g = given[name]
            if g is None:
                if state and name != "master":
                    raise ValueError(f"state {name!r} is missing (states in {self.bits} bits)")
                continue
            if g.shape != v.shape or (g.is_floating_point() != v.is_floating_point()):
                raise ValueError(f"state {name!r} of a parameter of shape {tuple(p.shape)} is {g.dtype} "
                                 f"{tuple(g.shape)}, expected {v.dtype} {tuple(v.shape)}")
            # (blocks of elements in this order share a scale)
            if not g.is_floating_point() and _order(g) != _order(v):
                raise ValueError(f"8-bit state {name!r} has strides {g.stride()}, its parameter {v.stride()}: codes belong to one "
                                 "order of memory")
            if g.device == v.device and g.untyped_storage().data_ptr() == v.untyped_storage().data_ptr():
                given[name] = g.clone()  # the places that are written below, maybe in another order
        for name, v in views.items():
            if given[name] is not None:
                v.copy_(given[name])
            elif name == "master":
                v.copy_(p.detach())
            else:
                v.zero_()
        return {"step": int(state.get("step", 0)), **views}

    def follow(self, i: int) -> None:
        """Parameter i's master where the parameter is not its rounding any more: its value."""
        p, master = self.params[i].detach(), self.views(i)["master"]
        if p.dtype != self.dtype or p.device != self.device:
            return  # (the step refuses it)
        torch.where(master.to(p.dtype) == p, master, p.float(), out=master)


_NOT_DENSE = "parameters must be dense (no gaps or overlaps in memory)"


def _order(t: torch.Tensor) -> tuple:
    """The dimensions as they lie in memory, the slowest first."""
    return tuple(sorted((i for i in range(t.dim()) if t.shape[i] > 1), key=lambda i: -t.stride(i)))


def _dense(p: torch.Tensor) -> bool:
    """Whether the elements fill p.numel() consecutive places (in any order of the dimensions)."""
    if p.is_contiguous():
        return True
    at = 1
    for size, stride in sorted(zip(p.shape, p.stride()), key=lambda v: v[1]):
        if size != 1:
            if stride != at:
                return False
            at *= size
    return True


def _refuse_variants(group: dict) -> None:
    """Options of torch's AdamW, as in the state it saves, that make another step than this one."""
    for name in ("amsgrad", "maximize"):
        if group.get(name):
            raise ValueError(f"TorchAdamW has no {name!r}")


class TorchAdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) on device tensors.

    Args:
        params: parameters or parameter groups (``lr``, ``betas``, ``eps``, ``weight_decay`` per group)
        lr, betas, eps, weight_decay: as in the formula p = p (1 - lr wd) - lr m^ / (sqrt(v^) + eps)
        state_bits: 32 or 8, the moments' width (for all groups)
    """

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
                 state_bits: int = 32):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        self.state_bits = state_bits
        self._arenas: Dict[int, List[_Arena]] = {}
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))

    def add_param_group(self, group) -> None:
        super().add_param_group(group)
        g = self.param_groups[-1]
        try:
            b1, b2 = g["betas"]
            if not (g["lr"] >= 0 and g["eps"] >= 0 and g["weight_decay"] >= 0):
                raise ValueError("lr, eps and weight_decay must be >= 0")
            if not (0 <= b1 < 1 and 0 <= b2 < 1):
                raise ValueError(f"betas must be in [0, 1), got {g['betas']}")
            _refuse_variants(g)
            for p in g["params"]:
                if p.dtype not in _DT:
                    raise TypeError(f"unsupported parameter dtype {p.dtype}")
                if not _dense(p):
                    raise ValueError(_NOT_DENSE)
        except Exception:
            self.param_groups.pop()
            raise

    # ---- states ----------------------------------------------------------------
    def _group_arenas(self, gi: int) -> List[_Arena]:
        arenas = self._arenas.get(gi)
        if arenas is None:
            kinds: Dict[tuple, List[torch.Tensor]] = {}
            for p in self.param_groups[gi]["params"]:
                if not p.is_cuda:
                    raise ValueError("TorchAdamW takes parameters on the GPU")
                kinds.setdefault((p.dtype, p.device), []).append(p)
            arenas = []
            for params in kinds.values():
                a = _Arena(params, self.state_bits)
                for i, p in enumerate(params):
                    if self.state.get(p):
                        self.state[p] = a.start(i, self.state[p])
                arenas.append(a)
            self._arenas[gi] = arenas
        return arenas

    def flat_state(self) -> List[Dict[str, torch.Tensor]]:
        """The states as flat buffers, one dict for each parameter group and dtype: ``exp_avg`` and
        ``exp_avg_sq`` in fp32 (the buffers themselves, or in 8 bits the values of the codes), ``master`` for
        16-bit parameters, and ``params``.  A parameter's elements start at the sum of the sizes before it, each rounded
        up to 256; what lies between is zero."""
        out = []
        for gi in range(len(self.param_groups)):
            for a in self._group_arenas(gi):
                load().adamw_hold(self.state, a.params, a.blocks_q, a.flat, lambda i, a=a: self._start(a, i))
                flat = dict(a.flat)
                if self.state_bits == 8:
                    avg, sq = (torch.empty(a.total * BLOCK, device=a.device) for _ in range(2))
                    stream = _current_stream(a.device)
                    device.check(device.get_metal_bridge().kans_adamw_values(
                        flat["exp_avg"].data_ptr(), flat["exp_avg_sq"].data_ptr(), flat.pop("exp_avg_scale").data_ptr(),
                        flat.pop("exp_avg_sq_scale").data_ptr(), avg.data_ptr(), sq.data_ptr(), a.total, stream),
                        "kans_adamw_values")
                    flat["exp_avg"], flat["exp_avg_sq"] = avg, sq
                flat["params"] = a.params
                out.append(flat)
        return out

    def state_dict(self):
        sd = super().state_dict()
        sd["state_bits"] = self.state_bits
        return sd

    def load_state_dict(self, state_dict) -> None:
        """As torch's, its hooks included, with the states kept in their own types; refuses states of the other width."""
        state_dict = dict(state_dict)
        for hook in self._optimizer_load_state_dict_pre_hooks.values():
            other = hook(self, state_dict)
            if other is not None:
                state_dict = other
        bits = state_dict.get("state_bits", self.state_bits)
        if bits != self.state_bits:
            raise ValueError(f"the states are in {bits} bits, the optimizer's in {self.state_bits}")
        groups = state_dict["param_groups"]
        if [len(g["params"]) for g in groups] != [len(g["params"]) for g in self.param_groups]:
            raise ValueError("the parameter groups differ in number or size")
        for g in groups:
            _refuse_variants(g)
        state, arenas = dict(self.state), self._arenas
        loaded = {}
        for g, sg in zip(self.param_groups, groups):
            for p, key in zip(g["params"], sg["params"]):
                if state_dict["state"].get(key):
                    loaded[p] = dict(state_dict["state"][key])
        self.state.clear()
        self.state.update(loaded)
        self._arenas = {}
        try:
            for gi in range(len(self.param_groups)):
                self._group_arenas(gi)
        except Exception:
            self.state.clear()
            self.state.update(state)
            self._arenas = arenas
            raise
        for g, sg in zip(self.param_groups, groups):
            g.update({k: v for k, v in sg.items() if k != "params"})
        for hook in self._optimizer_load_state_dict_post_hooks.values():
            hook(self)

    def __getstate__(self):
        return {**super().__getstate__(), "state_bits": self.state_bits}

    def __setstate__(self, state) -> None:
        super().__setstate__(state)
        self._arenas = {}  # made anew around the states at the next step

    # ---- step --------------------------------------------------------------------
    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        arenas = [(group, a) for gi, group in enumerate(self.param_groups) for a in self._group_arenas(gi)]
        masters = [a for _, a in arenas if "master" in a.flat]
        for a in masters:
            load().adamw_follow(self.state, a.params, a.blocks_q, a.flat, lambda i, a=a: self._start(a, i), a.seen, a.follow)
        for group, a in arenas:
            b1, b2 = group["betas"]
            load().adamw_step(self.state, a.params, a.numel_q, a.blocks_q, a.flat, _DT[a.dtype], a.bits,
                              lambda i, a=a: self._start(a, i), group["lr"], b1, b2, group["eps"], group["weight_decay"], a.seen)
        for a in masters:
            load().adamw_seen(a.params, a.seen)
        return loss

    def _start(self, a: _Arena, i: int) -> None:
        self.state[a.params[i]] = a.start(i, self.state.get(a.params[i], {}))
