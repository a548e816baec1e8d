"""metal_kans (MI355X build): fused KAN layer forward on hand-written gfx950 HIP kernels.

Drop-in for the hot-path surface of Shuril/metal-kans (metal_kans/__init__.py:6-40):
Chebyshev / Gaussian-RBF / cubic B-spline layers, the multi-layer container, the
GatedKAN block, INT8 / INT4 / ternary weight quantization, the Chebyshev layer
backward and the torch modules.  Around them, on torch tensors, the rest of a training
step: ``residual_norm``, ``linear_cross_entropy`` and ``TorchAdamW``.  The reference's NumPy
optimizers, pruning, symbolic export and the other KAN families are outside this build's scope.
"""
from .device import get_metal_bridge, is_gpu_available, is_metal_available, set_async, sync
from .cheby_kan import ChebyKAN
from .fast_kan import FastKAN
from .bspline_kan import BSplineKAN, KAN
from .metal_kan import MetalKAN
from .gated_kan import GatedKAN
from .quantization import (QuantizedWeight, TernaryQuantizedWeight, quantize, to_int4, to_int8, to_ternary)

__version__ = "0.6.0+mi355x"


# What works on torch tensors and the module it is in: imported on first use so that `import metal_kans` does
# not import torch; None without torch, as in the reference (metal_kans/__init__.py:34-38).
_TORCH = {"TorchMetalKANLinear": "torch_module", "TorchMetalKAN": "torch_module", "TorchAdamW": "adamw",
          "residual_norm": "residual", "linear_cross_entropy": "cross_entropy"}


def __getattr__(name):
    if name in _TORCH:
        from importlib import import_module
        try:
            import torch  # noqa: F401
        except ImportError:
            return None
        # (kept: the module's own name from here on, without this function's few microseconds at each use)
        value = globals()[name] = getattr(import_module("." + _TORCH[name], __name__), name)
        return value
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")

__all__ = [
    "set_async", "sync", "get_metal_bridge", "is_metal_available", "is_gpu_available",
    "ChebyKAN", "FastKAN", "BSplineKAN", "KAN", "MetalKAN", "GatedKAN",
    "QuantizedWeight", "TernaryQuantizedWeight", "quantize", "to_int8", "to_int4", "to_ternary",
    "TorchMetalKANLinear", "TorchMetalKAN", "TorchAdamW", "residual_norm", "linear_cross_entropy",
]
