"""The compiled torch operators of ``csrc/kans_torch.cpp``, bound to the library that ``device`` loaded."""
from __future__ import annotations

import ctypes

import torch  # noqa: F401  (the module below needs its libraries)

from . import device

_FUNCTIONS = ("kans_last_error", "kans_stream_keep", "kans_residual_norm_forward", "kans_residual_norm_workspace",
              "kans_residual_norm_backward", "kans_linear_xent_workspace", "kans_linear_xent_forward",
              "kans_linear_xent_backward", "kans_adamw_step")
_module = None


def load():
    """The module.  Raises RuntimeError where it is not built, or for another torch."""
    global _module
    if _module is None:
        lib = device.load_library()
        try:
            from . import _kans_torch
        except ImportError as e:
            raise RuntimeError(f"metal_kans/_kans_torch.so does not load ({e}); build it with metal-kans_amd/build.py") from e
        _kans_torch.bind({n: ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in _FUNCTIONS}, device.KansError)
        _module = _kans_torch
    return _module
