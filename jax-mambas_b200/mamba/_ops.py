"""The host side of rms_norm, fp8 and sampling: the module lib/_mamba_ops.so
(csrc/torch_ext/mamba_ops.cpp), which checks arguments, allocates outputs and
carries autograd in C++ over the C ABI of the library that the process has
loaded. Built by build.py (the CMake recipe gives the C library alone); without it
the calls raise."""
from __future__ import annotations

import ctypes
import importlib.util

from . import _native
from .selective_scan_cuda import _lib

_OPS = None


def ops():
    """The module, bound to the library; loaded once."""
    global _OPS
    if _OPS is None:
        lib = _lib()
        path = _native._PKG_ROOT / "lib" / "_mamba_ops.so"
        if not path.is_file():
            raise FileNotFoundError("The PyTorch binding of the operators is not built (python "
                                    f"jax-mambas_b200/build.py); searched: {path}")
        spec = importlib.util.spec_from_file_location("_mamba_ops", path)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        module.bind({name: ctypes.cast(getattr(lib, name), ctypes.c_void_p).value
                     for name in _native.SIGNATURES})
        _OPS = module
    return _OPS
