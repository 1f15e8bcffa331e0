"""The torch binding of the 8-bit and training operators (``binding/ops.cpp``, built by ``build.py`` next to the CUDA
library it calls)."""

from __future__ import annotations

import importlib.util
from pathlib import Path

from . import _lib

OPS_PATH = Path(__file__).resolve().with_name("_native_ops.so")
_ops = None


def ops():
    """The extension module, loaded once (raises if it was not built)."""

    global _ops
    if _ops is None:
        _lib.load()
        if not OPS_PATH.exists():
            raise RuntimeError(f"{OPS_PATH.name} is not built; run `python -m convrot_mlx_b200.build` "
                               "(there is no fallback)")
        spec = importlib.util.spec_from_file_location("_native_ops", OPS_PATH)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        _ops = module
    return _ops
