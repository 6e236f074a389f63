"""Load the required torch host module ``nimbleml_b200_host`` (csrc/torch_host.cpp).

It checks arguments, allocates and queues the kernels of the operators whose calls
would otherwise be bound by Python, and holds their autograd nodes. Like the
library itself it has no fallback: a missing module raises ImportError with the
build command.
"""
from __future__ import annotations

import importlib.util

import torch  # noqa: F401  (the module links against torch's libraries)

from nimbleml_b200._native_loader import native  # noqa: F401  (loads the library the module links against)
from nimbleml_b200.build_native import host_module_path


def load_host():
    path = host_module_path()
    hint = (f"nimbleml_b200 requires the compiled module '{path.name}'.\n"
            "Build it from the repo root with:\n  python -m nimbleml_b200.build_native")
    if not path.exists():
        raise ImportError(hint)
    try:
        spec = importlib.util.spec_from_file_location("nimbleml_b200_host", path)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
    except (ImportError, OSError) as exc:
        raise ImportError(f"{hint}\n(load error: {exc})") from exc
    return module


host = load_host()

__all__ = ["host", "load_host"]
