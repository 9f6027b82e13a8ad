"""The native torch entry points of the paged operators (csrc/oc_torch.cpp,
built to _lib/_oc_torch.so beside the library by the Makefile)."""

from __future__ import annotations

import importlib.machinery
import importlib.util
import os

import torch  # noqa: F401  (its libraries are the extension's)

from . import _native as N

PATH = os.path.join(os.path.dirname(N.LIB_PATH), "_oc_torch.so")
_module = None


def ops():
    """The loaded extension (raises if it has not been built)."""
    global _module
    if _module is None:
        N.lib()  # the library itself, with its layout checks
        if not os.path.exists(PATH):
            raise RuntimeError(f"orthocache_gpu: native extension {PATH} is missing; build it with "
                               "`make -C orthocache-gpu_amd` (or __graft_entry__.build()). There is no fallback.")
        loader = importlib.machinery.ExtensionFileLoader("_oc_torch", PATH)
        spec = importlib.util.spec_from_loader("_oc_torch", loader)
        module = importlib.util.module_from_spec(spec)
        loader.exec_module(module)
        _module = module
    return _module


def number(x, what: str) -> float:
    """A Python number: a tensor would be read back from the GPU."""
    if isinstance(x, torch.Tensor):
        raise TypeError(f"{what} is a number here, not a tensor")
    return float(x)
