"""Loaders for the in-tree native extensions.

The GPU path never silently falls back to Python: if ``_hip`` cannot be
imported while a GPU fit is requested, :func:`hip` raises with the build
command to run.
"""

from __future__ import annotations

import importlib
from types import ModuleType

import torch

_cache: dict = {}

_PLAIN = {torch.Tensor, torch.nn.Parameter, type(None)}
_no_dispatch = torch._C._disabled_torch_dispatch_impl
_modes = torch._C._len_torch_dispatch_stack
_tracing = torch._C._is_tracing
_Mode = torch._C._TorchDispatchModeKey


def check_memory(*tensors) -> None:
    """Refuse what a kernel that is given addresses would read or write wrongly: tensors whose
    values are not in their own memory (subclasses with a ``__torch_dispatch__``: fake, distributed
    or wrapped tensors), and calls whose torch operations are recorded or faked, where the launch
    itself would leave no trace. (Modes that only watch the operations pass.)"""
    for t in tensors:
        if type(t) not in _PLAIN and type(t).__torch_dispatch__ is not _no_dispatch:
            raise TypeError(f"native kernels take plain tensors, got {type(t).__name__}")
    if _modes() and any(torch._C._get_dispatch_mode(k) is not None
                        for k in (_Mode.PROXY, _Mode.FAKE, _Mode.FUNCTIONAL)):
        raise RuntimeError("native kernels cannot be traced or run on fake tensors")
    if _tracing():
        raise RuntimeError("native kernels cannot be recorded by torch.jit.trace")


def _load(name: str):
    if name not in _cache:
        try:
            _cache[name] = importlib.import_module(f"mpitree_amd.{name}")
        except ImportError as e:  # pragma: no cover - exercised when unbuilt
            _cache[name] = e
    mod = _cache[name]
    if isinstance(mod, Exception):
        raise ImportError(
            f"mpitree_amd native extension '{name}' is not built or failed to load ({mod}); "
            "run `python -m mpitree_amd.ops.build`"
        ) from mod
    return mod


def hip():
    """The gfx950 kernel module (raises if unavailable)."""
    mod = _cache.get("_hip")  # (0.2 us less a call of a kernel)
    return mod if type(mod) is ModuleType else _load("_hip")


def cpu():
    """The native host builder module (raises if unavailable)."""
    return _load("_cpu")


def has_cpu() -> bool:
    try:
        cpu()
        return True
    except ImportError:
        return False


def has_hip() -> bool:
    try:
        hip()
        return True
    except ImportError:
        return False


def host_threads() -> int:
    """Host worker threads for native helpers: ``MPITREE_HOST_THREADS`` or the
    CPUs this process may run on, capped at 16 (one GPU's share of a node)."""
    import os

    env = os.environ.get("MPITREE_HOST_THREADS")
    if env:
        return max(1, int(env))
    try:
        n = len(os.sched_getaffinity(0))
    except (AttributeError, OSError):  # pragma: no cover - non-Linux
        n = os.cpu_count() or 1
    return max(1, min(16, n))
