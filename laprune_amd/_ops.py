"""Compiled torch binding of the decode path's hot entry points.

``laprune_amd/_lib/liblaprune_torch.so`` (built in-tree by
``laprune_amd.build`` from ``csrc/torch_ops.cpp`` with hipcc against the
installed torch headers) registers torch custom ops in the ``laprune``
namespace, each a direct call into the C ABI of ``liblaprune_hip.so``: sizes
and strides come from the tensors and the stream is the tensors' current
torch stream, so a call costs one dispatcher hop instead of marshalling
every argument through ctypes.  Eager decode (the reference's call pattern,
one call per layer per token) goes through these ops; the rest of the C ABI
stays bound by ctypes (``_native``).  Loading raises when the library is
missing: there is no fallback.
"""
from __future__ import annotations

import threading
from pathlib import Path

import torch
from torch.autograd import forward_ad
from torch.utils._device import DeviceContext

from . import _native as N

LIB_PATH = Path(__file__).resolve().parent / "_lib" / "liblaprune_torch.so"

_lock = threading.Lock()
_ops = None

# looked up once: every wrapped call of an eager step asks them
_compiling, _grad_on = torch.compiler.is_compiling, torch.is_grad_enabled
_transforms, _modes = torch._C._functorch.peek_interpreter_stack, torch._C._len_torch_dispatch_stack
_trace = torch._C._get_tracing_state
_functions, _function_mode = torch._C._len_torch_function_stack, torch._C._get_function_stack_at


def _function_modes() -> bool:
    """Whether a function mode other than a default device looks on."""
    return any(type(_function_mode(i)) is not DeviceContext for i in range(_functions()))


def untraced() -> bool:
    """Whether no compiler, function transform (vmap, jvp), forward-mode level, dispatch
    mode (fake tensors, op counters), function mode or trace looks at the calling ops, all
    of which a kernel call would pass by."""
    return not (_compiling() or forward_ad._current_level >= 0 or _transforms() is not None or
                _modes() or _trace() is not None or (_functions() and _function_modes()))


def unwatched() -> bool:
    """Whether the calling ops only have to compute: untraced, and no gradients."""
    return not _grad_on() and untraced()


def ops():
    """``torch.ops.laprune`` after loading the binding (raises if it is not built)."""
    global _ops
    if _ops is not None:  # set once, after the load
        return _ops
    with _lock:
        if _ops is None:
            if not LIB_PATH.exists():
                raise RuntimeError(f"laprune_amd torch binding not built: {LIB_PATH} is missing "
                                   "(run `python -c 'import __graft_entry__ as g; g.build()'`)")
            N.lib()  # the HIP library it links against, loaded once from the same path
            torch.ops.load_library(str(LIB_PATH))
            _ops = torch.ops.laprune
        return _ops
