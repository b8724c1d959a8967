"""Attention operators over a key/value cache, callable on their own and inside compiled graphs.

The reference's only attention is ``scaled_dot_product_attention`` over q, k and v of one length
(``conductor/codegen/operator_registry.py:489-500`` lists no other); serving a decoder needs these two:

* :func:`window_attention` -- causal attention over a cache with a sliding window and a few first
  tokens that stay visible, for prompts, chunks of prompts and single tokens;
* :func:`prefix_attention` -- causal attention of a batch whose sequences share a prefix, which is
  read once for all of them.

Both work on CUDA tensors directly (asynchronously, on the current stream of the tensors' device) and
in a function compiled with ``backend='gcu'``, where they become one launch of the plan.  They are
forward-only, like the framework's other attention: a call that would need gradients, backward or forward-mode, raises.
Calls under a tracer, a dispatch mode or a function transform, and calls with tensor subclasses, go through torch's
dispatcher as ``torch.ops.conductor.*``.

Common to both: ``q`` is ``[B, Hq, Sq, D]``, the cache ``[B, Hkv, Skv, D]``, ``Hq`` a multiple of ``Hkv``
(query heads ``h*G .. h*G + G-1`` share key head ``h``); bf16 or f16; ``D`` 64 or 128.  Views are read in
place when ``D`` is contiguous and the other strides are multiples of 8 elements, otherwise they are
gathered first (and so are views made inside a compiled function).  ``lengths`` (``[B]``, int32 or int64, on the same device) is how many keys each
sequence uses, clamped to ``0 .. Skv``; what the cache holds behind them does not matter.  Query ``i`` stands
at position ``p = L - Sq + i``; a query with ``p < 0`` sees nothing, and a query that sees nothing
returns 0.  ``scale`` defaults to ``1 / sqrt(D)`` and is positive (a constant inside compiled functions).  The result is contiguous ``[B, Hq, Sq, D]``.
Among the keys in use, a non-finite value of ``k`` or ``v`` that some queries see and others do not may reach the others too
(0 times infinity); with ``Sq = 1`` hidden keys may hold anything.
"""
from __future__ import annotations

import ctypes
import functools
import operator
import threading
from typing import Optional

import torch
import torch.autograd.forward_ad as fwAD
from torch.overrides import has_torch_function, has_torch_function_variadic

from .codegen.kernel_templates import CdrLaunchItem, CdrTensor, prefix_attention_launch, window_attention_launch
from .compiler.executor import attention_view_ok, get_executor, make_descriptors, raise_for_status
from .compiler.loader import load_call_module, load_library
from .utils.exceptions import DeviceError, ExecutionError
from .utils.type_mapping import to_cdr_dtype

__all__ = ["window_attention", "prefix_attention"]


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int, sinks: int = 0, *,
                     lengths: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """``softmax(scale * q k^T) v`` over the keys ``j <= p`` with ``j > p - window`` or ``j < sinks``.

    ``window >= 1`` counts the query's own position; a window as long as the cache is plain causal
    attention.  ``Sq = 1`` is a decode step over a cache that already holds the new token's key and
    value, ``Sq = Skv`` a prompt, anything between a chunk of a prompt behind a filled cache."""
    if torch.compiler.is_compiling():
        # plans hold both as constants: an argument that changes from call to call makes another plan
        window, sinks = operator.index(window), operator.index(sinks)
        return torch.ops.conductor.window_attention(q, k, v, window, sinks, lengths, scale)
    if q.__class__ is not torch.Tensor and has_torch_function_variadic(q):
        return torch.ops.conductor.window_attention(q, k, v, window, sinks, lengths, scale)
    return _run_window(q, k, v, window, sinks, lengths, scale, _direct_run)


def prefix_attention(q: torch.Tensor, prefix_k: torch.Tensor, prefix_v: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
                     lengths: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """``softmax(scale * q [prefix_k; k]^T) [prefix_v; v]``: every query with ``p >= 0`` sees the whole prefix
    (``[Hkv, P, D]``, ``P >= 0``, the same for all sequences) and the keys ``j <= p`` of its own sequence."""
    if torch.compiler.is_compiling() or (q.__class__ is not torch.Tensor and has_torch_function_variadic(q)):
        return torch.ops.conductor.prefix_attention(q, prefix_k, prefix_v, k, v, lengths, scale)
    return _run_prefix(q, prefix_k, prefix_v, k, v, lengths, scale, _direct_run)


# ---------------------------------------------------------------- direct calls
# A decode step takes about as long on the GPU as a few Python statements do on the host, so a repeated
# call (same shapes, strides, types and parameters) only refreshes pointers: its descriptors, parameter
# block and launch item are kept per thread, and the compiled call module checks the tensors against them, takes
# output and scratch from torch's caching allocator and launches.  Nothing of the tensors themselves is kept.
_calls = threading.local()
_MAX_CALLS = 256


class _Call:
    """A marshalled launch for tensors of given shapes, strides and types on one device."""

    __slots__ = ("name", "call", "keep")

    def __init__(self, launch, tensors):
        lib = load_library()
        in_desc, out_desc = make_descriptors(tensors), (CdrTensor * 1)()
        out = torch.empty(launch.out_shapes[0], dtype=launch.out_dtypes[0], device="meta")
        out_desc[0].dtype, out_desc[0].rank = to_cdr_dtype(out.dtype), out.dim()
        for i, (n, st) in enumerate(zip(out.shape, out.stride())):
            out_desc[0].shape[i], out_desc[0].stride[i] = n, st
        params, size = ctypes.cast(ctypes.byref(launch.params), ctypes.c_void_p), ctypes.sizeof(launch.params)
        need = ctypes.c_size_t(0)
        out_desc[0].data = tensors[0].data_ptr()      # any valid pointer: only the size is asked for
        with torch.cuda.device(tensors[0].device):
            rc = lib.cdr_workspace_bytes(launch.template, in_desc, len(tensors), out_desc, 1, params, size, ctypes.byref(need))
        raise_for_status(lib, rc, launch.name)
        item = CdrLaunchItem(launch.template, len(tensors), 1, 0, ctypes.addressof(in_desc), ctypes.addressof(out_desc),
                             params.value, size, None, need.value)
        self.name = launch.name
        self.call = load_call_module().Call(ctypes.addressof(item), ctypes.addressof(in_desc), ctypes.addressof(out_desc),
                                    ctypes.cast(lib.cdr_launch_many, ctypes.c_void_p).value, tuple(tensors))
        self.keep = (launch, item, in_desc, out_desc)

    def __call__(self, tensors):
        """The output, or None when the tensors are not the ones this call was made for."""
        out = self.call.run(*tensors)
        if out.__class__ is int:
            raise_for_status(load_library(), out, self.name)
        return out


def _run(name, build, params, tensors, other):
    try:
        call = _calls.last.get((name, params))
    except AttributeError:                         # this thread's first call
        _calls.last, _calls.cache, call = {}, {}, None
    if call is not None:
        out = call(tensors)
        if out is not None:
            return out
    return other(name, build, params, tensors)


def _direct_run(name, build, params, tensors):
    """A direct call that is not the last one of its parameters again; left to the dispatcher where something besides the
    kernel has to see it."""
    special = [t for t in tensors if type(t) not in (torch.Tensor, torch.nn.Parameter)]
    if has_torch_function(special):
        return _dispatched(name, params, tensors)
    if not all(isinstance(t, torch.Tensor) for t in special):
        raise ExecutionError(f"{name}: expected tensors, got {[type(t).__name__ for t in tensors]}", kernel_name=name)
    if special:
        return _dispatched(name, params, tensors)
    if tensors[0].device.type == "cuda" and load_call_module().is_dispatched(*tensors):
        return _dispatched(name, params, tensors)
    return _other_run(name, build, params, tensors)


def _other_run(name, build, params, tensors):
    """The kernel's call: found among the kept ones, or made."""
    device = tensors[0].device
    if device.type != "cuda":
        raise DeviceError(f"{name}: kernel templates run on CUDA tensors, got {device}")
    for t in tensors:
        if t.device != device:
            raise ExecutionError(f"{name}: tensors on {device} and {t.device}", kernel_name=name)
    _refuse_gradients(name, tensors)
    key = (name, params, *[(t.shape, t.stride(), t.dtype) for t in tensors], device)
    call = _calls.cache.get(key)
    out = call(tensors) if call is not None else None
    if out is None:
        launch = build(tensors[0], *params)
        if any(not attention_view_ok(t) for t in tensors):
            return get_executor().execute(launch, tensors)[0]      # gathers what cannot be read in place
        if len(_calls.cache) >= _MAX_CALLS:
            _calls.cache.clear()
            _calls.last.clear()
        call = _calls.cache[key] = _Call(launch, tensors)
        out = call(tensors)
        if out is None:                                            # a tensor subclass: the general way
            return get_executor().execute(launch, tensors)[0]
    _calls.last[(name, params)] = call
    return out


def _autograd_run(name, build, params, tensors):
    """The operators' autograd kernel where the kept call does not apply: there is no gradient to give."""
    _refuse_gradients(name, tensors)
    with torch._C._AutoDispatchBelowAutograd():
        return _dispatched(name, params, tensors)


def _dispatched(name, params, tensors):
    *numbers, has_lengths, scale = params
    lengths = tensors[-1] if has_lengths else None
    return getattr(torch.ops.conductor, name)(*(tensors[:-1] if has_lengths else tensors), *numbers, lengths, scale)


def _refuse_gradients(name, tensors):
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise ExecutionError(f"{name}: an input requires grad but the operator has no backward; call it under "
                             "torch.no_grad() or detach the inputs", kernel_name=name)
    if fwAD._current_level >= 0 and fwAD._is_fwd_grad_enabled() and any(fwAD.unpack_dual(t).tangent is not None for t in tensors):
        raise ExecutionError(f"{name}: an input has a forward-mode gradient but the operator has no such formula; detach "
                             "the inputs", kernel_name=name)


def _build_window(q, window, sinks, has_lengths, scale):
    return window_attention_launch("window_attention", q.shape, q.dtype, window, sinks, has_lengths, scale)


def _build_prefix(q, has_lengths, scale):
    return prefix_attention_launch("prefix_attention", q.shape, q.dtype, has_lengths, scale)


def _run_window(q, k, v, window, sinks=0, lengths=None, scale=None, other=_other_run):
    window, sinks, scale = operator.index(window), operator.index(sinks), None if scale is None else float(scale)
    if lengths is None:
        return _run("window_attention", _build_window, (window, sinks, False, scale), (q, k, v), other)
    return _run("window_attention", _build_window, (window, sinks, True, scale), (q, k, v, lengths), other)


def _run_prefix(q, prefix_k, prefix_v, k, v, lengths=None, scale=None, other=_other_run):
    scale = None if scale is None else float(scale)
    if lengths is None:
        return _run("prefix_attention", _build_prefix, (False, scale), (q, prefix_k, prefix_v, k, v), other)
    return _run("prefix_attention", _build_prefix, (True, scale), (q, prefix_k, prefix_v, k, v, lengths), other)


# ---------------------------------------------------------------- graph form
_lib = torch.library.Library("conductor", "DEF")
_lib.define("window_attention(Tensor q, Tensor k, Tensor v, int window, int sinks=0, Tensor? lengths=None, float? scale=None) -> Tensor")
_lib.define("prefix_attention(Tensor q, Tensor prefix_k, Tensor prefix_v, Tensor k, Tensor v, Tensor? lengths=None, float? scale=None) -> Tensor")
_lib.impl("window_attention", _run_window, "CUDA")
_lib.impl("prefix_attention", _run_prefix, "CUDA")
_lib.impl("window_attention", functools.partial(_run_window, other=_autograd_run), "Autograd")
_lib.impl("prefix_attention", functools.partial(_run_prefix, other=_autograd_run), "Autograd")


@torch.library.register_fake("conductor::window_attention", lib=_lib)
def _(q, k, v, window, sinks=0, lengths=None, scale=None):
    return torch.empty(q.shape, dtype=q.dtype, device=q.device)


@torch.library.register_fake("conductor::prefix_attention", lib=_lib)
def _(q, prefix_k, prefix_v, k, v, lengths=None, scale=None):
    return torch.empty(q.shape, dtype=q.dtype, device=q.device)
