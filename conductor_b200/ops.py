"""Attention operators over a key/value cache, callable on their own and inside compiled graphs.

The reference's only attention is ``scaled_dot_product_attention`` over q, k and v of one length
(``conductor/codegen/operator_registry.py:489-500`` lists no other); serving a decoder needs these two:

* :func:`window_attention` -- causal attention over a cache with a sliding window and a few first
  tokens that stay visible, for prompts, chunks of prompts and single tokens;
* :func:`prefix_attention` -- causal attention of a batch whose sequences share a prefix, which is
  read once for all of them.

Both work on CUDA tensors directly (asynchronously, on the current stream of the tensors' device) and
in a function compiled with ``backend='gcu'``, where they become one launch of the plan.  They are
forward-only, like the framework's other attention: a call that would need gradients raises.

Common to both: ``q`` is ``[B, Hq, Sq, D]``, the cache ``[B, Hkv, Skv, D]``, ``Hq`` a multiple of ``Hkv``
(query heads ``h*G .. h*G + G-1`` share key head ``h``); bf16 or f16; ``D`` 64 or 128.  Views are read in
place when ``D`` is contiguous and the other strides are multiples of 8 elements, otherwise they are
gathered first.  ``lengths`` (``[B]``, int32 or int64, on the same device) is how many keys each
sequence uses, clamped to ``0 .. Skv``; what the cache holds behind them does not matter.  Query ``i`` stands
at position ``p = L - Sq + i``; a query with ``p < 0`` sees nothing, and a query that sees nothing
returns 0.  ``scale`` defaults to ``1 / sqrt(D)``.  The result is contiguous ``[B, Hq, Sq, D]``.
"""
from __future__ import annotations

import threading
from typing import Optional

import torch

from .codegen.kernel_templates import prefix_attention_launch, window_attention_launch
from .compiler.executor import get_executor
from .utils.exceptions import DeviceError, ExecutionError

__all__ = ["window_attention", "prefix_attention"]


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int, sinks: int = 0, *,
                     lengths: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """``softmax(scale * q k^T) v`` over the keys ``j <= p`` with ``j > p - window`` or ``j < sinks``.

    ``window >= 1`` counts the query's own position; a window as long as the cache is plain causal
    attention.  ``Sq = 1`` is a decode step over a cache that already holds the new token's key and
    value, ``Sq = Skv`` a prompt, anything between a chunk of a prompt behind a filled cache."""
    if torch.compiler.is_compiling():
        return torch.ops.conductor.window_attention(q, k, v, window, sinks, lengths, scale)
    return _run_window(q, k, v, window, sinks, lengths, scale)


def prefix_attention(q: torch.Tensor, prefix_k: torch.Tensor, prefix_v: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
                     lengths: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """``softmax(scale * q [prefix_k; k]^T) [prefix_v; v]``: every query with ``p >= 0`` sees the whole prefix
    (``[Hkv, P, D]``, ``P >= 0``, the same for all sequences) and the keys ``j <= p`` of its own sequence."""
    if torch.compiler.is_compiling():
        return torch.ops.conductor.prefix_attention(q, prefix_k, prefix_v, k, v, lengths, scale)
    return _run_prefix(q, prefix_k, prefix_v, k, v, lengths, scale)


# ---------------------------------------------------------------- direct calls
# A launch object keeps its marshalled descriptors, so one is kept per thread, operator and parameter
# set of recent calls; only data pointers change from call to call.
_calls = threading.local()
_MAX_LAUNCHES = 256


def _launch_for(key, build):
    cache = getattr(_calls, "cache", None)
    if cache is None:
        cache = _calls.cache = {}
    launch = cache.get(key)
    if launch is None:
        if len(cache) >= _MAX_LAUNCHES:
            cache.clear()
        launch = cache[key] = build()
    return launch


def _check(name, tensors):
    device = tensors[0].device
    if device.type != "cuda":
        raise DeviceError(f"{name}: kernel templates run on CUDA tensors, got {device}")
    needs_grad = False
    for t in tensors:
        if t.device != device:
            raise ExecutionError(f"{name}: tensors on {device} and {t.device}", kernel_name=name)
        needs_grad |= t.requires_grad
    if needs_grad and torch.is_grad_enabled():
        raise ExecutionError(f"{name}: an input requires grad but the operator has no backward; call it under "
                             "torch.no_grad() or detach the inputs", kernel_name=name)


def _run_window(q, k, v, window, sinks=0, lengths=None, scale=None):
    tensors = (q, k, v) if lengths is None else (q, k, v, lengths)
    _check("window_attention", tensors)
    key = (window, sinks, scale, lengths is None, q.shape, q.dtype, q.stride(), k.shape, k.stride(), v.stride())
    launch = _launch_for(key, lambda: window_attention_launch("window_attention", q.shape, q.dtype, window, sinks, lengths is not None, scale))
    return get_executor().execute(launch, tensors)[0]


def _run_prefix(q, prefix_k, prefix_v, k, v, lengths=None, scale=None):
    tensors = (q, prefix_k, prefix_v, k, v) if lengths is None else (q, prefix_k, prefix_v, k, v, lengths)
    _check("prefix_attention", tensors)
    key = (scale, lengths is None, q.shape, q.dtype, q.stride(), prefix_k.shape, k.shape, k.stride(), v.stride())
    launch = _launch_for(key, lambda: prefix_attention_launch("prefix_attention", q.shape, q.dtype, lengths is not None, scale))
    return get_executor().execute(launch, tensors)[0]


# ---------------------------------------------------------------- graph form
_lib = torch.library.Library("conductor", "DEF")
_lib.define("window_attention(Tensor q, Tensor k, Tensor v, int window, int sinks=0, Tensor? lengths=None, float? scale=None) -> Tensor")
_lib.define("prefix_attention(Tensor q, Tensor prefix_k, Tensor prefix_v, Tensor k, Tensor v, Tensor? lengths=None, float? scale=None) -> Tensor")
_lib.impl("window_attention", _run_window, "CUDA")
_lib.impl("prefix_attention", _run_prefix, "CUDA")


@torch.library.register_fake("conductor::window_attention", lib=_lib)
def _(q, k, v, window, sinks=0, lengths=None, scale=None):
    return torch.empty(q.shape, dtype=q.dtype, device=q.device)


@torch.library.register_fake("conductor::prefix_attention", lib=_lib)
def _(q, prefix_k, prefix_v, k, v, lengths=None, scale=None):
    return torch.empty(q.shape, dtype=q.dtype, device=q.device)
