"""Attention with a token-exact window and sinks over contiguous BTHD tensors.

``sol_attention`` keeps 64-token blocks around the query and the first blocks exact and folds the
others in through their means; ``window_attention`` sees single tokens and nothing outside the window
and the sinks.  It has no counterpart in the reference.
"""

from __future__ import annotations

import math

import torch

from . import _lib
from .attention import _is_b200
from .status import error_word

# The current stream's handle without the stream object around it (a third of a small call's cost).
current_stream = torch._C._cuda_getCurrentRawStream

# Window and lookahead without a bound, in the C ABI.
_NO_WINDOW, _NO_LOOKAHEAD = 0, -1
_MOST = (1 << 30) - 1
_WORKSPACE: dict = {}


def check_rule(window, lookahead, sink_tokens):
    """(window, lookahead, sink_tokens) of the C ABI, checked."""
    if window is None:
        window = _NO_WINDOW
    elif type(window) is not int or not 0 < window <= _MOST:
        raise ValueError("window must be a positive integer or None")
    if lookahead is None:
        lookahead = _NO_LOOKAHEAD
    elif type(lookahead) is not int or not 0 <= lookahead <= _MOST:
        raise ValueError("lookahead must be a nonnegative integer or None")
    if type(sink_tokens) is not int or not 0 <= sink_tokens <= _MOST:
        raise ValueError("sink_tokens must be a nonnegative integer")
    return window, lookahead, sink_tokens


def check_scale(scale, dim):
    if scale is None:
        return dim ** -0.5
    scale = float(scale)
    if not math.isfinite(scale) or scale <= 0:
        raise ValueError("scale must be finite and positive")
    return scale


def workspace(fn, key, device):
    """(tensor or None, address, bytes) of a call's scratch; its size is cached per shape."""
    size = _WORKSPACE.get(key)
    if size is None:
        size = getattr(_lib.load(), fn)(*key)
        if size < 0:
            raise _lib.SolAttnError("unsupported shape for libsolattn")
        if len(_WORKSPACE) >= 4096:
            _WORKSPACE.clear()
        _WORKSPACE[key] = size
    if size == 0:
        return None, None, 0
    x = torch.empty(size, dtype=torch.uint8, device=device)
    return x, x.data_ptr(), size


def checked(x):
    """``x`` (or an aligned copy) after the checks that the inference-only BF16 operators share beyond
    shapes and devices, with its strides.  Rows have to start on 16-byte boundaries; a copy is also made
    where only the stride of a dimension of size 1 or the start is odd."""
    if x.dtype is not torch.bfloat16:
        raise ValueError("Only BF16 Q/K/V are implemented")
    if x.requires_grad:
        raise ValueError("Inference only: Q/K/V must not require gradients")
    strides = x.stride()
    if strides[-1] != 1 or min(strides) <= 0:
        raise ValueError("Q/K/V need positive strides and contiguous head dimension")
    if x.shape[-1] not in (64, 128):
        raise ValueError("Only head dimensions 64 and 128 are implemented")
    odd = x.data_ptr() & 15
    for s in strides[:-1]:
        odd |= s & 7
    if odd:
        x = x.clone(memory_format=torch.contiguous_format)
        strides = x.stride()
    return x, strides


def on_device(device, fn, *args):
    """``fn(*args)`` with ``device`` current."""
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return fn(*args)
    return fn(*args)


def window_attention(q, k, v, *, window=None, lookahead=0, sink_tokens=0, scale=None):
    """Attention of each query over a window of tokens and the first ``sink_tokens`` keys.

    ``q`` is BTHD [B, Tq, Hq, D], ``k`` and ``v`` [B, Tk, Hkv, D] with Hq a multiple of Hkv (query
    head h reads K/V head h // (Hq // Hkv)); BF16, D 64 or 128.  The queries are the last tokens:
    query i has position p = Tk - Tq + i, and sees key j iff j <= p + ``lookahead`` (None: every
    later key) and (j > p - ``window`` (None: every earlier key) or j < ``sink_tokens``).
    ``window`` counts the query's own position.  A query that sees no key gives zeros, and keys that a
    query does not see have no influence on it whatever they hold.  FP32 softmax and sums.
    """
    if q.ndim != 4 or k.ndim != 4 or v.ndim != 4:
        raise ValueError("Q/K/V must have BTHD rank-4 layout")
    B, Tq, Hq, D = q.shape
    Bk, Tk, Hkv, Dk = k.shape
    if k.shape != v.shape or B != Bk or D != Dk or 0 in (B, Tq, Hq, D, Tk, Hkv) or Hq % Hkv:
        raise ValueError("Q/K/V batch and dimension shapes must agree and be nonempty, and Q heads "
                         "be a multiple of K/V heads")
    (q, sq), (k, sk), (v, sv) = checked(q), checked(k), checked(v)
    scale = check_scale(scale, D)
    rule = check_rule(window, lookahead, sink_tokens)
    device = q.device
    if (device.type != "cuda" or k.device != device or v.device != device
            or not _is_b200(device)):
        raise ValueError("The sm_100a backend requires Q/K/V on the same NVIDIA B200 CUDA GPU")
    return on_device(device, _launch, q, k, v, rule, scale, (B, Tq, Tk, Hq, Hkv, D), sq[:3] + sk[:3] + sv[:3])


def _launch(q, k, v, rule, scale, shape, strides):
    device = q.device
    word = error_word(device.index)  # an earlier call's device-side error surfaces here
    keep, ws, size = workspace("solattn_window_workspace_bytes", shape + rule, device)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    rc = _lib.load().solattn_window_attention(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), *shape, *strides, *rule, scale, ws, size, out.data_ptr(),
        word, current_stream(device.index))
    if rc:
        _lib.check(rc, "solattn_window_attention")
    return out
