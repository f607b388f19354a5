"""Sampling one token per row of logits from given uniform numbers.

The weight of token ``i`` is ``exp((x_i - max x) / temperature)`` in units of ``2^-44``
(zero below ``2^-45``). The candidates, ordered by falling logits and rising index, are
cut three times, each cut over what the one before left:

  top_k  the first ``top_k`` (all of them if less than 1)
  top_p  those before whose own place less than ``top_p`` of the weight lies, at least
         one (all if 1 or more)
  min_p  those with at least ``min_p`` of the largest's weight

The token is the first candidate, in the order of indices, at which the running sum of
weights passes ``u`` times their total. Sums are whole numbers: the same inputs give the
same token on every run. A temperature of zero picks the first largest logit. NaN counts
as ``-inf``, a token of which is never drawn; a row of nothing else gives -1.
"""

from __future__ import annotations

import ctypes
import math
import numbers

import torch

from . import _lib
from .hip_op import _ptr

__all__ = ["sample_tokens", "MAX_VOCAB"]

#: Widest row of logits a call takes.
MAX_VOCAB = 1 << 18


def _split(name: str, x, integer: bool = False):
    """A setting as (number, tensor or None); numbers are checked here."""
    if isinstance(x, torch.Tensor):
        return (0 if integer else 0.0), x
    if not isinstance(x, numbers.Real) or (integer and not isinstance(x, numbers.Integral)):
        raise ValueError(f"{name} must be {'an integer' if integer else 'a number'} or a tensor of one a row")
    if integer:
        return max(0, min(int(x), 0x7FFFFFFF)), None
    if math.isnan(x) or (name != "top_p" and x < 0):
        raise ValueError(f"{name} must not be negative or NaN, got {x}")
    return float(x), None


def sample_tokens(logits: torch.Tensor, u: torch.Tensor, *, temperature=1.0, top_k=0, top_p=1.0,
                  min_p=0.0) -> torch.Tensor:
    """One token (int64) for each row of ``logits [B, V]`` from the uniform numbers ``u [B]``
    (fp32, in ``[0, 1)``). Every setting is a number, or a tensor ``[B]`` of one a row
    (fp32; ``top_k`` int32) that is read on the device."""
    t, ts = _split("temperature", temperature)
    k, ks = _split("top_k", top_k, integer=True)
    p, ps = _split("top_p", top_p)
    m, ms = _split("min_p", min_p)
    if _lib.ordinary(logits, u) and logits.is_cuda and all(x is None or _lib.ordinary(x) for x in (ts, ks, ps, ms)):
        tokens = _lib.native().sample_tokens(logits, u, t, k, p, m, ts, ks, ps, ms)
        if tokens is not None:
            return tokens
    if torch.compiler.is_compiling():
        return _untraced(logits, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    if logits.ndim != 2:
        raise ValueError(f"logits must be [B, V], got {tuple(logits.shape)}")
    b, v = logits.shape
    if not 1 <= v <= MAX_VOCAB:
        raise ValueError(f"logits must have 1 to {MAX_VOCAB} columns, got {v}")
    if not logits.is_cuda:
        raise ValueError("logits must be on a CUDA device")
    code = _lib.dtype_code(logits.dtype)
    for name, x, dtype in (("u", u, torch.float32), ("temperature", ts, torch.float32), ("top_k", ks, torch.int32),
                           ("top_p", ps, torch.float32), ("min_p", ms, torch.float32)):
        if x is not None and (x.shape != (b,) or x.dtype != dtype or x.device != logits.device):
            raise ValueError(f"{name} must be a [{b}] tensor of {dtype} on the same CUDA device as logits")
    tokens = torch.empty(b, device=logits.device, dtype=torch.int64)
    if b == 0:
        return tokens
    if v > 1 and logits.stride(1) != 1:
        logits = logits.contiguous()
    u, ts, ks, ps, ms = (None if x is None else x.contiguous() for x in (u, ts, ks, ps, ms))
    how = _lib.Sampling(t, p, m, k, *(None if x is None else x.data_ptr() for x in (ts, ps, ms, ks)))
    with torch.cuda.device(logits.device):
        rc = _lib.lib().sy_sample(_ptr(logits), _ptr(u), _ptr(tokens), ctypes.byref(how), b, v, logits.stride(0), code,
                                  _lib.stream_ptr(logits.device))
    _lib.check(rc, "sy_sample")
    return tokens


_untraced = torch.compiler.disable(sample_tokens)  # what a compiler's trace calls
