"""What steers sampling: penalties for tokens that were there before, biases, and a mask of
the tokens that are allowed, in one pass over the logits.

For token ``v`` of a row, with ``x`` its logit and ``n`` its occurrences behind the prompt:

  y = x / repetition (x > 0), x * repetition (else)   if it is in the row's history at all
  y = y - frequency * n - presence * (n > 0)
  y = y + bias[v], and -inf where ``allowed`` says no

The result goes to ``sample_op.sample_tokens``. Histories, settings and masks are read on the
device: nothing waits for it, and a captured call can be replayed for others. A row that
allows nothing is ``-inf`` throughout (sampling gives -1 for it). No reference counterpart.
"""

from __future__ import annotations

import ctypes
import math
import numbers

import torch

from . import _lib
from .cache_op import _changed, _no_backward
from .hip_op import _ptr

__all__ = ["adjust_logits", "pack_allowed"]


def _need(ok: bool, message: str) -> None:
    if not ok:
        raise ValueError(message)


def _split(name: str, x):
    """A setting as (number, tensor or None); numbers are checked here."""
    if type(x) is float and (x > 0 or name != "repetition_penalty") and abs(x) < math.inf:
        return x, None
    if isinstance(x, torch.Tensor):
        return 1.0, x
    if not isinstance(x, numbers.Real) or not math.isfinite(x):
        raise ValueError(f"{name} must be a finite number or a tensor of one a row")
    if name == "repetition_penalty" and x <= 0:
        raise ValueError(f"{name} must be positive, got {x}")
    return float(x), None


def pack_allowed(allowed: torch.Tensor) -> torch.Tensor:
    """A mask ``[..., V]`` of truth values as int32 words ``[..., ceil(V / 32)]``: bit ``i`` of
    word ``j`` stands for token ``32 j + i``."""
    v = allowed.shape[-1]
    bits = torch.nn.functional.pad(allowed.bool(), (0, -v % 32)).unflatten(-1, (-1, 32))
    words = (bits.long() << torch.arange(32, device=allowed.device)).sum(-1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)


def adjust_logits(logits: torch.Tensor, tokens: torch.Tensor | None = None, *, lengths: torch.Tensor | None = None,
                  prompt_lengths: torch.Tensor | None = None, repetition_penalty=1.0, presence_penalty=0.0,
                  frequency_penalty=0.0, bias: torch.Tensor | None = None, allowed: torch.Tensor | None = None,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """``logits [B, V]`` adjusted, as a new tensor or in ``out``, which may be ``logits``
    (and overlaps with them in no other way).

    ``tokens [B, L]`` (int64 or int32) is each row's history, of which the first ``lengths``
    count (int32 ``[B]``; all without it) and the first ``prompt_lengths`` (int32 ``[B]``; none
    without it) are the prompt, which only ``repetition_penalty`` looks at. Tokens outside the
    vocabulary are passed over. A penalty is a number, or an fp32 tensor ``[B]`` of one a row.
    ``bias`` is ``[V]`` or ``[B, V]`` of the logits' dtype or fp32; ``allowed`` likewise, as
    truth values or as the int32 words of ``pack_allowed``. Penalties are computed in fp64, the
    bias is added in fp32, and the result is rounded once to the logits' dtype."""
    r, rs = _split("repetition_penalty", repetition_penalty)
    p, ps = _split("presence_penalty", presence_penalty)
    f, fs = _split("frequency_penalty", frequency_penalty)
    more = (tokens, lengths, prompt_lengths, rs, ps, fs, bias, allowed, out)
    if _lib.ordinary(logits, *[x for x in more if x is not None]) and logits.is_cuda:
        y = _lib.native().adjust_logits(logits, r, p, f, *more)
        if y is not None:
            return y
    if torch.compiler.is_compiling():
        return _untraced(logits, tokens, lengths=lengths, prompt_lengths=prompt_lengths,
                         repetition_penalty=repetition_penalty, presence_penalty=presence_penalty,
                         frequency_penalty=frequency_penalty, bias=bias, allowed=allowed, out=out)
    _no_backward("adjust_logits", logits, rs, ps, fs, bias, out)
    _need(logits.ndim == 2, f"logits must be [B, V], got {tuple(logits.shape)}")
    b, v = logits.shape
    _need(1 <= v <= 1 << 30, f"logits must have 1 to 2^30 columns, got {v}")
    _need(logits.is_cuda, "logits must be on a CUDA device")
    code = _lib.dtype_code(logits.dtype)
    dev = logits.device
    how = _lib.Adjusting(r, p, f, tokens_bytes=8, bias_dtype=_lib.SY_F32)
    keep = []  # (tensors that the call reads live until it is issued)
    if tokens is None:
        _need(lengths is None and prompt_lengths is None, "lengths and prompt_lengths go with tokens")
    else:
        _need(tokens.ndim == 2 and tokens.shape[0] == b and tokens.dtype in (torch.int64, torch.int32)
              and tokens.device == dev, f"tokens must be int64 or int32 [{b}, L] on the same CUDA device as logits")
        _need(tokens.shape[1] <= 1 << 30, "a history must hold at most 2^30 tokens")
        if tokens.shape[1] > 1 and tokens.stride(1) != 1:
            tokens = tokens.contiguous()
        keep.append(tokens)
        how.tokens, how.tokens_stride, how.n_tokens = tokens.data_ptr(), tokens.stride(0), tokens.shape[1]
        how.tokens_bytes = tokens.element_size()
    for name, field, x, dtype in (("lengths", "lengths", lengths, torch.int32),
                                  ("prompt_lengths", "prompt_lengths", prompt_lengths, torch.int32),
                                  ("repetition_penalty", "repetitions", rs, torch.float32),
                                  ("presence_penalty", "presences", ps, torch.float32),
                                  ("frequency_penalty", "frequencies", fs, torch.float32)):
        if x is not None:
            _need(x.shape == (b,) and x.dtype == dtype and x.device == dev,
                  f"{name} must be a [{b}] tensor of {dtype} on the same CUDA device as logits")
            keep.append(x.contiguous())
            setattr(how, field, keep[-1].data_ptr())
    if bias is not None:
        _need(bias.shape in ((v,), (b, v)) and bias.dtype in (logits.dtype, torch.float32) and bias.device == dev,
              f"bias must be [{v}] or [{b}, {v}] of the logits' dtype or fp32 on the same CUDA device")
        bias = bias if bias.stride(-1) == 1 or v == 1 else bias.contiguous()
        keep.append(bias)
        how.bias, how.bias_dtype = bias.data_ptr(), _lib.dtype_code(bias.dtype)
        how.bias_stride = bias.stride(0) if bias.ndim == 2 else 0
    if allowed is not None:
        n = -(-v // 32) if allowed.dtype == torch.int32 else v
        _need(allowed.shape in ((n,), (b, n)) and allowed.dtype in (torch.int32, torch.bool) and allowed.device == dev,
              f"allowed must be truth values [{v}] or [{b}, {v}], or int32 words of {-(-v // 32)}, on the same CUDA device")
        allowed = allowed if allowed.stride(-1) == 1 or n == 1 else allowed.contiguous()
        keep.append(allowed)
        how.mask, how.mask_kind = allowed.data_ptr(), 1 if allowed.dtype == torch.int32 else 2
        how.mask_stride = allowed.stride(0) if allowed.ndim == 2 else 0
    x = logits if v == 1 or logits.stride(1) == 1 else logits.contiguous()
    if out is not None:
        _need(out.shape == logits.shape and out.dtype == logits.dtype and out.device == dev
              and (v == 1 or out.stride(1) == 1) and (b <= 1 or out.stride(0) >= v),
              f"out must be a [{b}, {v}] tensor of the logits' dtype and device with dense rows")
    y = torch.empty_like(x, memory_format=torch.contiguous_format) if out is None else out
    if b > 0:
        with torch.cuda.device(dev):
            rc = _lib.lib().sy_adjust(_ptr(x), _ptr(y), ctypes.byref(how), b, v, x.stride(0), y.stride(0), code,
                                      _lib.stream_ptr(dev))
        _lib.check(rc, "sy_adjust")
    _changed(out)
    return y


_untraced = torch.compiler.disable(adjust_logits)  # what a compiler's trace calls
