"""A paged cache of keys and values: appending to it, and attention over it.

What generating with the decoder needs between its projections. The cache of a layer is a
pair of tensors ``k_cache``, ``v_cache`` ``[n_pages, kv_heads, page, head_dim]`` (any
strides with dense rows, the same for both); a sequence's tokens lie in the pages that
its row of ``page_table`` ``[B, columns]`` lists, ``page`` of them each, in order, at most
2^30 in all.

A call brings the new tokens of ``B`` sequences packed into one tensor: sequence ``b``
has the rows ``starts[b]`` to ``starts[b + 1]``; without ``starts`` every sequence has
the same number of rows (one, for a decoded token). ``lengths[b]`` counts the tokens of a
sequence in the cache, the new ones included, which are its last. ``page_table``,
``lengths`` and ``starts`` are int32 tensors on the device and are read by the kernels:
nothing waits for the device, and a captured call can be replayed for other lengths.

Sequences that continue one prompt share its pages: ``prefix_len`` tokens in the pages
that ``prefix_pages`` lists come before every sequence's own tokens. Where every sequence
brings few rows, attention reads the prefix once for all of them.

Not checked, as it would mean to wait for the device: ``starts`` out of order (results
are then undefined), and two new tokens whose places are the same one (which of them is
kept is). Pages outside the cache hold nothing: a token that would go there is not
cached and its queries are NaN, and attention leaves its position out. The same goes for
positions past the rotary tables or the table's row. Rows that belong to no sequence are
zero, or keep their content in a given ``out``, which may be the queries themselves.

There is no derivative: under autograd, and on tensors with tangents, the functions raise.
"""

from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from . import _lib
from .hip_op import _ptr
from .reference import DEFAULT_EPS

__all__ = ["paged_append", "paged_attention"]

#: Tokens at most in a row of the page table, and in a prefix.
_MOST_TOKENS = 1 << 30


def _need(ok: bool, message: str) -> None:
    if not ok:
        raise ValueError(message)


def _validate_cache(rows, heads: int, what: str, k, v, page_table, lengths, starts, prefix_len: int) -> _lib.Paged:
    """The checks shared by both functions; the C struct of a valid call."""
    _need(k.ndim == 4 and k.shape == v.shape and k.stride() == v.stride(),
          "k_cache and v_cache must be [n_pages, kv_heads, page, head_dim] of the same shape and strides")
    _need(page_table.ndim == 2 and page_table.shape[0] >= 1 and page_table.shape[1] >= 1,
          f"page_table must be [B, columns], got {tuple(page_table.shape)}")
    n_seq, n_tok = page_table.shape[0], rows.shape[0]
    _need(lengths.shape == (n_seq,), f"lengths must be [{n_seq}], got {tuple(lengths.shape)}")
    _need(starts is None or starts.shape == (n_seq + 1,), f"starts must be [{n_seq + 1}]")
    _need(starts is not None or n_tok % n_seq == 0,
          f"{n_tok} rows do not divide among {n_seq} sequences; starts says where each begins")
    for name, t in (("page_table", page_table), ("lengths", lengths), ("starts", starts)):
        if t is not None:
            _need(t.dtype == torch.int32 and (t.shape[-1] == 1 or t.stride(-1) == 1),
                  f"{name} must be int32 with dense rows")
    for name, t in (("k_cache", k), ("v_cache", v), ("page_table", page_table), ("lengths", lengths), ("starts", starts)):
        _need(t is None or t.device == rows.device, f"{name} must be on the same CUDA device as {what}")
    code = _lib.dtype_code(k.dtype)
    _need(v.dtype == k.dtype and rows.dtype == k.dtype, f"{what} and the caches must have the same dtype")
    n_pages, kv_heads, page, hd = k.shape
    chunk = 16 // k.element_size()
    _need(n_pages >= 1 and page >= 1 and page & (page - 1) == 0, f"a page must hold a power of two tokens, got {page}")
    _need(hd % 8 == 0 and 8 <= hd <= 256, f"head_dim must be a multiple of 8, at most 256, got {hd}")
    _need(kv_heads >= 1 and heads >= 1 and heads % kv_heads == 0 and heads <= 0xFFFF,
          f"{heads} query heads are no multiple of {kv_heads} kv heads")
    _need(k.stride(3) == 1 and all(s >= 0 and s % chunk == 0 for s in k.stride()[:3])
          and k.data_ptr() % 16 == 0 and v.data_ptr() % 16 == 0,
          "the caches' rows must be dense and start at 16-byte boundaries")
    span = 2**32 // k.element_size()
    _need(k.stride(0) < span and k.stride(2) * page < span, "a page must span less than 4 GiB, and so pages apart")
    _need(0 <= prefix_len <= _MOST_TOKENS, "prefix_len must not be negative, and at most 2^30")
    _need(page_table.shape[1] * page <= _MOST_TOKENS, "a row of page_table must hold at most 2^30 tokens")
    _need(rows.is_cuda, f"{what} must be on a CUDA device")
    return _lib.Paged(k.data_ptr(), v.data_ptr(), page_table.data_ptr(), lengths.data_ptr(),
                      None if starts is None else starts.data_ptr(), k.stride(0), k.stride(1), k.stride(2),
                      page_table.stride(0), n_seq, n_tok, n_pages, page_table.shape[1], page, heads, kv_heads, hd, code)


def _validate_out(out, like, shape) -> None:
    _need(out.shape == shape and out.dtype == like.dtype and out.device == like.device and out.is_contiguous()
          and out.data_ptr() % 16 == 0, f"out must be a dense {list(shape)} tensor of the inputs' dtype and device")


def _no_backward(name: str, *tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{name} has no backward; run it under torch.no_grad() for inference")
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{name} has no derivative; run it on tensors without tangents")


def _changed(*tensors) -> None:
    """Tell autograd that the kernels wrote into these."""
    for t in tensors:
        if t is not None and not t.is_inference():
            increment_version(t)


def paged_append(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, k_cache: torch.Tensor,
                 v_cache: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
                 starts: torch.Tensor | None = None, *, prefix_len: int = 0,
                 out: torch.Tensor | None = None, q_gain: torch.Tensor | None = None,
                 k_gain: torch.Tensor | None = None, eps: float = DEFAULT_EPS) -> torch.Tensor:
    """Rotate a fused projection's queries and keys to their positions, write the keys and
    values into the cache and return the queries ``[n_tok, heads, head_dim]``.

    ``qkv [n_tok, heads + 2 kv_heads, head_dim]`` holds queries, keys and values;
    ``cos``, ``sin`` are fp32 ``[positions, head_dim / 2]`` (``[positions, 1, ...]`` as
    the decoder's). Row ``i`` of ``n`` new ones stands at ``lengths[b] - n + i``, behind
    ``prefix_len``. Arithmetic is fp32, every output rounded once.

    With ``q_gain`` and ``k_gain`` (``[head_dim]``, of qkv's dtype or fp32) every query and key
    head is normalised before it turns, as ``rope_op.qk_norm_rope`` does:
    ``x / sqrt(mean(x^2) + eps) * gain``."""
    if (_lib.ordinary(qkv, cos, sin, k_cache, v_cache, page_table, lengths) and qkv.is_cuda
            and type(prefix_len) is int and (starts is None or _lib.ordinary(starts))
            and (out is None or _lib.ordinary(out)) and (q_gain is None or _lib.ordinary(q_gain, k_gain))):
        q = _lib.native().paged_append(qkv, cos, sin, k_cache, v_cache, page_table, lengths, starts, prefix_len, out,
                                       q_gain, k_gain, eps)
        if q is not None:
            return q
    if torch.compiler.is_compiling():
        return _append_untraced(qkv, cos, sin, k_cache, v_cache, page_table, lengths, starts, prefix_len=prefix_len,
                                out=out, q_gain=q_gain, k_gain=k_gain, eps=eps)
    _no_backward("paged_append", qkv, cos, sin, k_cache, v_cache, out, q_gain, k_gain)
    _need(qkv.ndim == 3, f"qkv must be [n_tok, heads + 2 kv_heads, head_dim], got {tuple(qkv.shape)}")
    _need(k_cache.ndim == 4, "k_cache must be [n_pages, kv_heads, page, head_dim]")
    heads = qkv.shape[1] - 2 * k_cache.shape[1]
    prefix_len = int(prefix_len)
    c = _validate_cache(qkv, heads, "qkv", k_cache, v_cache, page_table, lengths, starts, prefix_len)
    _need(qkv.shape[2] == c.hd, f"qkv must have heads of {c.hd}, got {qkv.shape[2]}")
    for name, t in (("cos", cos), ("sin", sin)):
        _need(t.dtype == torch.float32 and t.device == qkv.device and t.is_contiguous() and t.ndim >= 2
              and t.shape[-1] * 2 == c.hd and t.numel() == t.shape[0] * t.shape[-1] and t.shape == cos.shape,
              f"{name} must be a dense fp32 [positions, {c.hd // 2}] tensor on the same CUDA device")
    shape = (c.n_tok, heads, c.hd)
    if out is not None:
        _validate_out(out, qkv, shape)
    _need((q_gain is None) == (k_gain is None), "q_gain and k_gain go together")
    for name, g in (("q_gain", q_gain), ("k_gain", k_gain)):
        _need(g is None or (g.shape == (c.hd,) and g.device == qkv.device and g.dtype == q_gain.dtype
                            and g.dtype in (qkv.dtype, torch.float32)),
              f"{name} must be a [{c.hd}] tensor on the same CUDA device, of qkv's dtype or fp32, as the other gain is")
    if qkv.stride(2) != 1:
        qkv = qkv.contiguous()
    if q_gain is not None:
        q_gain, k_gain = q_gain.contiguous(), k_gain.contiguous()
        if qkv.stride(0) % 4 or qkv.stride(1) % 4 or qkv.data_ptr() % (4 * qkv.element_size()):
            qkv = qkv.clone(memory_format=torch.contiguous_format)
    q = torch.empty(shape, device=qkv.device, dtype=qkv.dtype) if out is None else out
    with torch.cuda.device(qkv.device):
        args = (_ptr(cos), _ptr(sin), cos.shape[0], prefix_len, _ptr(q), int(out is None), _lib.stream_ptr(qkv.device))
        rows = (ctypes.byref(c), _ptr(qkv), qkv.stride(0), qkv.stride(1))
        if q_gain is None:
            rc = _lib.lib().sy_paged_append(*rows, *args)
        else:
            rc = _lib.lib().sy_paged_append_norm(*rows, _ptr(q_gain), _ptr(k_gain), _lib.dtype_code(q_gain.dtype),
                                                 float(eps), *args)
    _lib.check(rc, "sy_paged_append" if q_gain is None else "sy_paged_append_norm")
    _changed(k_cache, v_cache, out)
    return q


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                    lengths: torch.Tensor, starts: torch.Tensor | None = None, *,
                    prefix_pages: torch.Tensor | None = None, prefix_len: int = 0, scale: float | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of the new tokens' queries ``q [n_tok, heads, head_dim]`` over the cache:
    each row sees its own position and every earlier one, and the whole prefix. Query head
    ``h`` reads kv head ``h * kv_heads // heads``; ``scale`` is ``head_dim**-0.5`` by
    default. A row that sees nothing is zero; an infinite value that a row sees makes its
    channel infinite or NaN, one that it does not see changes nothing.

    Scores, softmax statistics and sums are fp32. Where a sequence brings more than 16 rows a
    kv head to a 16-bit cache, the weights are rounded to its dtype for the second product
    (relative error 2.0e-3 in bf16, of which the output's own rounding is 1.7e-3); so they are
    for all sequences behind a prefix that bring more than 16 on average. Where there are fewer
    the product takes a weight as two numbers, the rounded one and what it lacks. fp16 weights
    below 2^-21 of the largest (as two numbers 2^-18) are off by up to 2^-32 (2^-40) of it."""
    if (_lib.ordinary(q, k_cache, v_cache, page_table, lengths) and q.is_cuda and type(prefix_len) is int
            and (starts is None or _lib.ordinary(starts)) and (out is None or _lib.ordinary(out))
            and (prefix_pages is None or _lib.ordinary(prefix_pages))):
        o = _lib.native().paged_attention(q, k_cache, v_cache, page_table, lengths, starts, prefix_pages, prefix_len,
                                          q.shape[-1] ** -0.5 if scale is None else scale, out)
        if o is not None:
            return o
    if torch.compiler.is_compiling():
        return _attention_untraced(q, k_cache, v_cache, page_table, lengths, starts, prefix_pages=prefix_pages,
                                   prefix_len=prefix_len, scale=scale, out=out)
    _no_backward("paged_attention", q, k_cache, v_cache, out)
    _need(q.ndim == 3, f"q must be [n_tok, heads, head_dim], got {tuple(q.shape)}")
    prefix_len = int(prefix_len)
    heads = q.shape[1]
    c = _validate_cache(q, heads, "q", k_cache, v_cache, page_table, lengths, starts, prefix_len)
    _need(q.shape[2] == c.hd, f"q must have heads of {c.hd}, got {q.shape[2]}")
    if prefix_len > 0:
        _need(prefix_pages is not None and prefix_pages.ndim == 1 and prefix_pages.dtype == torch.int32
              and prefix_pages.is_contiguous() and prefix_pages.device == q.device,
              "prefix_pages must be a dense int32 [pages] tensor on the same CUDA device")
        _need(prefix_pages.shape[0] * c.page >= prefix_len,
              f"{prefix_pages.shape[0]} prefix pages of {c.page} do not hold {prefix_len} tokens")
    if out is not None:
        _validate_out(out, q, (c.n_tok, heads, c.hd))
    chunk = 16 // q.element_size()
    if q.stride(2) != 1 or q.stride(0) % chunk or q.stride(1) % chunk or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
    o = torch.empty_like(q, memory_format=torch.contiguous_format) if out is None else out
    with torch.cuda.device(q.device):
        lib = _lib.lib()
        need = lib.sy_paged_attention_workspace_bytes(ctypes.byref(c), prefix_len)
        if need < 0:
            _lib.check(int(need), "sy_paged_attention_workspace_bytes")
        ws = torch.empty(max(1, need // 4), device=q.device, dtype=torch.float32)
        rc = lib.sy_paged_attention(ctypes.byref(c), _ptr(q), q.stride(0), q.stride(1), _ptr(o),
                                    _ptr(prefix_pages) if prefix_len > 0 else None, prefix_len,
                                    q.shape[-1] ** -0.5 if scale is None else float(scale), int(out is None),
                                    _ptr(ws), ws.numel() * 4, _lib.stream_ptr(q.device))
    _lib.check(rc, "sy_paged_attention")
    _changed(out)
    return o


# What a compiler's trace calls: the functions themselves, untraced.
_append_untraced = torch.compiler.disable(paged_append)
_attention_untraced = torch.compiler.disable(paged_attention)
