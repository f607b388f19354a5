"""Norms of query and key heads with the rotation to their positions, in one pass.

Each head of the queries and keys of a fused projection is divided by its root mean square
and multiplied by a learned gain, then turned by its token's position, and written where
attention reads it; values are moved. The gradient is one pass as well. For new tokens of
sequences in a paged cache ``cache_op.paged_append`` does the same with ``q_gain`` and
``k_gain``. No reference counterpart.
"""

from __future__ import annotations

import torch

from . import _lib
from .reference import DEFAULT_EPS

__all__ = ["qk_norm_rope"]


def _need(ok: bool, message: str) -> None:
    if not ok:
        raise ValueError(message)


def qk_norm_rope(qkv: torch.Tensor, q_gain: torch.Tensor, k_gain: torch.Tensor, cos: torch.Tensor,
                 sin: torch.Tensor, *, kv_heads: int | None = None,
                 eps: float = DEFAULT_EPS) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``qkv [B, T, heads + 2 kv_heads, hd]`` (queries, keys, values; as many of each without
    ``kv_heads``) to ``q [B, heads, T, hd]`` and ``k``, ``v`` ``[B, kv_heads, T, hd]``.

    With ``u = x / sqrt(mean(x^2) + eps) * gain`` over a head's channels, channel ``i`` of the
    first half turns with channel ``i`` of the second by ``cos``, ``sin`` (fp32 ``[positions,
    hd / 2]``, or ``[positions, 1, hd / 2]`` as the decoder's) of token ``t``. Gains are
    ``[hd]``, of qkv's dtype or fp32; ``hd`` is a multiple of 8, at most 256. Arithmetic is fp32,
    every output and gradient rounded once; the gains' gradients are summed in a fixed order.

    A backward that is captured into a graph while an eager graph of the same leaves lives is
    refused: it would take the leaves' stream into the capture.

    Calls that no kernel may stand in for (tracing, transforms, tensor subclasses) run as torch
    operations on the same numbers."""
    if (_lib.ordinary(qkv, q_gain, k_gain, cos, sin) and qkv.is_cuda
            and (kv_heads is None or (type(kv_heads) is int and kv_heads > 0))):
        r = _lib.native().qk_norm_rope(qkv, q_gain, k_gain, cos, sin, 0 if kv_heads is None else kv_heads, eps)
        if r is not None:
            return tuple(r)
    _need(qkv.ndim == 4, f"qkv must be [B, T, heads + 2 kv_heads, hd], got {tuple(qkv.shape)}")
    b, t, rows, hd = qkv.shape
    if kv_heads is None:
        _need(rows % 3 == 0, f"{rows} heads are not as many queries, keys and values; kv_heads says how many")
        kv_heads = rows // 3
    kv_heads = int(kv_heads)
    heads = rows - 2 * kv_heads
    _need(kv_heads >= 1 and heads >= 1 and rows <= 0xFFFF, f"{rows} heads hold no queries next to {kv_heads} kv heads")
    _need(hd % 8 == 0 and 8 <= hd <= 256, f"head_dim must be a multiple of 8, at most 256, got {hd}")
    _lib.dtype_code(qkv.dtype)
    _need(qkv.is_cuda, "qkv must be on a CUDA device")
    for name, g in (("q_gain", q_gain), ("k_gain", k_gain)):
        _need(g.shape == (hd,) and g.device == qkv.device and g.dtype == q_gain.dtype
              and g.dtype in (qkv.dtype, torch.float32),
              f"{name} must be a [{hd}] tensor on the same CUDA device, of qkv's dtype or fp32, as the other gain is")
    for name, x in (("cos", cos), ("sin", sin)):
        _need(x.dtype == torch.float32 and x.device == qkv.device and x.shape == cos.shape
              and x.ndim in (2, 3) and x.shape[-1] * 2 == hd and x.numel() == x.shape[0] * x.shape[-1]
              and x.shape[0] >= t,
              f"{name} must be fp32 [at least {t} positions, {hd // 2}] on the same CUDA device")
    return _by_operations(qkv, q_gain, k_gain, cos, sin, heads, kv_heads, float(eps))


def _by_operations(qkv, q_gain, k_gain, cos, sin, heads: int, kv_heads: int, eps: float):
    t, hd = qkv.shape[1], qkv.shape[3]
    q, k, v = qkv.transpose(1, 2).split([heads, kv_heads, kv_heads], dim=1)
    cos, sin = cos.reshape(-1, hd // 2)[:t], sin.reshape(-1, hd // 2)[:t]

    def turned(x, gain):
        x = x.float()
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * gain.float()
        lo, hi = x.chunk(2, dim=-1)
        return torch.cat((lo * cos - hi * sin, lo * sin + hi * cos), dim=-1).to(qkv.dtype).contiguous()

    return turned(q, q_gain), turned(k, k_gain), v.contiguous()
