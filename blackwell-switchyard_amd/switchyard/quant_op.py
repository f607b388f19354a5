"""Projections with 4-bit weights: what a decoded token reads is a quarter of the bytes.

A weight is ``scale * (code - zero)``: codes of 0 to 15, a scale (and a whole zero point, or 8)
for each group of 32, 64 or 128 neighbouring columns of a row. ``quantize4`` rounds weights to
that, ``Weight4`` holds them laid out for the kernels, ``linear4`` multiplies with them and
``Linear4`` is the module. Products of activations and codes are exact and summed in fp32,
group sums are scaled in fp32, and the output is rounded once. There is no derivative: under
autograd, and on tensors with tangents, ``linear4`` raises. No reference counterpart.
"""

from __future__ import annotations

import ctypes

import torch
import torch.nn as nn

from . import _lib
from .cache_op import _no_backward
from .hip_op import _ptr

__all__ = ["Weight4", "Linear4", "quantize4", "linear4", "GROUPS"]

#: Columns that may share a scale.
GROUPS = (32, 64, 128)

_TILE_K = 128  # columns of a tile of the layout, which has 16 features


def _need(ok: bool, message: str) -> None:
    if not ok:
        raise ValueError(message)


def _check_sizes(out_features: int, in_features: int, group: int) -> None:
    _need(group in GROUPS, f"a group must have one of {GROUPS} columns, got {group}")
    _need(1 <= out_features <= 1 << 24 and 1 <= in_features <= 1 << 24,
          f"weights must have 1 to 2^24 rows and columns, got {out_features} by {in_features}")


class Weight4:
    """4-bit weights ``[out_features, in_features]`` in tiles of 16 rows by 128 columns
    (``tiles`` int32 ``[row tiles, column tiles, 64, 4]``; ``scales`` and ``zeros``, which may be
    None, ``[row tiles, column tiles, 16, groups of a tile]``). Made by ``quantize4`` or ``from_codes``."""

    __slots__ = ("tiles", "scales", "zeros", "out_features", "in_features", "group")

    def __init__(self, tiles: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None, out_features: int,
                 in_features: int, group: int) -> None:
        _check_sizes(out_features, in_features, group)
        rows, cols = -(-out_features // 16), -(-in_features // _TILE_K)
        _need(tiles.shape == (rows, cols, 64, 4) and tiles.dtype == torch.int32 and tiles.is_contiguous()
              and tiles.data_ptr() % 16 == 0, f"tiles must be a dense int32 [{rows}, {cols}, 64, 4] tensor")
        shape = (rows, cols, 16, _TILE_K // group)
        _lib.dtype_code(scales.dtype)
        _need(scales.shape == shape and scales.is_contiguous() and scales.device == tiles.device
              and scales.data_ptr() % 16 == 0, f"scales must be a dense {list(shape)} tensor on the tiles' device")
        _need(zeros is None or (zeros.shape == shape and zeros.dtype == torch.uint8 and zeros.is_contiguous()
                                and zeros.device == tiles.device and zeros.data_ptr() % 4 == 0),
              f"zeros must be a dense uint8 {list(shape)} tensor on the tiles' device")
        self.tiles, self.scales, self.zeros = tiles, scales, zeros
        self.out_features, self.in_features, self.group = out_features, in_features, group

    @classmethod
    def from_codes(cls, codes: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None, *,
                   in_features: int, group: int) -> Weight4:
        """Weights that are 4-bit already: ``codes`` uint8 ``[N, ceil(K / 2)]``, two columns a byte
        with the even one in the low half, ``scales [N, ceil(K / group)]`` of the activations'
        dtype, ``zeros`` uint8 of the same shape or None for 8 throughout."""
        _need(codes.ndim == 2 and codes.dtype == torch.uint8, "codes must be a uint8 [N, ceil(K / 2)] tensor")
        n, k = codes.shape[0], int(in_features)
        _check_sizes(n, k, group)
        _need(codes.shape[1] == -(-k // 2), f"codes must have {-(-k // 2)} bytes a row, got {codes.shape[1]}")
        shape = (n, -(-k // group))
        code = _lib.dtype_code(scales.dtype)
        _need(scales.shape == shape and scales.device == codes.device,
              f"scales must be {list(shape)} on the codes' device, got {tuple(scales.shape)}")
        _need(zeros is None or (zeros.shape == shape and zeros.dtype == torch.uint8 and zeros.device == codes.device),
              f"zeros must be uint8 {list(shape)} on the codes' device")
        _need(codes.is_cuda, "codes must be on a CUDA device")
        dev, rows, cols = codes.device, -(-n // 16), -(-k // _TILE_K)
        tiles = torch.empty(rows, cols, 64, 4, device=dev, dtype=torch.int32)
        tile_scales = torch.empty(rows, cols, 16, _TILE_K // group, device=dev, dtype=scales.dtype)
        tile_zeros = None if zeros is None else torch.empty(tile_scales.shape, device=dev, dtype=torch.uint8)
        codes, scales = codes.detach().contiguous(), scales.detach().contiguous()
        zeros = None if zeros is None else zeros.contiguous()
        with torch.cuda.device(dev):
            rc = _lib.lib().sy_pack4(_ptr(codes), _ptr(scales), None if zeros is None else _ptr(zeros), _ptr(tiles),
                                     _ptr(tile_scales), None if zeros is None else _ptr(tile_zeros), n, k, group, code,
                                     _lib.stream_ptr(dev))
        _lib.check(rc, "sy_pack4")
        return cls(tiles, tile_scales, tile_zeros, n, k, group)

    def codes(self) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
        """Codes (uint8 ``[N, K]``, one a byte), scales and zeros by rows and groups again."""
        n, k, g = self.out_features, self.in_features, -(-self.in_features // self.group)
        w = (self.tiles >> 3) & 0x1FFFFFFF | (self.tiles << 29)  # (the tiles' words are turned by three bits)
        order = torch.tensor([c // 2 + 4 * (c % 2) for c in range(8)], device=w.device, dtype=torch.int32)
        c = (w[..., None] >> (4 * order)) & 15  # [row tile, column tile, 16 (column) + row, word, column]
        c = c.unflatten(2, (4, 16)).permute(0, 3, 1, 4, 2, 5).reshape(-1, self.tiles.shape[1] * _TILE_K)
        by_rows = lambda x: x.transpose(1, 2).flatten(2, 3).flatten(0, 1)[:n, :g].contiguous()  # noqa: E731
        return (c[:n, :k].to(torch.uint8).contiguous(), by_rows(self.scales),
                None if self.zeros is None else by_rows(self.zeros))

    def dequantize(self) -> torch.Tensor:
        """The weights ``[N, K]`` in fp32."""
        c, s, z = self.codes()
        of = torch.arange(self.in_features, device=c.device) // self.group
        return (c.float() - (8.0 if z is None else z.float()[:, of])) * s.float()[:, of]

    def __repr__(self) -> str:
        kind = "symmetric" if self.zeros is None else "with zero points"
        return f"Weight4({self.out_features} x {self.in_features}, groups of {self.group}, {self.scales.dtype}, {kind})"


def quantize4(w: torch.Tensor, group: int = 64, *, symmetric: bool = True) -> Weight4:
    """Round weights ``w [N, K]`` to 4 bits: each group to the nearest of ``s (c - 8)`` with ``s =
    max|w| / 7``, or without ``symmetric`` to ``s (c - z)`` over its range with zero, ``s = (max -
    min) / 15``. Scales have w's dtype, to which they are rounded before the codes are chosen (up
    where the codes would not reach the group's ends else, among the type's last steps). A group
    with an infinity or NaN has the scale NaN, and all its weights are NaN."""
    _need(w.ndim == 2, f"w must be [N, K], got {tuple(w.shape)}")
    n, k = w.shape
    _check_sizes(n, k, group)
    code = _lib.dtype_code(w.dtype)
    _need(w.is_cuda, "w must be on a CUDA device")
    w = w.detach()
    if k > 1 and w.stride(1) != 1:
        w = w.contiguous()
    shape = (n, -(-k // group))
    codes = torch.empty(n, -(-k // 2), device=w.device, dtype=torch.uint8)
    scales = torch.empty(shape, device=w.device, dtype=w.dtype)
    zeros = None if symmetric else torch.empty(shape, device=w.device, dtype=torch.uint8)
    with torch.cuda.device(w.device):
        rc = _lib.lib().sy_quantize4(_ptr(w), w.stride(0), _ptr(codes), _ptr(scales),
                                     None if zeros is None else _ptr(zeros), n, k, group, code, _lib.stream_ptr(w.device))
    _lib.check(rc, "sy_quantize4")
    return Weight4.from_codes(codes, scales, zeros, in_features=k, group=group)


def linear4(x: torch.Tensor, weight: Weight4) -> torch.Tensor:
    """``x [..., in_features]`` times the weights, ``[..., out_features]``; x has the scales'
    dtype. A row with an infinity or NaN gives NaN, and so may sums that pass fp32's range on the way
    (activations past 2^112).

    16-bit rows meet ``1 + c / 16``, less ``(1 + z / 16)`` of their sum over the group: two sums of
    the size of ``16 s |x| (2 + (c + z) / 16)``, where ``s (c - z) x`` added up directly are of ``s
    |x| |c - z|``. fp32's error in them, about ten times that of the direct sum, shows past the
    output's rounding only where a result all but cancels. fp32 rows meet ``c - z``."""
    return _linear4(x, weight.tiles, weight.scales, weight.zeros, weight.out_features, weight.in_features, weight.group)


def _linear4(x, tiles, scales, zeros, n: int, k: int, group: int) -> torch.Tensor:
    if _lib.ordinary(x, tiles, scales) and x.is_cuda and (zeros is None or _lib.ordinary(zeros)):
        y = _lib.native().linear4(x, tiles, scales, zeros, n, k, group)
        if y is not None:
            return y
    if torch.compiler.is_compiling():
        return _untraced(x, tiles, scales, zeros, n, k, group)
    _no_backward("linear4", x, scales)
    Weight4(tiles, scales, zeros, n, k, group)  # (checks them)
    _need(x.ndim >= 1 and x.shape[-1] == k, f"x must have {k} columns, got {tuple(x.shape)}")
    _need(x.dtype == scales.dtype, f"x must have the weights' dtype {scales.dtype}, got {x.dtype}")
    _need(x.is_cuda and x.device == tiles.device, f"x must be on the weights' CUDA device, which is {tiles.device}")
    rows = x.reshape(-1, k) if x.numel() else x.new_empty(0, k)
    if k > 1 and rows.stride(1) != 1:
        rows = rows.contiguous()
    out = torch.empty(*x.shape[:-1], n, device=x.device, dtype=x.dtype)
    if rows.shape[0] > 0:
        with torch.cuda.device(x.device):
            rc = _lib.lib().sy_linear4(_ptr(rows), rows.stride(0), _ptr(tiles), _ptr(scales),
                                       None if zeros is None else _ptr(zeros), _ptr(out), rows.shape[0], n, k, group,
                                       _lib.dtype_code(x.dtype), _lib.stream_ptr(x.device))
        _lib.check(rc, "sy_linear4")
    return out


_untraced = torch.compiler.disable(_linear4)  # what a compiler's trace calls


class Linear4(nn.Module):
    """A projection with 4-bit weights, for inference. Under autocast activations are taken in
    the scales' dtype and the output has autocast's."""

    def __init__(self, weight: Weight4) -> None:
        super().__init__()
        self.out_features, self.in_features, self.group = weight.out_features, weight.in_features, weight.group
        self.register_buffer("tiles", weight.tiles)
        self.register_buffer("scales", weight.scales)
        self.register_buffer("zeros", weight.zeros)

    @classmethod
    def from_linear(cls, linear: nn.Linear, group: int = 64, *, symmetric: bool = True) -> Linear4:
        """The 4-bit form of a projection that is its weights' product and nothing else: no bias, no
        hooks, no ``forward`` of its own."""
        cls.check(linear)
        return cls(quantize4(linear.weight, group, symmetric=symmetric))

    @staticmethod
    def check(linear: nn.Module) -> None:
        """Raise ValueError where ``from_linear`` would."""
        _need(getattr(linear, "bias", None) is None, "a projection with a bias has no 4-bit form")
        _need(isinstance(linear, nn.Linear) and type(linear).forward is nn.Linear.forward and "forward" not in linear.__dict__,
              f"{type(linear).__name__} is no plain projection: one with a forward of its own has no 4-bit form")
        _need(not (linear._forward_hooks or linear._forward_pre_hooks or linear._backward_hooks or linear._backward_pre_hooks),
              "a projection with hooks has no 4-bit form")

    @property
    def weight4(self) -> Weight4:
        return Weight4(self.tiles, self.scales, self.zeros, self.out_features, self.in_features, self.group)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        args = (self.tiles, self.scales, self.zeros, self.out_features, self.in_features, self.group)
        if torch.is_autocast_enabled("cuda"):
            return _linear4(x.to(self.scales.dtype), *args).to(torch.get_autocast_dtype("cuda"))
        return _linear4(x, *args)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, group={self.group}"
