"""Weights in 4 bits, and products with them, on hand-written gfx950 kernels.

* ``quantize``                a weight into codes and scales (a ``QuantizedWeight``)
* ``quantized_linear``        residual + x W^T + b
* ``quantized_gated_linear``  value * act(gate), (value, gate) the two halves of x W^T + b

A weight that does not train is kept so: what a trained adapter was merged into or a frozen layer (``guass_amd.layers.QuantizedLinear``,
``QuantizedFeedForward``).  Gradients go through it to the inputs of these functions; a layer that trains an adapter beside a 4-bit base is not
here (``GaussianLinear`` has a dense one).  The format is the OCP microscaling formats' MXFP4: groups of
32 along a row share a scale 2^e, and an element is a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6.  4.25 bits an element; its value is exact in
bfloat16, and in float16 where the scale lies in [2^-23, 2^13] (past that, it is rounded to float16).

The products' other tensors are of one type, float32, bfloat16 or float16; sums are accumulated in 32 bits.  Under ``torch.autocast``
x and the bias take its type, as in nn.Linear.  At most 128 rows read the codes as they are; more, and
a gated product's training pass, write the weight's values out for the call and run the products of ``guass_amd.feedforward``, backward too: the
gradients of x, bias and residual, none of the weight.  As there, a gated product's backward keeps value and gate in 20 (bfloat16) or 24
bits (float16) and rounds dz, the products' gradient, to the tensors' type before dx = dz W: in 16 bits dx has two roundings, a
linear product's one.  Every call runs on torch's current stream of its tensors' device and does not synchronise.
"""

from __future__ import annotations

import threading

import torch
from torch import Tensor

from guass_amd import _native as N
from guass_amd import feedforward
from guass_amd.feedforward import ACTIVATIONS

__all__ = ["QuantizedWeight", "quantize", "quantized_gated_linear", "quantized_linear"]

GROUP = 32

_OPS = None
_LOADING = threading.Lock()


def _ops() -> tuple:
    """(q4_linear, q4_quantize, q4_dequantize), loaded once a process (a global: a trace reads it as it is)."""
    global _OPS
    if _OPS is None:
        with _LOADING:
            if _OPS is None:
                feedforward._ops()  # loads the operators' library
                _register_shapes()
                ops = torch.ops.guass_amd
                _OPS = ops.q4_linear.default, ops.q4_quantize.default, ops.q4_dequantize.default
    return _OPS


def _register_shapes() -> None:
    fake = torch.library.register_fake

    @fake("guass_amd::q4_quantize")
    def _(weight):
        tiles = (weight.shape[0] + 15) // 16, (weight.shape[1] + 127) // 128
        return weight.new_empty((*tiles, 1024), dtype=torch.uint8), weight.new_empty((*tiles, 64), dtype=torch.uint8)

    @fake("guass_amd::q4_dequantize")
    def _(codes, scales, rows, cols, dtype):
        return codes.new_empty((rows, cols), dtype=dtype)

    @fake("guass_amd::q4_forward")
    def _(x, codes, scales, bias, residual, rows, cols, activation, save):
        out = rows // (2 if activation else 1)
        y = x.new_empty((*x.shape[:-1], out))
        if not (save and activation):
            return y, None
        return y, x.new_empty((y.numel() // out * feedforward._saved_bytes(x.dtype, out),), dtype=torch.uint8)

    @fake("guass_amd::q4_backward")
    def _(dy, codes, scales, saved, rows, cols, activation, want_x, want_b):
        return dy.new_empty((*dy.shape[:-1], cols)) if want_x else None, dy.new_empty((rows,)) if want_b else None


def _fill(t: Tensor, rows: int, cols: int) -> Tensor:
    """t with zeros below and right of it."""
    return torch.nn.functional.pad(t, (0, cols - t.shape[1], 0, rows - t.shape[0]))


class QuantizedWeight:
    """A weight [rows, in_features] in 4 bits, made of ``codes`` uint8 [rows, 16 ceil(in_features / 32)] (two elements a byte, the first in
    the low half, each a sign (8) and the place of its magnitude among 0, 0.5, 1, 1.5, 2, 3, 4, 6; zero past the row) and ``scales`` uint8
    [rows, ceil(in_features / 32)] (e + 127 of a group's 2^e, 255 for NaN).

    Held as the kernels read it, in tiles of 16 rows and 128 columns: ``tile_codes`` uint8 [ceil(rows / 16), ceil(in_features / 128), 1024]
    and ``tile_scales`` [..., 64].  Of the words of 8 codes of a tile's row, word 4 j + q lies at (16 q + row) * 4 + j; the scale of
    group j at 4 row + j."""

    __slots__ = ("tile_codes", "tile_scales", "rows", "in_features")

    def __init__(self, codes: Tensor, scales: Tensor, in_features: int):
        for name, t in (("codes", codes), ("scales", scales)):
            if not isinstance(t, Tensor):
                raise TypeError(f"{name} must be a tensor")
            if t.dtype != torch.uint8:
                raise ValueError(f"{name} must be uint8 (got {t.dtype})")
        if in_features < 1:
            raise ValueError(f"in_features must be positive (got {in_features})")
        groups = (in_features + GROUP - 1) // GROUP
        if codes.dim() != 2 or scales.shape != (codes.shape[0], groups) or codes.shape[1] != 16 * groups:
            raise ValueError(f"a weight of {in_features} features has codes [rows, {16 * groups}] and scales [rows, {groups}] "
                             f"(got {list(codes.shape)} and {list(scales.shape)})")
        if codes.device != scales.device:
            raise ValueError(f"codes and scales must be on the same device (got {codes.device} and {scales.device})")
        bands, across = (codes.shape[0] + 15) // 16, (in_features + 127) // 128
        words = _fill(codes, 16 * bands, 64 * across).view(bands, 16, across, 4, 4, 4)  # row, tile, j, q, byte
        self.tile_codes = words.permute(0, 2, 4, 1, 3, 5).reshape(bands, across, 1024)
        self.tile_scales = _fill(scales, 16 * bands, 4 * across).view(bands, 16, across, 4).permute(0, 2, 1, 3).reshape(bands, across, 64)
        self.rows, self.in_features = codes.shape[0], in_features

    @classmethod
    def from_tiles(cls, tile_codes: Tensor, tile_scales: Tensor, rows: int, in_features: int) -> "QuantizedWeight":
        """Of tiles as another one holds them."""
        tiles = (rows + 15) // 16, (in_features + 127) // 128
        for name, t, size in (("tile_codes", tile_codes, 1024), ("tile_scales", tile_scales, 64)):
            if t.dtype != torch.uint8 or t.shape != (*tiles, size):
                raise ValueError(f"{name} of a weight [{rows}, {in_features}] must be uint8 {[*tiles, size]} (got {t.dtype} {list(t.shape)})")
        if tile_codes.device != tile_scales.device:
            raise ValueError(f"tiles must be on the same device (got {tile_codes.device} and {tile_scales.device})")
        self = cls.__new__(cls)
        self.tile_codes, self.tile_scales, self.rows, self.in_features = tile_codes, tile_scales, rows, in_features
        return self

    @property
    def codes(self) -> Tensor:
        bands, across, _ = self.tile_codes.shape
        words = self.tile_codes.reshape(bands, across, 4, 16, 4, 4).permute(0, 3, 1, 4, 2, 5)
        return words.reshape(16 * bands, 64 * across)[:self.rows, :(self.in_features + GROUP - 1) // GROUP * 16].contiguous()

    @property
    def scales(self) -> Tensor:
        bands, across, _ = self.tile_scales.shape
        groups = self.tile_scales.reshape(bands, across, 16, 4).permute(0, 2, 1, 3)
        return groups.reshape(16 * bands, 4 * across)[:self.rows, :(self.in_features + GROUP - 1) // GROUP].contiguous()

    @property
    def shape(self) -> torch.Size:
        return torch.Size((self.rows, self.in_features))

    @property
    def device(self) -> torch.device:
        return self.tile_codes.device

    def to(self, device) -> "QuantizedWeight":
        return QuantizedWeight.from_tiles(self.tile_codes.to(device), self.tile_scales.to(device), self.rows, self.in_features)

    def dequantize(self, dtype: torch.dtype = torch.float32) -> Tensor:
        """The values that it stands for, [rows, in_features], rounded to ``dtype``."""
        if not self.tile_codes.is_cuda:
            raise RuntimeError("codes must be a CUDA tensor")
        return _ops()[2](self.tile_codes, self.tile_scales, self.rows, self.in_features, dtype)

    def __repr__(self) -> str:
        return f"QuantizedWeight({list(self.shape)}, device={str(self.device)!r})"


def quantize(weight: Tensor) -> QuantizedWeight:
    """weight [rows, in_features] in 4 bits.  A group's scale is the least 2^e with max |w| <= 7 * 2^e (e in [-125, 125]), an element
    the nearest value, of two as near the one with an even place.  A group with an infinity or a NaN is NaN as a whole."""
    if not isinstance(weight, Tensor):
        raise TypeError("weight must be a tensor")
    if not weight.is_cuda:
        raise RuntimeError("weight must be a CUDA tensor")
    if weight.dim() != 2:
        raise ValueError(f"weight must have two dimensions (got {list(weight.shape)})")
    weight = weight.detach()
    return QuantizedWeight.from_tiles(*_ops()[1](weight), *weight.shape)


def _check(x, weight) -> None:
    if not isinstance(x, Tensor):
        raise TypeError("x must be a tensor")
    if not isinstance(weight, QuantizedWeight):
        raise TypeError("weight must be a QuantizedWeight")


def quantized_linear(x: Tensor, weight: QuantizedWeight, bias: Tensor | None = None, residual: Tensor | None = None) -> Tensor:
    """residual + x W^T + bias of x [..., in], weight [out, in], bias [out], residual [..., out]."""
    _check(x, weight)
    return _ops()[0](x, weight.tile_codes, weight.tile_scales, bias, residual, weight.rows, weight.in_features, 0)


def quantized_gated_linear(x: Tensor, weight: QuantizedWeight, bias: Tensor | None = None, *, activation: str = "gelu") -> Tensor:
    """value * activation(gate) of x [..., in]: the first half of weight's rows [2 out, in] (and of bias [2 out]) makes the
    value, the second the gate.  Activations as ``guass_amd.feedforward.gated_linear``."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {ACTIVATIONS} (got {activation!r})")
    _check(x, weight)
    return _ops()[0](x, weight.tile_codes, weight.tile_scales, bias, None, weight.rows, weight.in_features, N.GF_ACTIVATIONS[activation])
