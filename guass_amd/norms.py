"""The norms before and after a block, with its gate and the residual's scale, on hand-written gfx950 kernels.

* ``norm``           norm(x) * weight + bias, times (1 + scale) plus shift: what a block gets
* ``gate_add``       residual_scale * residual + gate * norm(x): its way back into the stream
* ``gate_add_norm``  both in one pass: the stream, and the norm that the next block gets

each with its gradients.  A row is the last dimension; statistics and sums are held in 32 bits, and an output is rounded
once: ``gate_add_norm``'s norm is that of the stream before its rounding.  For the backward they keep their inputs, and nothing else:
``gate_add`` x where a norm or the gate's gradient needs it, and not the residual.

Types: float32, bfloat16 and float16, one type for all of a call's tensors; under ``torch.autocast`` float32, as torch's
layer_norm.  Rows of 1 to 16384 elements.  ``weight`` and ``bias`` have a row's shape.  ``gate``, ``scale`` and ``shift`` have it too, or
that of x with ones behind its first dimensions ([samples, 1, features] of x [samples, places, features]: one row a
sample); those of a call that are not shared by all rows are shared by the same ones.  Rows of a larger matrix (slices of one
modulation, say) are read in place.  Every call runs on torch's current stream of its tensors' device and does not synchronise.
Squares are summed in 32 bits: a row with elements past about 10^19 has no statistics.  A factor goes into weight and bias before the row does:
an infinite gate or scale beside a bias gives a NaN where its two infinities differ in sign.
"""

from __future__ import annotations

import threading

import torch
from torch import Tensor

from guass_amd import _native as N
from guass_amd import feedforward

NORMS = tuple(k for k in N.GF_NORMS if k is not None)

__all__ = ["NORMS", "gate_add", "gate_add_norm", "norm"]

_OPS = None
_LOADING = threading.Lock()


def _ops():
    """The operator, loaded once a process (a global: a trace reads it as it is)."""
    global _OPS
    if _OPS is None:
        with _LOADING:
            if _OPS is None:
                feedforward._ops()  # loads the operators' library
                _register_shapes()
                _OPS = torch.ops.guass_amd.block_norm.default
    return _OPS


def _register_shapes() -> None:
    fake = torch.library.register_fake

    @fake("guass_amd::block_norm_forward")
    def _(x, residual, weight, bias, gate, gate_value, residual_scale, kind, eps, next_weight, next_bias, scale, shift, next_kind, next_eps,
          want_stream):
        return (x.new_empty(x.shape) if residual is not None and want_stream else None, x.new_empty(x.shape) if next_kind else None)

    @fake("guass_amd::block_norm_backward")
    def _(x, residual, weight, bias, gate, gate_value, residual_scale, kind, eps, next_weight, next_bias, scale, shift, next_kind, next_eps,
          dstream, dnormed, wants):
        inputs = (x, residual, weight, bias, gate, next_weight, next_bias, scale, shift)
        return tuple(x.new_empty(t.shape) if t is not None and wants >> i & 1 else None for i, t in enumerate(inputs))


def _check(x, kinds: dict, numbers: dict) -> None:
    if not isinstance(x, Tensor):
        raise TypeError("x must be a tensor")
    for name, (kind, names) in kinds.items():
        if kind not in names:
            raise ValueError(f"{name} must be one of {names} (got {kind!r})")
    for name, v in numbers.items():
        if not 0.0 <= v <= 1e30:
            raise ValueError(f"{name} must be finite and not negative (got {v})")


def norm(x: Tensor, weight: Tensor | None = None, bias: Tensor | None = None, *, kind: str = "layer", scale: Tensor | None = None,
         shift: Tensor | None = None, eps: float = 1e-5) -> Tensor:
    """(n(x) * weight + bias) * (1 + scale) + shift; n(x) = (x - mean) / sqrt(variance + eps) ("layer") or
    x / sqrt(mean square + eps) ("rms")."""
    _check(x, {"kind": (kind, NORMS)}, {"eps": eps})
    return _ops()(x, None, None, None, None, 1.0, 1.0, 0, 0.0, weight, bias, scale, shift, N.GF_NORMS[kind], eps)[1]


def _branch(x, residual, weight, bias, kind, gate, residual_scale, eps) -> tuple:
    if not isinstance(residual, Tensor):
        raise TypeError("residual must be a tensor")
    if kind is None and (weight is not None or bias is not None):
        raise ValueError("a branch without a norm takes no weight or bias")
    if isinstance(gate, Tensor):
        return x, residual, weight, bias, gate, 1.0, float(residual_scale), N.GF_NORMS[kind], eps
    return x, residual, weight, bias, None, float(gate), float(residual_scale), N.GF_NORMS[kind], eps


def gate_add(x: Tensor, residual: Tensor, weight: Tensor | None = None, bias: Tensor | None = None, *, kind: str | None = None,
             gate: float | Tensor = 1.0, residual_scale: float = 1.0, eps: float = 1e-5) -> Tensor:
    """residual_scale * residual + gate * (n(x) * weight + bias); n(x) as in ``norm``, or x itself (kind None)."""
    _check(x, {"kind": (kind, (None, *NORMS))}, {"eps": eps})
    return _ops()(*_branch(x, residual, weight, bias, kind, gate, residual_scale, eps), None, None, None, None, 0, 0.0)[0]


def gate_add_norm(x: Tensor, residual: Tensor, weight: Tensor | None = None, bias: Tensor | None = None, next_weight: Tensor | None = None,
                  next_bias: Tensor | None = None, *, kind: str | None = None, gate: float | Tensor = 1.0, residual_scale: float = 1.0,
                  eps: float = 1e-5, next_kind: str = "layer", scale: Tensor | None = None, shift: Tensor | None = None,
                  next_eps: float = 1e-5) -> tuple[Tensor, Tensor]:
    """(stream, normed): stream = gate_add(x, residual, weight, bias, ...), normed = norm(stream, next_weight, next_bias,
    scale=scale, shift=shift, ...)."""
    _check(x, {"kind": (kind, (None, *NORMS)), "next_kind": (next_kind, NORMS)}, {"eps": eps, "next_eps": next_eps})
    return _ops()(*_branch(x, residual, weight, bias, kind, gate, residual_scale, eps), next_weight, next_bias, scale, shift,
                  N.GF_NORMS[next_kind], next_eps)
