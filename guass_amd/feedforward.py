"""The feed-forward half of an adapted transformer block on hand-written gfx950 kernels.

* ``gated_linear``        dropout(value * act(gate)), (value, gate) the two halves of x W^T + b
* ``linear_dropout_add``  residual + dropout(x W^T + b)
* ``dropout_add``         residual + dropout(x)

each with its gradients.  W may be what an adapted layer renders (weight + delta-W): its gradient is then
the field's dL/d(delta-W), and ``guass_amd.layers.GaussianFeedForward`` runs the three that way.

Types: float32, bfloat16 and float16, one type for all of a call's tensors (under ``torch.autocast`` the products
take its type, and a residual of another type is added by torch's rules); sums are accumulated in 32 bits.  Every call runs on torch's current stream of its tensors' device and does not synchronise.  A
matrix whose last dimension is contiguous is taken whatever its row stride is; others are copied.  The products
read 16-bit matrices in place whose rows begin at 16 bytes and are a multiple of 8 wide, and lay others out in the
workspace first, as they do float32; of at most 64 rows the forward reads everything in place.
float32 products go through the matrix cores as three bfloat16 planes of each operand (errors as of float32
sums; an infinity times a number below 2^-100 may be a NaN); of at most 64 rows the forward multiplies
float32 as such.

Dropout draws from a counter-based generator, Philox4x32-10, keyed by ``seed``: element (row, col) takes 16
bits of the block at counter (col // 8, row, ``offset``), the output seen as a matrix of its last dimension's
rows.  Nothing is stored: the backward makes the mask again, and two calls with the same seed and offset drop
the same elements, so give every call of a step an offset (or seed) of its own.  An element is dropped, and
then exactly 0, with the probability p rounded to a multiple of 2^-16, and divided by the share kept
otherwise.  ``seed`` may be an int64 tensor of one element on the device, read when the kernels run: a
captured graph draws anew at every replay if the program changes it between them.
"""

from __future__ import annotations

import threading
from pathlib import Path

import torch
from torch import Tensor

from guass_amd import _native as N

ACTIVATIONS = tuple(a for a in N.GF_ACTIVATIONS if a is not None)

__all__ = ["ACTIVATIONS", "dropout_add", "gated_linear", "linear_dropout_add"]


_OPS = None
_LOADING = threading.Lock()


def _ops() -> tuple:
    """What _load found, once a process (a global: a trace reads it as it is)."""
    global _OPS
    if _OPS is None:
        with _LOADING:
            if _OPS is None:
                _OPS = _load()
    return _OPS


def _load() -> tuple:
    """torch.ops.guass_amd: the operators of libguass_torch.so (csrc/torch_ops.cpp), which checks the tensors, makes
    outputs and workspaces and carries the gradients."""
    N.lib()  # raises if the kernels' library is not built
    path = Path(__file__).with_name("libguass_torch.so")  # it takes the library that is loaded, wherever that lies
    if not path.exists():
        raise RuntimeError(f"{path} is not built; run `python -m guass_amd.build`")
    torch.ops.load_library(str(path))
    _register_shapes()
    ops = torch.ops.guass_amd
    return ops.dropout_add.default, ops.linear.default, ops.linear_forward.default, ops.linear_backward.default


def _register_shapes() -> None:
    """The operators' outputs without data: what a trace (torch.compile, FakeTensorMode) runs instead of the kernels."""
    fake = torch.library.register_fake

    @fake("guass_amd::dropout_forward")
    def _(x, residual, p, seed, seed_tensor, offset):
        return x.new_empty(x.shape)

    @fake("guass_amd::linear_forward")
    def _(x, weight, bias, residual, activation, p, seed, seed_tensor, offset, save):
        out = weight.shape[0] // (2 if activation else 1)
        y = x.new_empty((*x.shape[:-1], out))
        if not (save and activation):
            return y, None
        return y, x.new_empty((y.numel() // out * _saved_bytes(x.dtype, out),), dtype=torch.uint8)

    @fake("guass_amd::linear_backward")
    def _(x, weight, saved, dy, activation, p, seed, seed_tensor, offset, want_x, want_weight, want_bias):
        return (x.new_empty(x.shape) if want_x else None, x.new_empty(weight.shape) if want_weight else None,
                x.new_empty(weight.shape[:1]) if want_bias else None)


def _saved_bytes(dtype: torch.dtype, out: int) -> int:
    """What gf_ff_saved_bytes says of one row: whole groups of 8 elements, value and gate together."""
    return (out + 7) // 8 * 8 * {torch.float32: 8, torch.float16: 6, torch.bfloat16: 5}[dtype]


def _signed(v: int, name: str) -> int:
    """An unsigned 64-bit number as the signed one of the same bits (what an operator's argument takes)."""
    if 0 <= v < 2**63:
        return v
    if not 0 <= v < 2**64:
        raise ValueError(f"{name} must lie in [0, 2^64) (got {v})")
    return v - 2**64


def _rng(p: float, seed: int | Tensor, offset: int) -> tuple:
    """(p, seed, seed tensor, offset) as the operators take them."""
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p must lie in [0, 1] (got {p})")
    if isinstance(seed, Tensor):
        return p, 0, seed, _signed(offset, "offset")
    return p, _signed(seed, "seed"), None, _signed(offset, "offset")


def _check_tensors(**tensors) -> None:
    for name, t in tensors.items():
        if not isinstance(t, Tensor):
            raise TypeError(f"{name} must be a tensor")


def _linear_forward(x, weight, bias, residual, act, p, seed, offset, save):
    """The forward phase by itself, without autograd (a HIP graph captures this): (y, what the backward of a gated product
    needs if ``save``, else None)."""
    return _ops()[2](x, weight, bias, residual, N.GF_ACTIVATIONS[act], *_rng(p, seed, offset), save)


def _linear_backward(x, weight, saved, dy, act, p, seed, offset, want):
    """The backward phase by itself: the gradients of x, weight and bias that are wanted, None for the others."""
    return _ops()[3](x, weight, saved, dy, N.GF_ACTIVATIONS[act], *_rng(p, seed, offset), *want)


def dropout_add(x: Tensor, residual: Tensor | None = None, *, p: float, seed: int | Tensor, offset: int = 0) -> Tensor:
    """residual + dropout(x), or dropout(x); x of any shape, residual of x's."""
    _check_tensors(x=x)
    return _ops()[0](x, residual, *_rng(p, seed, offset))


def gated_linear(x: Tensor, weight: Tensor, bias: Tensor | None = None, *, activation: str = "gelu", p: float = 0.0,
                 seed: int | Tensor = 0, offset: int = 0) -> Tensor:
    """dropout(value * activation(gate)) of x [..., in]: the first half of weight's rows [2 out, in] (and of bias
    [2 out]) makes the value, the second the gate.  ``activation``: "gelu" (by the error function), "gelu_tanh"
    or "silu".  Where a gradient is wanted, value and gate are kept for the backward: of bfloat16 in 20 bits each, of
    float16 in 24, of float32 as they are."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {ACTIVATIONS} (got {activation!r})")
    _check_tensors(x=x, weight=weight)
    return _ops()[1](x, weight, bias, None, N.GF_ACTIVATIONS[activation], *_rng(p, seed, offset))


def linear_dropout_add(x: Tensor, weight: Tensor, bias: Tensor | None = None, residual: Tensor | None = None, *,
                       p: float = 0.0, seed: int | Tensor = 0, offset: int = 0) -> Tensor:
    """residual + dropout(x W^T + bias) of x [..., in], weight [out, in], bias [out], residual [..., out]."""
    _check_tensors(x=x, weight=weight)
    return _ops()[1](x, weight, bias, residual, 0, *_rng(p, seed, offset))
