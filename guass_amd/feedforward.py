"""The feed-forward half of an adapted transformer block on hand-written gfx950 kernels.

* ``gated_linear``        dropout(value * act(gate)), (value, gate) the two halves of x W^T + b
* ``linear_dropout_add``  residual + dropout(x W^T + b)
* ``dropout_add``         residual + dropout(x)

each with its gradients.  W may be what an adapted layer renders (weight + delta-W): its gradient is then
the field's dL/d(delta-W), and ``guass_amd.layers.GaussianFeedForward`` runs the three that way.

Types: float32, bfloat16 and float16, one type for all of a call's tensors; sums are accumulated in 32
bits.  Every call runs on torch's current stream of its tensors' device and does not synchronise.  A
matrix whose last dimension is contiguous is read in place whatever its row stride is; others are copied.

Dropout draws from a counter-based generator, Philox4x32-10, keyed by ``seed``: element (row, col) takes 16
bits of the block at counter (col // 8, row, ``offset``), the output seen as a matrix of its last dimension's
rows.  Nothing is stored: the backward makes the mask again, and two calls with the same seed and offset drop
the same elements, so give every call of a step an offset (or seed) of its own.  An element is dropped, and
then exactly 0, with the probability p rounded to a multiple of 2^-16, and divided by the share kept
otherwise.  ``seed`` may be an int64 tensor of one element on the device, read when the kernels run: a
captured graph draws anew at every replay if the program changes it between them.
"""

from __future__ import annotations

import ctypes

import torch
from torch import Tensor

from guass_amd import _native as N
from guass_amd.cuda_field.ext import _on_device

ACTIVATIONS = tuple(a for a in N.GF_ACTIVATIONS if a is not None)

__all__ = ["ACTIVATIONS", "dropout_add", "gated_linear", "linear_dropout_add"]


# ------------------------------------------------------------------------------------ checks

def _check_tensor(t: Tensor, name: str, like: Tensor | None) -> None:
    """A CUDA tensor of x's type and device (like None: x itself)."""
    if not isinstance(t, Tensor):
        raise TypeError(f"{name} must be a tensor")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    if like is None:
        if t.dtype not in N.GF_DTYPES:
            raise RuntimeError(f"{name} must be float32, bfloat16 or float16 (got {t.dtype})")
    elif t.dtype != like.dtype:
        raise RuntimeError(f"{name} must be {like.dtype} like x (got {t.dtype})")
    elif t.device != like.device:
        raise RuntimeError(f"all tensors must be on the same device (got {like.device} and {t.device})")


def _check_rng(p: float, seed, offset: int, x: Tensor) -> None:
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p must lie in [0, 1] (got {p})")
    if not 0 <= offset < 2**64:
        raise ValueError(f"offset must lie in [0, 2^64) (got {offset})")
    if isinstance(seed, Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1 or seed.device != x.device:
            raise RuntimeError("a seed tensor must be one int64 element on x's device")
    elif not 0 <= seed < 2**64:
        raise ValueError(f"seed must lie in [0, 2^64) (got {seed})")


def _check_linear(x: Tensor, weight: Tensor, bias: Tensor | None, out_rows: int) -> None:
    """out_rows: rows of weight per output column (2: gated)."""
    _check_tensor(x, "x", None)
    _check_tensor(weight, "weight", x)
    if x.dim() < 1 or weight.dim() != 2:
        raise RuntimeError("x must have shape [..., in_features] and weight two dimensions")
    rows, cols = weight.shape
    if rows == 0 or cols == 0:
        raise RuntimeError("weight must not be empty")
    if rows % out_rows:
        raise RuntimeError("a gated weight must have an even number of rows: the value's, then the gate's")
    if x.size(-1) != cols:
        raise RuntimeError(f"x has {x.size(-1)} features, weight takes {cols}")
    if bias is not None:
        _check_tensor(bias, "bias", x)
        if bias.dim() != 1 or bias.size(0) != rows:
            raise RuntimeError(f"bias must have shape [{rows}]")


def _matrix(t: Tensor) -> tuple[Tensor, int, int]:
    """(t as a matrix of its last dimension's rows with unit column stride, its rows, its row stride); a copy
    only where no view is one."""
    cols = t.size(-1)
    if t.is_contiguous():
        return t, t.numel() // cols, cols
    if t.dim() != 2:
        t = t.reshape(-1, cols)
    rows, (ld, one) = t.size(0), t.stride()
    if one != 1 and cols > 1 or ld < cols and rows > 1:
        t, ld = t.contiguous(), cols
    return t, rows, ld if rows > 1 else cols


def _dropout_struct(p: float, seed, offset: int) -> N.GfDropout:
    if isinstance(seed, Tensor):
        return N.GfDropout(p, 0, seed.data_ptr(), offset)
    return N.GfDropout(p, seed, None, offset)


# ------------------------------------------------------------------------------- the kernels

def _dropout_kernel(x: Tensor, residual: Tensor | None, p: float, seed, offset: int) -> Tensor:
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    if y.numel() == 0:
        return y
    dev = x.device
    if x.dim() == 0:
        x, residual = x.view(1), None if residual is None else residual.view(1)
    x, rows, ldx = _matrix(x)
    cols = x.size(-1)
    r, ldr = None, 0
    if residual is not None:
        r, _, ldr = _matrix(residual)
    with _on_device(dev):
        rc = N.lib().gf_dropout_add(N.GF_DTYPES[y.dtype], ctypes.byref(_dropout_struct(p, seed, offset)), rows, cols,
                                    x.data_ptr(), ldx, None if r is None else r.data_ptr(), ldr, y.data_ptr(), cols,
                                    N.stream_handle(dev))
        if rc:
            N.check(rc, "gf_dropout_add")
    return y


# Workspace bytes by what they depend on: a product's sizes, strides and the alignment of what it reads.
_WORKSPACE: dict[tuple, int] = {}


def _call(a: N.GfFfArgs, backward: bool, device: torch.device) -> None:
    """Runs a phase on the current stream, its workspace from torch's allocator on that stream."""
    L, ref = N.lib(), ctypes.byref(a)
    key = (backward, a.dtype, a.activation, a.rows, a.in_features, a.out_features, a.ldx, a.ldw, a.lddy, a.x % 16, a.weight % 16,
           (a.dy or 0) % 16, a.dropout.p, a.dx is None, a.dweight is None, a.dbias is None)
    n = _WORKSPACE.get(key)
    if n is None:
        if len(_WORKSPACE) > 4096:
            _WORKSPACE.clear()
        n = _WORKSPACE[key] = int(L.gf_ff_workspace_bytes(ref, int(backward)))
    ws = torch.empty(n, dtype=torch.uint8, device=device) if n else None
    name = "gf_ff_backward" if backward else "gf_ff_forward"
    rc = getattr(L, name)(ref, ws.data_ptr() if n else None, n, N.stream_handle(device))
    if rc:
        N.check(rc, name)


def _args(x: Tensor, weight: Tensor, act: str | None, p: float, seed, offset: int) -> tuple[N.GfFfArgs, tuple]:
    """The arguments both phases share, and the tensors they point into."""
    x, rows, ldx = _matrix(x)
    weight, weight_rows, ldw = _matrix(weight)
    a = N.GfFfArgs(N.GF_DTYPES[x.dtype], N.GF_ACTIVATIONS[act], rows, x.size(-1), weight_rows if act is None else weight_rows // 2,
                   x.data_ptr(), ldx, weight.data_ptr(), ldw)
    a.dropout = _dropout_struct(p, seed, offset)
    return a, (x, weight)


def _linear_forward(x: Tensor, weight: Tensor, bias: Tensor | None, residual: Tensor | None, act: str | None, p: float,
                    seed, offset: int, save: bool) -> tuple[Tensor, Tensor | None]:
    """(y, what the backward needs of the products; None for a linear product)."""
    dev = x.device
    y = x.new_empty((*x.shape[:-1], weight.size(0) // (1 if act is None else 2)))
    if y.numel() == 0:
        return y, None
    with _on_device(dev):
        a, keep = _args(x, weight, act, p, seed, offset)
        saved = None
        if save and act is not None:
            saved = torch.empty(N.lib().gf_ff_saved_bytes(ctypes.byref(a)), dtype=torch.uint8, device=dev)
            a.saved = saved.data_ptr()
        a.y = y.data_ptr()
        if bias is not None:
            bias = bias.contiguous()
            a.bias = bias.data_ptr()
        if residual is not None:
            residual, _, a.ldr = _matrix(residual)
            a.residual = residual.data_ptr()
        _call(a, False, dev)
    return y, saved


def _linear_backward(x: Tensor, weight: Tensor, saved: Tensor | None, dy: Tensor, act: str | None, p: float, seed,
                     offset: int, want: tuple[bool, bool, bool]) -> tuple[Tensor | None, Tensor | None, Tensor | None]:
    """The gradients of x, weight and bias that are wanted."""
    make = Tensor.new_empty if dy.numel() else Tensor.new_zeros  # no rows: every sum is empty
    dx = make(x, x.shape) if want[0] else None
    dw = make(x, weight.shape) if want[1] else None
    db = make(x, weight.shape[:1]) if want[2] else None
    if dy.numel() and any(want):
        with _on_device(x.device):
            a, keep = _args(x, weight, act, p, seed, offset)
            dy, _, a.lddy = _matrix(dy)
            a.dy = dy.data_ptr()
            if saved is not None:
                a.saved = saved.data_ptr()
            if dx is not None:
                a.dx = dx.data_ptr()
            if dw is not None:
                a.dweight = dw.data_ptr()
            if db is not None:
                a.dbias = db.data_ptr()
            _call(a, True, x.device)
    return dx, dw, db


# ---------------------------------------------------------------------------------- autograd

class _Once(torch.autograd.Function):
    """Differentiated once only: a backward under create_graph gives gradients that refuse another one.  (Without
    it grad mode is off, and the decorator's cost is saved.)"""

    @classmethod
    def run(cls, ctx, dy):
        if torch.is_grad_enabled():
            return torch.autograd.function.once_differentiable(cls.gradients)(ctx, dy)
        return cls.gradients(ctx, dy)


class _DropoutAdd(_Once):
    @staticmethod
    def forward(ctx, x, residual, p, seed, offset):
        ctx.rng = (p, seed, offset)
        if isinstance(seed, Tensor):
            ctx.rng = (p, None, offset)
            ctx.save_for_backward(seed)
        return _dropout_kernel(x, residual, p, seed, offset)

    @staticmethod
    def gradients(ctx, dy):
        p, seed, offset = ctx.rng
        if seed is None:
            seed, = ctx.saved_tensors
        need = ctx.needs_input_grad
        return _dropout_kernel(dy, None, p, seed, offset) if need[0] else None, dy if need[1] else None, None, None, None

    @staticmethod
    def backward(ctx, dy):
        return _DropoutAdd.run(ctx, dy)


class _Linear(_Once):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, p, seed, offset):
        y, saved = _linear_forward(x, weight, bias, residual, act, p, seed, offset, save=any(ctx.needs_input_grad[:3]))
        ctx.call = (act, p, None if isinstance(seed, Tensor) else seed, offset)
        ctx.save_for_backward(x, weight, saved, seed if isinstance(seed, Tensor) else None)
        return y

    @staticmethod
    def gradients(ctx, dy):
        act, p, seed, offset = ctx.call
        x, weight, saved, seed_tensor = ctx.saved_tensors
        need = ctx.needs_input_grad
        grads = _linear_backward(x, weight, saved, dy, act, p, seed if seed_tensor is None else seed_tensor, offset, need[:3])
        return *grads, dy if need[3] else None, None, None, None, None

    @staticmethod
    def backward(ctx, dy):
        return _Linear.run(ctx, dy)


def _wants_grad(*ts: Tensor | None) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


# ----------------------------------------------------------------------------------- public

def dropout_add(x: Tensor, residual: Tensor | None = None, *, p: float, seed: int | Tensor, offset: int = 0) -> Tensor:
    """residual + dropout(x), or dropout(x); x of any shape, residual of x's."""
    _check_tensor(x, "x", None)
    if residual is not None:
        _check_tensor(residual, "residual", x)
        if residual.shape != x.shape:
            raise RuntimeError(f"residual must have x's shape {tuple(x.shape)} (got {tuple(residual.shape)})")
    _check_rng(p, seed, offset, x)
    if _wants_grad(x, residual):
        return _DropoutAdd.apply(x, residual, p, seed, offset)
    return _dropout_kernel(x, residual, p, seed, offset)


def gated_linear(x: Tensor, weight: Tensor, bias: Tensor | None = None, *, activation: str = "gelu", p: float = 0.0,
                 seed: int | Tensor = 0, offset: int = 0) -> Tensor:
    """dropout(value * activation(gate)) of x [..., in]: the first half of weight's rows [2 out, in] (and of bias
    [2 out]) makes the value, the second the gate.  ``activation``: "gelu" (by the error function), "gelu_tanh"
    or "silu".  Where a gradient is wanted, value and gate are kept in x's type for the backward."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {ACTIVATIONS} (got {activation!r})")
    _check_linear(x, weight, bias, 2)
    _check_rng(p, seed, offset, x)
    if _wants_grad(x, weight, bias):
        return _Linear.apply(x, weight, bias, None, activation, p, seed, offset)
    return _linear_forward(x, weight, bias, None, activation, p, seed, offset, save=False)[0]


def linear_dropout_add(x: Tensor, weight: Tensor, bias: Tensor | None = None, residual: Tensor | None = None, *,
                       p: float = 0.0, seed: int | Tensor = 0, offset: int = 0) -> Tensor:
    """residual + dropout(x W^T + bias) of x [..., in], weight [out, in], bias [out], residual [..., out]."""
    _check_linear(x, weight, bias, 1)
    if residual is not None:
        _check_tensor(residual, "residual", x)
        if residual.shape != (*x.shape[:-1], weight.size(0)):
            raise RuntimeError(f"residual must have shape {(*x.shape[:-1], weight.size(0))} (got {tuple(residual.shape)})")
    _check_rng(p, seed, offset, x)
    if _wants_grad(x, weight, bias, residual):
        return _Linear.apply(x, weight, bias, residual, None, p, seed, offset)
    return _linear_forward(x, weight, bias, residual, None, p, seed, offset, save=False)[0]
