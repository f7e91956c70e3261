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
from guass_amd.cuda_field.ext import _on_device, _same_device

ACTIVATIONS = tuple(a for a in N.GF_ACTIVATIONS if a is not None)

__all__ = ["ACTIVATIONS", "dropout_add", "gated_linear", "linear_dropout_add"]


# ------------------------------------------------------------------------------------ checks

def _check_tensor(t: Tensor, name: str, dtype: torch.dtype | None) -> None:
    if not isinstance(t, Tensor):
        raise TypeError(f"{name} must be a tensor")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    if dtype is None:
        if t.dtype not in N.GF_DTYPES:
            raise RuntimeError(f"{name} must be float32, bfloat16 or float16 (got {t.dtype})")
    elif t.dtype != dtype:
        raise RuntimeError(f"{name} must be {dtype} like x (got {t.dtype})")


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
    _check_tensor(weight, "weight", x.dtype)
    if x.dim() < 1 or weight.dim() != 2:
        raise RuntimeError("x must have shape [..., in_features] and weight two dimensions")
    if weight.size(0) == 0 or weight.size(1) == 0:
        raise RuntimeError("weight must not be empty")
    if weight.size(0) % out_rows:
        raise RuntimeError("a gated weight must have an even number of rows: the value's, then the gate's")
    if x.size(-1) != weight.size(1):
        raise RuntimeError(f"x has {x.size(-1)} features, weight takes {weight.size(1)}")
    if bias is not None:
        _check_tensor(bias, "bias", x.dtype)
        if bias.shape != weight.shape[:1]:
            raise RuntimeError(f"bias must have shape [{weight.size(0)}]")
    _same_device(*(t for t in (x, weight, bias) if t is not None))


def _rows(t: Tensor) -> Tensor:
    """t as a matrix of its last dimension's rows, unit column stride; a copy only where no view is one."""
    if t.dim() != 2:
        t = t.reshape(-1, t.size(-1)) if t.numel() else t.new_empty(t.shape[:-1].numel(), t.size(-1))
    if t.stride(1) != 1 and t.size(1) > 1 or t.stride(0) < t.size(1) and t.size(0) > 1:
        t = t.contiguous()
    return t


def _ld(t: Tensor) -> int:
    return t.stride(0) if t.size(0) > 1 else t.size(1)


def _dropout_struct(p: float, seed, offset: int) -> N.GfDropout:
    if isinstance(seed, Tensor):
        return N.GfDropout(p, 0, seed.data_ptr(), offset)
    return N.GfDropout(p, seed, None, offset)


# ------------------------------------------------------------------------------- the kernels

def _dropout_kernel(x: Tensor, residual: Tensor | None, p: float, seed, offset: int) -> Tensor:
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if x.numel() == 0:
        return y
    a = _rows(x if x.dim() else x.reshape(1))
    r = None if residual is None else _rows(residual if residual.dim() else residual.reshape(1))
    with _on_device(x.device):
        N.check(N.lib().gf_dropout_add(N.GF_DTYPES[x.dtype], ctypes.byref(_dropout_struct(p, seed, offset)), a.size(0),
                                       a.size(1), a.data_ptr(), _ld(a), None if r is None else r.data_ptr(),
                                       0 if r is None else _ld(r), y.data_ptr(), a.size(1), N.stream_handle(x.device)),
                "gf_dropout_add")
    return y


def _args(x: Tensor, weight: Tensor, act: str | None, p: float, seed, offset: int) -> N.GfFfArgs:
    a = N.GfFfArgs()
    a.dtype, a.activation = N.GF_DTYPES[x.dtype], N.GF_ACTIVATIONS[act]
    a.rows, a.in_features = x.shape
    a.out_features = weight.size(0) // (1 if act is None else 2)
    a.x, a.ldx, a.weight, a.ldw = x.data_ptr(), _ld(x), weight.data_ptr(), _ld(weight)
    a.dropout = _dropout_struct(p, seed, offset)
    return a


def _call(name: str, a: N.GfFfArgs, backward: bool, device: torch.device) -> None:
    """Runs a phase on the current stream, its workspace from torch's allocator on that stream."""
    L, ref = N.lib(), ctypes.byref(a)
    n = L.gf_ff_workspace_bytes(ref, int(backward))
    ws = torch.empty(n, dtype=torch.uint8, device=device) if n else None
    N.check(getattr(L, name)(ref, N.ptr(ws), n, N.stream_handle(device)), name)


def _linear_forward(x: Tensor, weight: Tensor, bias: Tensor | None, residual: Tensor | None, act: str | None, p: float,
                    seed, offset: int, save: bool) -> tuple[Tensor, Tensor | None]:
    """(y, what the backward needs of the products; None for a linear product)."""
    x2, w2 = _rows(x), _rows(weight)
    with _on_device(x.device):
        a = _args(x2, w2, act, p, seed, offset)
        y = torch.empty(*x.shape[:-1], a.out_features, dtype=x.dtype, device=x.device)
        if y.numel() == 0:
            return y, None
        saved = None
        if save and act is not None:
            saved = torch.empty(N.lib().gf_ff_saved_bytes(ctypes.byref(a)), dtype=torch.uint8, device=x.device)
        b = None if bias is None else bias.contiguous()
        r = None if residual is None else _rows(residual)
        a.y, a.saved, a.bias = y.data_ptr(), N.ptr(saved), N.ptr(b)
        a.residual, a.ldr = (None, 0) if r is None else (r.data_ptr(), _ld(r))
        _call("gf_ff_forward", a, False, x.device)
    return y, saved


def _linear_backward(x: Tensor, weight: Tensor, saved: Tensor | None, dy: Tensor, act: str | None, p: float, seed,
                     offset: int, want: tuple[bool, bool, bool]) -> tuple[Tensor | None, Tensor | None, Tensor | None]:
    """The gradients of x, weight and bias that are wanted."""
    make = torch.empty if dy.numel() else torch.zeros  # no rows: every sum is empty
    new = {"dtype": x.dtype, "device": x.device}
    dx = make(x.shape, **new) if want[0] else None
    dw = make(weight.shape, **new) if want[1] else None
    db = make(weight.size(0), **new) if want[2] else None
    if dy.numel() and any(want):
        x2, w2, dy2 = _rows(x), _rows(weight), _rows(dy)
        with _on_device(x.device):
            a = _args(x2, w2, act, p, seed, offset)
            a.dy, a.lddy, a.saved = dy2.data_ptr(), _ld(dy2), N.ptr(saved)
            a.dx, a.dweight, a.dbias = N.ptr(dx), N.ptr(dw), N.ptr(db)
            _call("gf_ff_backward", a, True, x.device)
    return dx, dw, db


# ---------------------------------------------------------------------------------- autograd

class _DropoutAdd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, offset):
        ctx.rng = (p, None if isinstance(seed, Tensor) else seed, offset)
        if isinstance(seed, Tensor):
            ctx.save_for_backward(seed)
        return _dropout_kernel(x, residual, p, seed, offset)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        p, seed, offset = ctx.rng
        if seed is None:
            seed, = ctx.saved_tensors
        dx = _dropout_kernel(dy, None, p, seed, offset) if ctx.needs_input_grad[0] else None
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, p, seed, offset):
        y, saved = _linear_forward(x, weight, bias, residual, act, p, seed, offset, save=any(ctx.needs_input_grad[:3]))
        ctx.call = (act, p, None if isinstance(seed, Tensor) else seed, offset)
        ctx.save_for_backward(x, weight, saved, seed if isinstance(seed, Tensor) else None)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        act, p, seed, offset = ctx.call
        x, weight, saved, seed_tensor = ctx.saved_tensors
        need = ctx.needs_input_grad
        grads = _linear_backward(x, weight, saved, dy, act, p, seed if seed_tensor is None else seed_tensor, offset, need[:3])
        return *grads, dy if need[3] else None, None, None, None, None


def _wants_grad(*ts: Tensor | None) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


# ----------------------------------------------------------------------------------- public

def dropout_add(x: Tensor, residual: Tensor | None = None, *, p: float, seed: int | Tensor, offset: int = 0) -> Tensor:
    """residual + dropout(x), or dropout(x); x of any shape, residual of x's."""
    _check_tensor(x, "x", None)
    if residual is not None:
        _check_tensor(residual, "residual", x.dtype)
        if residual.shape != x.shape:
            raise RuntimeError(f"residual must have x's shape {tuple(x.shape)} (got {tuple(residual.shape)})")
        _same_device(x, residual)
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
        _check_tensor(residual, "residual", x.dtype)
        if residual.shape != (*x.shape[:-1], weight.size(0)):
            raise RuntimeError(f"residual must have shape {(*x.shape[:-1], weight.size(0))} (got {tuple(residual.shape)})")
        _same_device(x, residual)
    _check_rng(p, seed, offset, x)
    if _wants_grad(x, weight, bias, residual):
        return _Linear.apply(x, weight, bias, residual, None, p, seed, offset)
    return _linear_forward(x, weight, bias, residual, None, p, seed, offset, save=False)[0]
