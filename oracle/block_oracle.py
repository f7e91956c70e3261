"""The norms around a block, and weights in 4 bits, in 64 bits on the CPU, with bounds of what rounding may do to them.

Test infrastructure only.  ``norms`` carries every number with a bound of the distance at which 32-bit arithmetic may have left it
(a running error analysis, u = 2^-24 a rounding):

* a sum or a product adds u of its result to what its terms' bounds make of it;
* a sum of n terms adds min(n, depth) u of its terms' absolute sum: `depth` 64 for a row (24 a lane at most, the lanes by halves, 16
  waves), twice the number of rows and 64 more for a column (within groups of rows, then over them);
* 1 / sqrt(v) to within 3 u of itself, and half its argument's relative bound;
* a rounding to the tensors' type adds eps / 2 of the value, or half the smallest subnormal.
"""

from __future__ import annotations

import torch

U = 2.0**-24
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


class Approx:
    """A number in 64 bits and a bound of its 32-bit counterpart's distance."""

    def __init__(self, value, bound=None):
        self.v = value
        self.e = torch.zeros_like(value) if bound is None else bound

    def __add__(self, other):
        v = self.v + other.v
        e = self.e + other.e
        return Approx(v, e + U * (v.abs() + e))

    def __sub__(self, other):
        return self + Approx(-other.v, other.e)

    def __mul__(self, other):
        v = self.v * other.v
        e = self.v.abs() * other.e + other.v.abs() * self.e + self.e * other.e
        return Approx(v, e + U * (v.abs() + e) + 2.0**-149)

    def times(self, number: float):
        """By a number that is rounded to 32 bits itself."""
        v = self.v * number
        e = self.e * abs(number)
        return Approx(v, e + 2 * U * (v.abs() + e) + 2.0**-149)

    def row_sum(self):
        n = min(self.v.shape[-1], 64)
        return Approx(self.v.sum(-1, keepdim=True), (self.e + n * U * (self.v.abs() + self.e)).sum(-1, keepdim=True))

    def column_sum(self, dims):
        n = 1
        for d in dims:
            n *= self.v.shape[d]
        return Approx(self.v.sum(dims, keepdim=True), (self.e + (2 * n + 64) * U * (self.v.abs() + self.e)).sum(dims, keepdim=True))

    def rsqrt(self):
        v = self.v.rsqrt()
        return Approx(v, v * (0.5 * self.e / (self.v - self.e).clamp_min(1e-300) + 3 * U))

    def rounded(self, dtype):
        info = torch.finfo(dtype)
        return self.v, self.e + info.eps / 2 * (self.v.abs() + self.e) + info.smallest_normal * info.eps / 2


def _statistics(x: Approx, kind, eps):
    """(n(x), 1 / deviation)."""
    if kind is None:
        return x, None
    inverse = 1.0 / x.v.shape[-1]
    if kind == "layer":
        x = x - x.row_sum().times(inverse)
    square = (x * x).row_sum().times(inverse)
    rstd = (square + Approx(torch.full_like(square.v, eps), torch.full_like(square.v, eps * U))).rsqrt()
    return x * rstd, rstd


def _through(g: Approx, n: Approx, rstd, kind):
    if kind is None:
        return g
    inverse = 1.0 / g.v.shape[-1]
    out = g - n * (g * n).row_sum().times(inverse)
    if kind == "layer":
        out = out - g.row_sum().times(inverse)
    return out * rstd


def _reduce(t: Approx, like: torch.Tensor):
    """t summed down to like's shape ([cols], or x's with ones)."""
    if like.dim() == 1:
        s = t.column_sum(tuple(range(t.v.dim() - 1))) if t.v.dim() > 1 else t
        return Approx(s.v.reshape(-1), s.e.reshape(-1))
    dims = tuple(i for i in range(like.dim() - 1) if like.shape[i] == 1 and t.v.shape[i] != 1)
    return t.column_sum(dims) if dims else t


def _factor(d: Approx, n: Approx, like: torch.Tensor, weight, bias):
    """The gradient of what multiplies n * weight + bias, from the sums of d n and of d: these may cancel, so the bound is theirs."""
    s = _reduce(d * n, like)
    if weight is not None:
        s = s * weight
    return s if bias is None else s + _reduce(d, like) * bias


ORDER = ("x", "residual", "weight", "bias", "gate", "next_weight", "next_bias", "scale", "shift")


def norms(t: dict, *, kind=None, gate=1.0, residual_scale=1.0, eps=1e-5, next_kind=None, next_eps=1e-5, dstream=None, dnormed=None,
          dtype=torch.float32) -> dict:
    """{name: (value, bound)} of stream and normed, and where a gradient is given those of the inputs by their names.

    t: x [..., cols], and where they are there residual, weight, bias, gate (a tensor), next_weight, next_bias, scale, shift."""
    f = {k: Approx(v.detach().cpu().double()) for k, v in t.items() if v is not None}
    x, out = f["x"], {}
    branch, stream = "residual" in f, f["x"]
    one = Approx(torch.ones((), dtype=torch.float64))
    if branch:
        n1, rstd1 = _statistics(x, kind, eps)
        u = n1
        if "weight" in f:
            u = u * f["weight"]
        if "bias" in f:
            u = u + f["bias"]
        gated = u * f["gate"] if "gate" in f else u.times(gate)
        stream = f["residual"].times(residual_scale) + gated
        out["stream"] = stream.rounded(dtype)
    if next_kind is not None:
        n2, rstd2 = _statistics(stream, next_kind, next_eps)
        h = n2 * f["next_weight"] if "next_weight" in f else n2
        if "next_bias" in f:
            h = h + f["next_bias"]
        factor = one + f["scale"] if "scale" in f else one
        h = h * factor
        if "shift" in f:
            h = h + f["shift"]
        out["normed"] = h.rounded(dtype)
    if dstream is None and dnormed is None:
        return out
    d = None if dstream is None else Approx(dstream.detach().cpu().double())
    grads = {}
    if next_kind is not None:
        dnormed = torch.zeros(x.v.shape) if dnormed is None else dnormed
        dh = Approx(dnormed.detach().cpu().double())
        g = dh * factor
        for name, v in (("next_weight", g * n2), ("next_bias", g), ("shift", dh)):
            if name in f:
                grads[name] = _reduce(v, t[name])
        if "scale" in f:
            grads["scale"] = _factor(dh, n2, t["scale"], f.get("next_weight"), f.get("next_bias"))
        if "next_weight" in f:
            g = g * f["next_weight"]
        through = _through(g, n2, rstd2, next_kind)
        d = through if d is None else d + through
    if not branch:
        grads["x"] = d
    else:
        grads["residual"] = d.times(residual_scale)
        if "gate" in f:
            grads["gate"] = _factor(d, n1, t["gate"], f.get("weight"), f.get("bias"))
        du = d * f["gate"] if "gate" in f else d.times(gate)
        if "weight" in f:
            grads["weight"] = _reduce(du * n1, t["weight"])
        if "bias" in f:
            grads["bias"] = _reduce(du, t["bias"])
        if "weight" in f:
            du = du * f["weight"]
        grads["x"] = _through(du, n1, rstd1, kind)
    for k, v in grads.items():
        out["d" + k] = v.rounded(dtype)
    return out


def power(e: torch.Tensor) -> torch.Tensor:
    """2^e, exactly, in 64 bits."""
    return torch.tensor([2.0**i for i in range(-200, 201)], dtype=torch.float64)[e.long() + 200]


def quantize(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of w [rows, cols], by the definition: every value's distance looked at."""
    w = w.detach().cpu().double()
    rows, cols = w.shape
    groups = -(-cols // 32)
    full = torch.zeros(rows, groups * 32, dtype=torch.float64)
    full[:, :cols] = w
    full = full.view(rows, groups, 32)
    finite = torch.isfinite(full).all(-1)
    amax = torch.where(finite, full.abs().amax(-1), 0.0)
    e = torch.full(amax.shape, -125)
    for i in range(-125, 125):  # the least that holds it, at most 125
        e = torch.where((amax > 7 * 2.0**i), i + 1, e)
    a = torch.where(finite[..., None], full, 0.0) / power(e)[..., None]
    near = (a.abs()[..., None] - torch.tensor(VALUES, dtype=torch.float64)).abs()
    # of two as near, the even place: those first
    order = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7])
    place = order[near[..., order].argmin(-1)]
    code = torch.where(torch.signbit(a), place + 8, place).to(torch.uint8)
    code = torch.where(finite[..., None], code, 0).to(torch.uint8).view(rows, -1, 2)
    return code[..., 0] | code[..., 1] << 4, torch.where(finite, e + 127, 255).to(torch.uint8)


def dequantize(codes: torch.Tensor, scales: torch.Tensor, cols: int) -> torch.Tensor:
    """The values in 64 bits."""
    codes, scales = codes.cpu(), scales.cpu()
    table = torch.tensor(VALUES + tuple(-v for v in VALUES), dtype=torch.float64)
    code = torch.stack((codes & 15, codes >> 4), -1).view(codes.shape[0], -1, 32).long()
    scale = torch.where(scales == 255, float("nan"), power(scales.int() - 127))
    return (table[code] * scale[..., None]).view(codes.shape[0], -1)[:, :cols]
