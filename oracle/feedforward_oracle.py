"""The feed-forward operators in 64 bits on the CPU, with bounds of what rounding may do to them.

Test infrastructure only.  ``linear`` and ``gated`` return every output with a bound, element by element, of
the distance at which a right kernel can lie from it:

* a sum of n products in 32 bits, each product to within 8 units of 2^-24 and taken in at most 6 parts, lies
  within (6 n + 16) 2^-24 of its terms' absolute sum: 6 n additions, the 8 units, and 8 for the roundings after;
* an activation or its slope is evaluated to within 2^-20 (1 + |gate|) absolutely, and moves by at most 1.2
  times its argument (the largest slope is 1.13, the largest second derivative 0.8);
* a rounding to the tensors' type moves by u = eps / 2 of the value, or by half the smallest subnormal:
  the outputs once, a gated dz (the products' gradient) once more.  The bounds allow one to value, gate and
  a linear dz as well, more than a kernel needs that keeps value and gate in more bits and takes dy itself.
"""

from __future__ import annotations

import math

import numpy as np
import torch

MASK32 = np.uint64(0xFFFFFFFF)


def philox(counter: np.ndarray, key: tuple[int, int]) -> np.ndarray:
    """Philox4x32-10 of counters [..., 4] (uint64 holding 32 bits each)."""
    c = [counter[..., i].astype(np.uint64) for i in range(4)]
    k = list(key)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & MASK32,
             (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & MASK32]
        k = [(k[0] + 0x9E3779B9) % 2**32, (k[1] + 0xBB67AE85) % 2**32]
    return np.stack(c, axis=-1)


def keep_scale(rows: int, cols: int, p: float, seed: int, offset: int) -> torch.Tensor:
    """[rows, cols] float64: 0 where dropped, the scale elsewhere."""
    t = math.floor(p * 65536 + 0.5)
    if t == 0:
        return torch.ones(rows, cols, dtype=torch.float64)
    if t >= 65536:
        return torch.zeros(rows, cols, dtype=torch.float64)
    n = -(-cols // 8)
    ctr = np.zeros((rows, n, 4), dtype=np.uint64)
    ctr[..., 0] = np.arange(n)
    ctr[..., 1] = np.arange(rows)[:, None]
    ctr[..., 2], ctr[..., 3] = offset % 2**32, offset // 2**32
    words = philox(ctr, (seed % 2**32, seed // 2**32))
    half = np.stack((words & np.uint64(0xFFFF), words >> np.uint64(16)), axis=-1).reshape(rows, n * 8)[:, :cols]
    return torch.from_numpy((half >= t).astype(np.float64) * (65536 / (65536 - t)))


def activation(g: torch.Tensor, name: str) -> tuple[torch.Tensor, torch.Tensor]:
    """act(g) and act'(g) in float64."""
    if name == "gelu":
        cdf = 0.5 * torch.special.erfc(-g * math.sqrt(0.5))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s + g * s * (1 - s)
    a = math.sqrt(2 / math.pi)
    t = torch.tanh(a * (g + 0.044715 * g**3))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * a * (1 + 3 * 0.044715 * g * g)


def _gamma(n: int) -> float:
    return (6 * n + 16) * 2.0**-24


class _Rounding:
    def __init__(self, dtype: torch.dtype):
        info = torch.finfo(dtype)
        self.u = info.eps / 2
        self.least = info.smallest_normal * info.eps / 2  # half the smallest subnormal

    def __call__(self, value: torch.Tensor, bound: torch.Tensor) -> torch.Tensor:
        """The bound after a rounding of something within `bound` of `value`."""
        return bound + self.u * (value.abs() + bound) + self.least


def _products(dz, e_dz, x, w, rnd):
    """dx, dweight, dbias and their bounds from dz, each element of which is known to within e_dz."""
    adz = dz.abs() + e_dz
    dx, dw, db = dz @ w, dz.t() @ x, dz.sum(0)
    e_dx = e_dz @ w.abs() + _gamma(dz.shape[1]) * (adz @ w.abs())
    e_dw = e_dz.t() @ x.abs() + _gamma(dz.shape[0]) * (adz.t() @ x.abs())
    e_db = e_dz.sum(0) + _gamma(dz.shape[0]) * adz.sum(0)
    return [(v, rnd(v, e)) for v, e in ((dx, e_dx), (dw, e_dw), (db, e_db))]


def linear(x, w, b, residual, dy, *, p=0.0, seed=0, offset=0, dtype=torch.float32):
    """[(value, bound)] of y, and where dy is given dx, dweight, dbias."""
    x, w, b, residual, dy = (None if t is None else t.detach().cpu().double() for t in (x, w, b, residual, dy))
    rnd = _Rounding(dtype)
    k = keep_scale(x.shape[0], w.shape[0], p, seed, offset)
    z = x @ w.t()
    e = _gamma(x.shape[1]) * (x.abs() @ w.abs().t())
    if b is not None:
        z = z + b
        e = e + 2.0**-23 * (z.abs() + e + b.abs())
    y, e = z * k, e * k * (1 + 2.0**-22) + 2.0**-22 * (z * k).abs()
    if residual is not None:
        y = y + residual
        e = e + 2.0**-23 * (y.abs() + e)
    out = [(y, rnd(y, e))]
    if dy is not None:
        dz = dy * k
        exact = p == 0
        e_dz = torch.zeros_like(dz) if exact else rnd(dz, 2.0**-22 * dz.abs()) * (k != 0)
        out += _products(dz, e_dz, x, w, rnd)
    return out


def gated(x, w, b, dy, *, act="gelu", p=0.0, seed=0, offset=0, dtype=torch.float32):
    """[(value, bound)] of h, and where dy is given dx, dweight, dbias."""
    x, w, b, dy = (None if t is None else t.detach().cpu().double() for t in (x, w, b, dy))
    rnd = _Rounding(dtype)
    F = w.shape[0] // 2
    k = keep_scale(x.shape[0], F, p, seed, offset)
    z = x @ w.t()
    e = _gamma(x.shape[1]) * (x.abs() @ w.abs().t())
    if b is not None:
        z = z + b
        e = e + 2.0**-23 * (z.abs() + e + b.abs())
    v, g, ev, eg = z[:, :F], z[:, F:], e[:, :F], e[:, F:]
    a, slope = activation(g, act)
    fn = 2.0**-20 * (1 + g.abs())
    ea = 1.2 * eg + fn
    h = v * a * k
    eh = k * (a.abs() * ev + v.abs() * ea + ev * ea) + 2.0**-21 * h.abs()
    out = [(h, rnd(h, eh))]
    if dy is not None:
        ev, eg = rnd(v, ev), rnd(g, eg)  # as the forward keeps them
        ea, es = 1.2 * eg + fn, 1.2 * eg + fn
        d = dy * k
        dv, dg = d * a, d * v * slope
        e_dv = rnd(dv, d.abs() * ea + 2.0**-21 * dv.abs())
        e_dg = rnd(dg, d.abs() * (slope.abs() * ev + v.abs() * es + ev * es) + 2.0**-21 * dg.abs())
        out += _products(torch.cat((dv, dg), 1), torch.cat((e_dv, e_dg), 1), x, w, rnd)
    return out


def dropout_add(x, residual, *, p, seed, offset, dtype):
    """(value, bound) of residual + dropout(x) for matrices."""
    x = x.detach().cpu().double()
    k = keep_scale(*x.shape, p, seed, offset)
    y = torch.where(k != 0, x * k, torch.zeros_like(x))
    e = 2.0**-22 * y.abs()
    if residual is not None:
        y = y + residual.detach().cpu().double()
        e = e + 2.0**-23 * (y.abs() + e)
    return y, _Rounding(dtype)(y, e)
