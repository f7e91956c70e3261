"""How near the feed-forward operators come to their definitions as a whole, and over their types' whole range.

Beside the element-by-element bounds of tests/test_feedforward.py, whose worst cases are wide: the root of the
mean square of an output's error, against that of the output, with limits that follow from how independent
roundings add up.
"""

from __future__ import annotations

import math

import pytest
import torch

from guass_amd import feedforward as ff
from oracle import feedforward_oracle as fo

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
ids = lambda v: str(v).replace("torch.", "") if isinstance(v, torch.dtype) else None  # noqa: E731
RNG = dict(seed=11, offset=5)


def _say(*what):
    print("[gpu-test] feedforward precision", *what, flush=True)


def _rand(device, *shape, dtype, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dtype).to(device)


def _case(device, kind, rows, d, n, dtype, seed):
    w_rows = 2 * n if kind == "gated" else n
    return {"x": _rand(device, rows, d, dtype=dtype, seed=seed), "w": _rand(device, w_rows, d, dtype=dtype, seed=seed + 1, std=d**-0.5),
            "b": _rand(device, w_rows, dtype=dtype, seed=seed + 2, std=0.3), "dy": _rand(device, rows, n, dtype=dtype, seed=seed + 3, std=0.5)}


def _exact(kind, t, act, p):
    """y, dx, dweight and dbias in 64 bits, where the tensors are."""
    x, w, b, dy = (None if t[k] is None else t[k].double() for k in ("x", "w", "b", "dy"))
    n = dy.shape[1]
    keep = fo.keep_scale(*dy.shape, p, **RNG).to(x.device)
    z = x @ w.t()
    if b is not None:
        z = z + b
    if kind == "linear":
        y, dz = z * keep, dy * keep
    else:
        a, slope = fo.activation(z[:, n:], act)
        y = z[:, :n] * a * keep
        dz = torch.cat((dy * keep * a, dy * keep * z[:, :n] * slope), dim=1)
    return [y, dz @ w, dz.t() @ x] + ([] if b is None else [dz.sum(0)])


def _run(kind, t, act, p):
    leaves = [t[k].detach().requires_grad_(True) for k in ("x", "w", "b") if t[k] is not None]
    if kind == "gated":
        y = ff.gated_linear(*leaves, activation=act, p=p, **RNG)
    else:
        y = ff.linear_dropout_add(*leaves, p=p, **RNG)
    return [y.detach(), *torch.autograd.grad(y, leaves, t["dy"])]


def _rms(got, want):
    return float((got.double() - want).norm() / want.norm())


def _limits(kind, dtype, want, inner):
    """For y, dx, dweight and dbias, each a sum of inner[i] terms.

    32 bits: six products for each term leave out at most 8 2^-24 of it, and 6 n additions each round by 1/sqrt(12) of a unit of
    the sum so far, which is at most 2^-23 of it and whose mean square is half the final one's: sqrt(6 n / 24) 2^-23.
    16 bits: what rounding the right result once does to it (measured on the result itself), with a tenth on top, which is
    more than what 32-bit sums add; for a gated product's dx and dweight twice that rounding, independently, because dz is
    rounded to the tensors' type too.
    """
    out = []
    for i, (v, n) in enumerate(zip(want, inner)):
        if dtype == torch.float32:
            out.append((8 + math.sqrt(n)) * 2.0**-24)
        else:
            out.append(1.1 * _rms(v.to(dtype), v) * (math.sqrt(2) if kind == "gated" and i in (1, 2) else 1))
    return out


def _check(device, kind, rows, d, n, dtype, act="gelu", p=0.0, seed=200, change=None):
    t = _case(device, kind, rows, d, n, dtype, seed)
    if change is not None:
        t = change(t)
    want = _exact(kind, t, act, p)
    inner = (d, t["w"].shape[0], rows, rows)
    for name, got, v, limit in zip(("y", "dx", "dweight", "dbias"), _run(kind, t, act, p), want, _limits(kind, dtype, want, inner)):
        off = _rms(got, v)
        _say(kind, (rows, d, n), ids(dtype), act, p, name, f"{off:.3e} of {limit:.3e}")
        assert off <= limit, f"{name}: {off:.3e}, limit {limit:.3e}"


# few rows, splits along k, odd sizes
SIZES = [(48, 320, 264), (300, 640, 1000), (1025, 2560, 640), (4089, 331, 2037), (8100, 328, 1279), (4089, 2037, 331)]


@pytest.mark.gpu
@pytest.mark.parametrize("p", [0.0, 0.1])
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_linear_loses_its_outputs_rounding_only(device, size, dtype, p):
    _check(device, "linear", *size, dtype, p=p)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [40, 300])
def test_linear_gradients_beyond_float16(device, rows):
    """What is kept times 1 / (1 - p) passes float16's largest number, or falls among its smallest; the gradients do
    neither."""
    large = lambda t: dict(t, b=None, dy=(t["dy"] * 16000).clamp(-60000, 60000), w=t["w"] * 2.0**-8, x=t["x"] * 2.0**-8)  # noqa: E731
    _check(device, "linear", rows, 72, 104, torch.float16, p=0.9, change=large)
    small = lambda t: dict(t, b=None, dy=t["dy"] * 2.0**-18, w=t["w"] * 2.0**5, x=t["x"] * 2.0**5)  # noqa: E731
    _check(device, "linear", rows, 72, 104, torch.float16, p=0.1, change=small)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("act", ff.ACTIVATIONS)
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_gated_loses_its_outputs_rounding_and_the_gradients(device, size, act, dtype):
    _check(device, "gated", *size, dtype, act=act, p=0.1)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [40, 300])
def test_gated_gradients_beyond_float16(device, rows):
    """dy times the value passes float16's largest number (values near 1000), or falls among its smallest; dx and dweight do
    neither.  A NaN and an infinity in one row of dy leave the others' dx as it was."""
    def large(t):
        n = t["dy"].shape[1]
        b = t["b"].clone()
        b[:n] = 1000.0
        return dict(t, b=b, dy=t["dy"] * 300, w=t["w"] * 2.0**-8, x=t["x"] * 2.0**-8)

    t = large(_case(device, "gated", rows, 72, 104, torch.float16, 200))
    n = t["dy"].shape[1]
    want = _exact("gated", t, "gelu", 0.1)
    assert float((t["dy"].double() * 1000).abs().max()) > 65504
    got = _run("gated", t, "gelu", 0.1)
    limits = _limits("gated", torch.float16, want, (72, 2 * n, rows, rows))
    for i in range(3):  # dbias passes the range by itself
        assert _rms(got[i], want[i]) <= limits[i]

    small = lambda t: dict(t, b=t["b"] * 0, dy=t["dy"] * 2.0**-16, w=t["w"] * 2.0**2, x=t["x"] * 2.0**-5)  # noqa: E731
    t = small(_case(device, "gated", rows, 72, 104, torch.float16, 200))
    want = _exact("gated", t, "gelu", 0.1)
    got = _run("gated", t, "gelu", 0.1)
    limits = _limits("gated", torch.float16, want, (72, 2 * n, rows, rows))
    for i in range(4):
        assert _rms(got[i], want[i]) <= limits[i]

    t = large(_case(device, "gated", rows, 72, 104, torch.float16, 200))
    t["dy"][3, 5], t["dy"][7, 6] = math.nan, math.inf
    dx = _run("gated", t, "gelu", 0.0)[1]
    fine = torch.isfinite(dx).all(dim=1).cpu()
    assert not fine[3] and not fine[7] and int(fine.sum()) == rows - 2


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [4, 200])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=ids)
def test_dropped_places_give_no_gradient_whatever_they_were(device, dtype, rows):
    """A place whose value and gate overflow to infinities, dropped: its output is 0, and so are its gradients."""
    d, n = 8, 16
    keep = fo.keep_scale(rows, n, 0.5, **RNG) != 0
    row, col = (int(v) for v in (~keep).nonzero()[0])
    x, w = _rand(device, rows, d, dtype=dtype, seed=1), _rand(device, 2 * n, d, dtype=dtype, seed=2)
    x[:, 0] = 0
    w[:, 0] = 0
    x[row, 0], w[col, 0], w[n + col, 0] = 1e20, 1e20, 1e20
    t = {"x": x, "w": w, "b": torch.zeros(2 * n, dtype=dtype, device=device), "dy": torch.ones(rows, n, dtype=dtype, device=device)}
    calm = dict(t, w=w.clone())
    calm["w"][col, 0] = calm["w"][n + col, 0] = 0
    got, want = _run("gated", t, "gelu", 0.5), _run("gated", calm, "gelu", 0.5)
    got[1], want[1] = got[1].clone(), want[1].clone()
    assert bool((got[1][row, 0] == 0).all())
    got[1][:, 0] = want[1][:, 0] = 0  # the other rows' dx there goes by the weight that was taken out
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("rows", [40, 200])
def test_infinities_come_out_as_the_sums_have_them(device, dtype, rows):
    """An infinity in x, in dy or in the weight makes infinities of its products' signs, and a NaN where it meets a zero,
    in every type and at every number of rows.  The numbers that it meets have few bits (0.5, -1) and many (0.1)."""
    d, n = 96, 64
    t = _case(device, "linear", rows, d, n, dtype, 210)
    t["x"][3, 17], t["x"][4, 17] = math.inf, -math.inf
    t["w"][5, 17], t["w"][6, 17], t["w"][7, 17], t["w"][8, 17], t["w"][9, 18] = 0.0, 0.5, -1.0, 0.1, -math.inf
    t["x"][10, 18], t["x"][11, 18], t["x"][12, 18] = 1.0, 0.0, -0.25
    t["dy"][3, 20], t["dy"][4, 21], t["dy"][14, 9], t["dy"][15, 9] = 1.0, 0.0, 0.0, 2.0
    t["dy"][16, 30] = math.inf
    t["x"][16, 40], t["w"][30, 40] = -0.5, 2.0
    for name, got, want in zip(("y", "dx", "dweight", "dbias"), _run("linear", t, None, 0.0), _exact("linear", t, None, 0.0)):
        assert bool(torch.isinf(want).any()), name
        assert torch.equal(torch.isnan(got), torch.isnan(want)), name
        assert torch.equal(torch.isinf(got), torch.isinf(want)), name
        assert torch.equal(torch.sign(got[torch.isinf(want)]).double(), torch.sign(want[torch.isinf(want)])), name


# ------------------------------------------------------------------------------ what the limits tell apart, on the CPU


def _planes(t):
    """Three bfloat16 planes of float32 numbers, by truncation, in 64 bits."""
    out, left = [], t.clone()
    for _ in range(3):
        top = (left.view(torch.int32) & -65536).view(torch.float32)
        out.append(top.double())
        left = left - top
    return out


@pytest.mark.parametrize("inner", [40, 320, 1279, 4089])
def test_limits_see_a_lost_plane(inner):
    """Six products of planes keep the float32 limit; without the three small ones, or without either operand's third plane,
    the result lies beyond it."""
    g = torch.Generator().manual_seed(inner)
    a, b = torch.randn(64, inner, generator=g), torch.randn(96, inner, generator=g)
    want = a.double() @ b.double().t()
    p, q = _planes(a), _planes(b)
    limit = _limits("linear", torch.float32, [want], (inner,))[0]
    terms = {(i, j): p[i] @ q[j].t() for i in range(3) for j in range(3) if i + j <= 2}
    assert _rms(sum(terms.values()), want) <= limit
    for lost in ([(2, 0), (0, 2), (1, 1)], [(2, 0)], [(0, 2)]):
        assert _rms(sum(v for k, v in terms.items() if k not in lost), want) > limit, lost


@pytest.mark.parametrize("act", ff.ACTIVATIONS)
@pytest.mark.parametrize("dtype,bits", [(torch.bfloat16, 12), (torch.float16, 16)], ids=str)
def test_limits_see_value_and_gate_lose_their_low_bits(dtype, bits, act):
    """Value and gate in the bits that are kept meet a gated product's limits for dx and dweight; rounded to the tensors'
    own type they do not."""
    t = _case("cpu", "gated", 300, 72, 104, dtype, 220)
    want = _exact("gated", t, act, 0.0)
    limits = _limits("gated", dtype, want, (72, 208, 300, 300))

    def gradients(keep):
        x, w, b, dy = (t[k].double() for k in ("x", "w", "b", "dy"))
        z = keep(x @ w.t() + b)
        a, slope = fo.activation(z[:, 104:], act)
        dz = torch.cat((dy * a, dy * z[:, :104] * slope), dim=1).to(dtype).double()
        return [(dz @ w).to(dtype), (dz.t() @ x).to(dtype)]

    def short(z):  # to `bits` significant ones
        m, e = torch.frexp(z)
        return torch.ldexp((m * 2**bits).round() / 2**bits, e)

    assert all(_rms(g, v) <= limit for g, v, limit in zip(gradients(short), want[1:3], limits[1:3]))
    assert any(_rms(g, v) > limit for g, v, limit in zip(gradients(lambda z: z.to(dtype).double()), want[1:3], limits[1:3]))


# ------------------------------------------------------------------------------ large tiles; dy as dz


# sizes at which the products take each of the large tiles, in each operand layout: odd ones, and ones that are read in place
LARGE = [("gated", 4089, 331, 2037), ("linear", 4089, 331, 4075), ("linear", 8100, 328, 1279), ("linear", 4089, 4075, 331),
         ("linear", 331, 4075, 4089), ("gated", 1030, 1031, 2090), ("gated", 4000, 2201, 600), ("linear", 331, 1279, 8100)]
WHOLE = [("linear", 8104, 328, 1280), ("linear", 4088, 4072, 328), ("linear", 328, 4072, 4088), ("linear", 328, 1280, 8104)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("kind,rows,d,n", LARGE)
def test_large_tiles_keep_the_limits(device, kind, rows, d, n, dtype):
    _check(device, kind, rows, d, n, dtype, p=0.1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES[1:], ids=ids)
@pytest.mark.parametrize("kind,rows,d,n", WHOLE)
def test_large_tiles_of_dy_itself(device, kind, rows, d, n, dtype):
    _check(device, kind, rows, d, n, dtype, p=0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("rows", [1, 5, 40, 64, 65, 300])
@pytest.mark.parametrize("n", [64, 72, 61])
def test_nothing_dropped_takes_dy_as_it_lies(device, rows, n, dtype):
    """Without dropout the products of a linear backward read dy in place where they can: a contiguous one, rows of a larger
    matrix (aligned and not), an odd base, a broadcast one, a transposed one.  Each gives the contiguous one's gradients to
    the bit, element by element within the oracle's bounds, with every gradient or the bias's alone."""
    d = 56
    t = _case(device, "linear", rows, d, n, dtype, 230)
    leaves = [t[k].requires_grad_(True) for k in ("x", "w", "b")]
    y = ff.linear_dropout_add(*leaves)

    def layouts(dy):
        yield "contiguous", dy
        for left, right in ((8, 8), (8, 3), (1, 2)):
            big = torch.full((rows + 1, left + n + right), math.nan, dtype=dtype, device=device)
            big[:-1, left:left + n] = dy
            yield f"rows {left} {right}", big[:-1, left:left + n]
        yield "odd base", torch.empty(rows * n + 1, dtype=dtype, device=device)[1:].view(rows, n).copy_(dy)
        yield "transposed", dy.t().contiguous().t()

    for dy in (t["dy"], torch.full((1, 1), 0.75, dtype=dtype, device=device).expand(rows, n)):
        want = fo.linear(t["x"], t["w"], t["b"], None, dy, dtype=dtype)[1:]
        first = None
        for name, view in layouts(dy.contiguous()):
            _say("dy as it lies", rows, n, ids(dtype), name)
            got = torch.autograd.grad(y, leaves, view, retain_graph=True)
            for g, (value, bound) in zip(got, want):
                assert bool(((g.cpu().double() - value).abs() <= bound).all()), name
            first = first or got
            assert all(torch.equal(a, b) for a, b in zip(got, first)), name
            alone, = torch.autograd.grad(y, leaves[2], view, retain_graph=True)
            assert torch.equal(alone, first[2]), name
        got = torch.autograd.grad(y, leaves, dy, retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(got, first))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [3, 200])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=ids)
@pytest.mark.parametrize("act", ff.ACTIVATIONS)
def test_gates_far_past_where_the_activations_are_flat(device, act, dtype, rows):
    """Gates whose squares overflow: the activation is the gate or 0 there, its slope 1 or 0."""
    gates = [1e15, -1e15, 1e19, -1e19, 1e20, -1e20, 1e30, -1e30]
    n = len(gates)
    x = torch.zeros(rows, 8)
    x[:, :2] = 1.0
    w = torch.zeros(2 * n, 8)
    w[:n, 0] = 1.0
    w[n:, 1] = torch.tensor(gates)
    t = {"x": x.to(dtype).to(device), "w": w.to(dtype).to(device), "b": None, "dy": torch.ones(rows, n, dtype=dtype, device=device)}
    want = _exact("gated", t, act, 0.0)
    for got, v in zip(_run("gated", t, act, 0.0), want):
        assert bool(((got.double() - v).abs() <= 2.0**-7 * v.abs() + 1e-30).all())
