"""Weights in 4 bits (guass_amd/quantized.py) against their definitions in 64 bits.

Codes and scales have to be equal to the oracle's (oracle/block_oracle.py); products are held to the bounds of
oracle/feedforward_oracle.py with the weight's exact values.  No counterpart in the reference.
"""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from guass_amd import _native as N
from guass_amd import quantized as q4
from guass_amd.feedforward import ACTIVATIONS
from oracle import block_oracle as bo
from oracle import feedforward_oracle as fo

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
ids = lambda v: str(v).replace("torch.", "") if isinstance(v, torch.dtype) else None  # noqa: E731


def _say(*what):
    print("[gpu-test] quantized", *what, flush=True)


def _rand(device, *shape, dtype, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dtype).to(device)


def _close(got, want, what):
    value, bound = want
    got = got.detach().cpu().double()
    assert got.shape == value.shape, f"{what}: {got.shape} for {value.shape}"
    off = (got - value).abs()
    assert bool((off <= bound).all()), f"{what}: {float((off - bound).max()):.3e} past its bound, off {float(off.max()):.3e}"


def _weight(device, rows, cols, seed=0):
    """A quantised weight made by the oracle, and its exact values."""
    g = torch.Generator().manual_seed(seed)
    codes, scales = bo.quantize(torch.randn(rows, cols, generator=g) * cols**-0.5)
    return q4.QuantizedWeight(codes.to(device), scales.to(device), cols), bo.dequantize(codes, scales, cols)


# ------------------------------------------------------------------------------------ the CPU


def test_oracle_known_values():
    """Every magnitude, every border between two with what lies on either side, the scales' steps; a short last group."""
    up = 1 + 2.0**-20
    row = [0.0, 0.25, 0.25 * up, 0.75 / up, 0.75, 1.25, 1.25 * up, 1.75 / up, 1.75, 2.5, 2.5 * up, 3.5 / up, 3.5, 5.0, 5.0 * up, 6.0, 7.0, -0.25, -0.5, -6.5]
    want = [0.0, 0.0, 0.5, 0.5, 1.0, 1.0, 1.5, 1.5, 2.0, 2.0, 3.0, 3.0, 4.0, 4.0, 6.0, 6.0, 6.0, 0.0, -0.5, -6.0]
    codes, scales = bo.quantize(torch.tensor([row + [0.0] * 13, [7.0 * up] + [0.0] * 32, [1e-45] + [0.0] * 32]))
    assert scales.tolist() == [[127, 2], [128, 2], [2, 2]] and codes.shape == (3, 32)
    got = bo.dequantize(codes, scales, 33)
    assert got[0, :20].tolist() == want and got[1, 0] == 8.0 and got[2, 0] == 0.0
    bad = torch.zeros(3, 64)
    bad[0, 40], bad[1, 3], bad[2, 63] = math.nan, math.inf, -math.inf
    codes, scales = bo.quantize(bad)
    assert scales.tolist() == [[2, 255], [255, 2], [2, 255]]
    assert torch.isnan(bo.dequantize(codes, scales, 64)).sum() == 96


def test_refusals_without_a_gpu():
    w = q4.QuantizedWeight(torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.uint8), 8)
    assert w.shape == (4, 8) and w.device.type == "cpu"
    for call, msg in ((lambda: q4.quantize(torch.zeros(2, 8)), "weight must be a CUDA tensor"), (lambda: w.dequantize(), "codes must be a CUDA tensor"),
                      (lambda: q4.quantized_linear(torch.zeros(2, 8), w), "x must be a CUDA tensor"),
                      (lambda: q4.quantized_gated_linear(torch.zeros(2, 8), w), "x must be a CUDA tensor")):
        with pytest.raises(RuntimeError, match=msg):
            call()
    with pytest.raises(ValueError, match="activation must be one of"):
        q4.quantized_gated_linear(torch.zeros(2, 8), w, activation="relu")
    with pytest.raises(TypeError, match="weight must be a QuantizedWeight"):
        q4.quantized_linear(torch.zeros(2, 8), torch.zeros(4, 8))
    with pytest.raises(TypeError, match="x must be a tensor"):
        q4.quantized_linear([1.0], w)
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8)  # noqa: E731
    for codes, scales, cols, msg in ((u8(4, 16), u8(4, 1), 33, "has codes"), (u8(4, 16), u8(4, 2), 32, "has codes"), (u8(4, 16), u8(3, 1), 32, "has codes"),
                                     (u8(64), u8(4, 1), 32, "has codes"), (u8(4, 16), u8(4, 1), 0, "must be positive"),
                                     (torch.zeros(4, 16), u8(4, 1), 32, "codes must be uint8"), (u8(4, 16), torch.zeros(4, 1), 32, "scales must be uint8")):
        with pytest.raises(ValueError, match=msg):
            q4.QuantizedWeight(codes, scales, cols)
    with pytest.raises(TypeError, match="codes must be a tensor"):
        q4.QuantizedWeight([0], u8(4, 1), 32)


def _args(**kw):
    a = N.GfQ4Args()
    base = dict(dtype=1, activation=1, rows=4, in_features=40, out_features=8, x=4096, ldx=40, codes=4096, scales=4096, bias=4096, y=4096, dy=4096, lddy=8,
                saved=4096, dx=4096)
    for k, v in {**base, **kw}.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=3), "unknown dtype"), (dict(activation=4), "unknown activation"), (dict(rows=-1), "rows must not be negative"),
    (dict(in_features=0), "must be positive"), (dict(out_features=0), "must be positive"), (dict(rows=2**31), "too large"),
    (dict(in_features=2**30, out_features=2**29), "too large"), (dict(codes=None), "codes and scales must not be NULL"),
    (dict(scales=None), "codes and scales must not be NULL"), (dict(codes=4104), "codes must be 16-byte aligned"), (dict(ldr=2**62), "row stride too large"),
])
@pytest.mark.parametrize("phase", ["forward", "backward"])
def test_abi_refuses_before_device_work(kw, msg, phase):
    lib = N.lib()
    rc = getattr(lib, f"gf_q4_{phase}")(ctypes.byref(_args(**kw)), 4096, 2**40, None)
    assert rc == 1 and msg in lib.gf_last_error().decode(), lib.gf_last_error()


def test_abi_refuses_by_phase():
    lib = N.lib()
    err = lambda: lib.gf_last_error().decode()  # noqa: E731
    fwd = lambda **kw: lib.gf_q4_forward(ctypes.byref(_args(**kw)), None, 0, None)  # noqa: E731
    assert lib.gf_q4_forward(None, None, 0, None) == 1 and lib.gf_q4_saved_bytes(None) == 0 and lib.gf_q4_workspace_bytes(None, 0) == 0
    assert fwd(x=None) == 1 and "x must not be NULL" in err()
    assert fwd(ldx=39) == 1 and "row stride 39" in err()
    assert fwd(x=4097) == 1 and "x is not aligned" in err()
    assert fwd(bias=4097) == 1 and "bias is not aligned" in err()
    assert fwd(y=None) == 1 and "y must not be NULL" in err()
    assert fwd(residual=4096, ldr=8) == 1 and "takes no residual" in err()
    assert fwd(activation=0, residual=4096, ldr=7) == 1 and "residual: row stride 7" in err()
    assert fwd() == 2 and "workspace" in err()  # it saves, so it goes through the weight's values
    assert fwd(rows=129, saved=None) == 2
    assert fwd(rows=0, x=None) == 0
    back = lambda **kw: lib.gf_q4_backward(ctypes.byref(_args(**kw)), 4096, 2**40, None)  # noqa: E731
    assert back(rows=0) == 1 and "needs rows" in err()
    assert back(dy=None) == 1 and "dy must not be NULL" in err()
    assert back(saved=None) == 1 and "saved must not be NULL" in err()
    assert back(lddy=7) == 1 and "dy: row stride 7" in err()
    for call in (lambda d, r, c, p: lib.gf_q4_quantize(d, r, c, p, 40, 4096, 4096, None), lambda d, r, c, p: lib.gf_q4_dequantize(d, r, c, 4096, 4096, p, None)):
        assert call(3, 4, 40, 4096) == 1 and "unknown dtype" in err()
        assert call(0, -1, 40, 4096) == 1 and call(0, 4, 0, 4096) == 1 and call(0, 2**31, 40, 4096) == 1 and call(0, 2**31 - 1, 2**29, 4096) == 1
        assert call(0, 4, 40, None) == 1 and "weight must not be NULL" in err()
        assert call(0, 4, 40, 4098) == 1 and "weight is not aligned" in err()
        assert call(0, 0, 40, None) == 0
    assert lib.gf_q4_quantize(0, 4, 40, 4096, 39, 4096, 4096, None) == 1 and "row stride 39" in err()
    assert lib.gf_q4_quantize(0, 4, 40, 4096, 40, None, 4096, None) == 1 and lib.gf_q4_quantize(0, 4, 40, 4096, 40, 4100, 4096, None) == 1


@pytest.mark.parametrize("dtype,size", [(0, 4), (1, 2), (2, 2)])
def test_abi_workspaces(dtype, size):
    """None for few rows that save nothing; else the weight's values at least, without overflow up to the limits."""
    lib = N.lib()
    ws = lambda back, **kw: lib.gf_q4_workspace_bytes(ctypes.byref(_args(dtype=dtype, **kw)), back)  # noqa: E731
    assert ws(0, saved=None) == 0 and ws(0, saved=None, rows=128) == 0 and ws(0, saved=None, rows=129) > 0
    for rows, d, n in ((1, 40, 8), (64, 8, 8), (65, 8, 8), (129, 8, 8), (2**31 - 1, 8, 2**10), (1, 2**21, 2**20), (2**20, 2**21, 2**19)):
        for back in (0, 1):
            got = ws(back, rows=rows, in_features=d, out_features=n, ldx=d, lddy=n)
            assert 2 * n * d * size <= got < 2**62
    a, f = _args(dtype=dtype), N.GfFfArgs()
    f.dtype, f.activation, f.rows, f.in_features, f.out_features = dtype, 1, 4, 40, 8
    assert lib.gf_q4_saved_bytes(ctypes.byref(a)) == lib.gf_ff_saved_bytes(ctypes.byref(f)) > 0


# ------------------------------------------------------------------------------------ the GPU


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 32), (3, 31), (2, 33), (5, 64), (7, 129), (64, 1280), (33, 333), (300, 95), (1000, 8)])
def test_quantize(device, rows, cols, dtype):
    """Codes and scales as the oracle has them, and back; rows of a larger matrix and a transposed one too."""
    _say("quantize", rows, cols, dtype)
    w = _rand(device, rows, cols, dtype=dtype, seed=rows + cols, std=0.05)
    codes, scales = bo.quantize(w)
    big = torch.full((rows + 1, cols + 5), math.nan, dtype=dtype, device=device)
    big[:-1, 3:3 + cols] = w
    for source in (w, big[:-1, 3:3 + cols], w.t().contiguous().t(), w.clone().requires_grad_(True)):
        got = q4.quantize(source)
        assert got.shape == w.shape and torch.equal(got.codes.cpu(), codes) and torch.equal(got.scales.cpu(), scales)
    values = bo.dequantize(codes, scales, cols)
    for out in DTYPES:
        assert torch.equal(got.dequantize(out).cpu(), values.to(out))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
def test_quantize_borders(device, dtype):
    """Every border between two values and its neighbours, at every scale of the type; zeros, subnormals, the largest numbers."""
    _say("borders", dtype)
    info = torch.finfo(dtype)
    points = torch.tensor([0.25, 0.5, 0.75, 1.0, 1.25, 1.5, 1.75, 2.0, 2.5, 3.0, 3.5, 4.0, 5.0, 6.0, 6.5, 7.0], dtype=torch.float64)
    near = torch.cat([points, points * (1 + info.eps), points * (1 - info.eps / 2)])  # 48 numbers of the type
    rows = []
    lo, hi = (-24, 13) if dtype == torch.float16 else (-140, 125)
    for e in range(lo, hi):
        for top in (6.0, 7.0, 7.0 * (1 + info.eps)):
            for part in (near[:31], near[17:]):
                rows.append(torch.cat([torch.tensor([top], dtype=torch.float64), part * torch.where(torch.arange(31) % 2 == 0, 1.0, -1.0)]) * 2.0**e)
    rows += [torch.zeros(32, dtype=torch.float64), torch.full((32,), float(info.max)), torch.full((32,), -float(info.tiny))]
    w = torch.stack([r.double() for r in rows]).to(dtype)
    codes, scales = bo.quantize(w)
    got = q4.quantize(w.to(device))
    assert torch.equal(got.scales.cpu(), scales)
    assert torch.equal(got.codes.cpu(), codes)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_bad_weight_takes_its_group(device, bad):
    w = _rand(device, 4, 100, dtype=torch.float32, seed=1)
    w[2, 70] = bad
    got = q4.quantize(w)
    codes, scales = bo.quantize(w)
    assert torch.equal(got.codes.cpu(), codes) and torch.equal(got.scales.cpu(), scales)
    nan = torch.isnan(got.dequantize())
    assert bool(nan[2, 64:96].all()) and int(nan.sum()) == 32
    for rows in (3, 70):
        y = q4.quantized_linear(_rand(device, rows, 100, dtype=torch.bfloat16, seed=2), got)
        assert bool(torch.isnan(y[:, 2]).all()) and int(torch.isnan(y).sum()) == rows


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
def test_every_code_and_scale(device, dtype):
    """All 16 codes at all 256 scales: the values, and a product that picks out each (as what dequantize gives)."""
    _say("every code", dtype)
    codes = torch.tensor([[2 * i | (2 * i + 1) << 4 for i in range(8)] * 2], dtype=torch.uint8).expand(256, 16).contiguous()
    scales = torch.arange(256, dtype=torch.uint8)[:, None].contiguous()
    w = q4.QuantizedWeight(codes.to(device), scales.to(device), 32)
    values = bo.dequantize(codes, scales, 32)
    got = w.dequantize(dtype).cpu()
    want = values.float().to(dtype)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))
    sane = slice(127 - 20, 127 + 10)  # scales whose values and sums every type holds
    eye = torch.eye(32, dtype=dtype, device=device)
    y = q4.quantized_linear(eye, w).cpu()
    assert torch.equal(y[:, sane], want[sane].t())
    assert bool(torch.isnan(y[:, 255]).all())
    if dtype == torch.float16:  # past the scales at which values are exact: as they are rounded to the type
        sane = slice(127 - 30, 127 + 14)
        assert torch.equal(y[:, sane], want[sane].t())


def _products(device, kind, rows, d, n, dtype, act="gelu", bias=True, residual=True, seed=0, x=None):
    """Forward without and with gradients, and the gradients, against the oracle."""
    w, values = _weight(device, 2 * n if kind == "gated" else n, d, seed=seed + 1)
    t = {"x": _rand(device, rows, d, dtype=dtype, seed=seed) if x is None else x,
         "b": _rand(device, w.shape[0], dtype=dtype, seed=seed + 2, std=0.3) if bias else None,
         "r": _rand(device, rows, n, dtype=dtype, seed=seed + 3) if residual and kind == "linear" else None}
    dy = _rand(device, rows, n, dtype=dtype, seed=seed + 4, std=0.5)
    what = f"{kind} {rows} x {d} -> {n}"

    def run(t):
        if kind == "gated":
            return q4.quantized_gated_linear(t["x"], w, t["b"], activation=act)
        return q4.quantized_linear(t["x"], w, t["b"], t["r"])

    if kind == "gated":
        want = fo.gated(t["x"], values, t["b"], dy, act=act, dtype=dtype)
    else:
        want = fo.linear(t["x"], values, t["b"], t["r"], dy, dtype=dtype)
    with torch.no_grad():
        _close(run(t), want[0], f"{what} y")
    leaves = {k: v.detach().requires_grad_(True) for k, v in t.items() if v is not None}
    y = run({**t, **leaves})
    _close(y, want[0], f"{what} y with gradients")
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))
    _close(grads["x"], want[1], f"{what} dx")
    if bias:
        _close(grads["b"], want[3], f"{what} dbias")
    if "r" in grads:
        assert torch.equal(grads["r"], dy)


# one token; tiny and odd; groups and tiles by one each way; a long contraction; more rows than go by the codes
SHAPES = [(1, 64, 64), (1, 1, 1), (2, 3, 5), (5, 33, 7), (16, 32, 16), (17, 31, 17), (33, 320, 96), (48, 129, 15), (64, 127, 33), (65, 128, 40), (127, 129, 50), (128, 40, 8200), (130, 200, 136),
          (3, 2056, 16), (1, 8200, 40), (40, 8, 1288), (300, 77, 100), (1, 40, 8200), (4, 129, 8192), (5, 1100, 8200), (20, 96, 8208), (33, 300, 8195)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("kind", ["linear", "gated"])
def test_products(device, kind, shape, dtype):
    _say("products", kind, shape, dtype)
    _products(device, kind, *shape, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("rows", [1, 2, 4, 5, 15, 16, 17, 32, 33, 63, 64, 65, 100, 128, 129])
def test_rows_at_a_wide_block(device, rows, dtype):
    _say("rows", rows, dtype)
    _products(device, "linear", rows, 1280, 320, dtype, seed=20)
    _products(device, "gated", rows, 320, 640, dtype, seed=30, bias=False)
    _products(device, "linear", rows, 5120, 80, dtype, seed=40, residual=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("act", ACTIVATIONS)
def test_activations(device, act, dtype):
    for rows in (3, 100):
        _products(device, "gated", rows, 96, 48, dtype, act=act, seed=50)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
def test_layouts(device, dtype):
    """Rows of larger matrices beside which NaN lies, odd bases, three dimensions; codes that are slices or not aligned."""
    _say("layouts", dtype)
    for rows in (5, 80, 150):
        d, n = 72, 40
        w, values = _weight(device, n, d, seed=3)
        x, b, r = (_rand(device, *s, dtype=dtype, seed=60 + i) for i, s in enumerate(((rows, d), (n,), (rows, n))))
        want = q4.quantized_linear(x, w, b, r)

        def wide(m, left, right):
            big = torch.full((m.shape[0] + 1, left + m.shape[1] + right), math.nan, dtype=dtype, device=device)
            big[:-1, left:left + m.shape[1]] = m
            return big[:-1, left:left + m.shape[1]]

        for left, right in ((8, 8), (1, 2), (16, 3)):
            got = q4.quantized_linear(wide(x, left, right), w, torch.stack((b, b), 1)[:, 0], wide(r, left, right))
            assert torch.equal(got, want) or (dtype == torch.float32 and torch.allclose(got, want, rtol=1e-5, atol=1e-5))
        assert torch.equal(q4.quantized_linear(x.t().contiguous().t(), w, b, r), want)
        assert torch.equal(q4.quantized_linear(x.view(1, rows, d), w, b, r.view(1, rows, n)), want[None])
        assert torch.equal(q4.quantized_linear(x[0], w, b, r[0]), q4.quantized_linear(x[:1], w, b, r[:1])[0])
        flat = torch.zeros(w.codes.numel() + 3, dtype=torch.uint8, device=device)
        odd = flat[3:].view_as(w.codes).copy_(w.codes)
        both = torch.cat((w.codes, w.codes), 1)[:, :w.codes.shape[1]]
        for codes in (odd, both):
            u = q4.QuantizedWeight(codes, torch.cat((w.scales, w.scales), 1)[:, :w.scales.shape[1]], d)
            assert torch.equal(q4.quantized_linear(x, u, b, r), want) and torch.equal(u.dequantize(), w.dequantize())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_bad_row_stays_in_its_row(device, bad, dtype):
    """Also behind an odd width, where the kernels read past nothing; an infinity times the code 0 is a NaN, times another infinite."""
    for rows, d in ((3, 50), (20, 50), (100, 50), (150, 50)):
        w, values = _weight(device, 24, d, seed=4)
        x = _rand(device, rows, d, dtype=dtype, seed=5)
        want = q4.quantized_linear(x, w)
        at = rows - 1 - rows // 3
        x[at, 49] = bad
        got = q4.quantized_linear(x, w)
        keep = torch.arange(rows, device=device) != at
        assert torch.equal(got[keep], want[keep])
        row = got[at].cpu()
        if math.isnan(bad):
            assert bool(torch.isnan(row).all())
        elif rows <= 128:
            exact = values[:, 49].float() * bad
            assert torch.equal(torch.isnan(row), torch.isnan(exact)) and torch.equal(row.float().nan_to_num(0.0, 1.0, -1.0), exact.nan_to_num(0.0, 1.0, -1.0))


@pytest.mark.gpu
def test_no_rows(device):
    w, _ = _weight(device, 16, 40)
    x, b = torch.zeros(0, 40, device=device, requires_grad=True), torch.zeros(16, device=device, requires_grad=True)
    for y in (q4.quantized_linear(x, w, b), q4.quantized_gated_linear(x, w, b)):
        assert y.shape[0] == 0
        dx, db = torch.autograd.grad(y.sum(), (x, b))
        assert dx.shape == x.shape and not bool(db.any())
    assert q4.quantize(torch.zeros(0, 40, device=device)).dequantize().shape == (0, 40)


@pytest.mark.gpu
def test_refusals(device):
    w, _ = _weight(device, 6, 40)
    x = torch.zeros(2, 40, device=device)
    m = lambda *s, **k: torch.zeros(*s, device=device, **k)  # noqa: E731
    odd, _ = _weight(device, 5, 40)
    for call, msg in (
        (lambda: q4.quantized_linear(m(2, 41), w), "x has 41 features"), (lambda: q4.quantized_linear(x.double(), w), "x must be float32"),
        (lambda: q4.quantized_linear(x, w.to("cpu")), "same device"), (lambda: q4.quantized_linear(x, w, m(5)), "bias must have shape"),
        (lambda: q4.quantized_linear(x, w, m(6, dtype=torch.bfloat16)), "bias must be torch.float32"), (lambda: q4.quantized_linear(x, w, None, m(2, 5)), "residual must"),
        (lambda: q4.quantized_gated_linear(x, odd), "even number of rows"), (lambda: q4.quantize(x.double()), "weight must be float32"),
        (lambda: w.dequantize(torch.float64), "dtype must be float32"), (lambda: q4.quantize(m(3, 0)), "not empty"),
        (lambda: q4.quantized_linear(m(()), w), "x must have shape"),
    ):
        with pytest.raises(RuntimeError, match=msg):
            call()
    with pytest.raises(ValueError, match="two dimensions"):
        q4.quantize(m(3))


@pytest.mark.gpu
def test_on_another_stream(device):
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        _products(device, "gated", 70, 96, 48, torch.bfloat16, seed=8)
        _products(device, "linear", 7, 96, 48, torch.bfloat16, seed=8)
    side.synchronize()


@pytest.mark.gpu
def test_captured_phases_replay(device):
    """Quantising, both ways of the forward and the backward in one graph, replayed with other inputs between eager work."""
    q4._ops()
    ops = torch.ops.guass_amd
    w = _rand(device, 96, 200, dtype=torch.float32, seed=1)
    few, many, dy = (_rand(device, *s, dtype=torch.bfloat16, seed=2 + i) for i, s in enumerate(((3, 200), (90, 200), (90, 48))))

    def step():
        codes, scales = ops.q4_quantize(w)
        y, saved = ops.q4_forward(many, codes, scales, None, None, 96, 200, 1, True)
        return [codes, scales, ops.q4_forward(few, codes, scales, None, None, 96, 200, 0, False)[0], y, *ops.q4_backward(dy, codes, scales, saved, 96, 200, 1, True, True)]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for k in range(4):
        for i, v in enumerate((w, few, many, dy)):
            v.copy_(_rand(device, *v.shape, dtype=v.dtype, seed=1000 * k + i))
        graph.replay()
        torch.cuda.synchronize()
        got = [c.clone() for c in captured]
        for a, b in zip(got, step()):
            assert torch.equal(a, b), f"replay {k}"


@pytest.mark.gpu
def test_more_elements_than_32_bits_count(device):
    """A weight of more than 2^31 elements: its last rows as by themselves."""
    _say("large")
    rows, cols = 2**31 // 16384 + 40, 16384
    w = torch.empty(rows, cols, dtype=torch.bfloat16, device=device)
    w[-19:] = _rand(device, 19, cols, dtype=torch.bfloat16, seed=1)
    w[:-19] = w[-1]
    big, last = q4.quantize(w), q4.quantize(w[-19:])
    del w
    values = big.dequantize(torch.bfloat16)
    assert torch.equal(values[-19:], last.dequantize(torch.bfloat16))
    for m in (1, 20):
        x = _rand(device, m, cols, dtype=torch.bfloat16, seed=2)
        y = q4.quantized_linear(x, big)[:, -19:].double()
        want = x.double() @ values[-19:].double().t()
        assert float((y - want).norm() / want.norm()) < 2.0**-8
