"""The norms around a block (guass_amd/norms.py) against their definitions in 64 bits.

The bounds are the oracle's (oracle/block_oracle.py): what 32-bit arithmetic and one rounding to the tensors' type may do,
element by element.  No counterpart in the reference.
"""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from guass_amd import _native as N
from guass_amd import norms
from oracle import block_oracle as bo

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
ids = lambda v: str(v).replace("torch.", "") if isinstance(v, torch.dtype) else None  # noqa: E731


def _say(*what):
    print("[gpu-test] norms", *what, flush=True)


def _rand(device, *shape, dtype, seed, std=1.0, mean=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std + mean).to(dtype).to(device)


def _tensors(device, shape, dtype, *, op, affine=True, per=None, seed=0):
    """The inputs of a call on x of `shape`; `per`: how many leading dimensions gate, scale and shift have of their own (None: a
    row's shape)."""
    cols = shape[-1]
    mod = (cols,) if per is None else (*shape[:per], *([1] * (len(shape) - 1 - per)), cols)
    t = {"x": _rand(device, *shape, dtype=dtype, seed=seed, mean=0.5)}
    if op != "norm":
        t["residual"] = _rand(device, *shape, dtype=dtype, seed=seed + 1, std=2.0)
        t["gate"] = _rand(device, *mod, dtype=dtype, seed=seed + 2, std=0.5)
        if affine:
            t["weight"], t["bias"] = (_rand(device, cols, dtype=dtype, seed=seed + 3 + i, std=0.3, mean=1.0 - i) for i in range(2))
    if op != "gate_add":
        t["scale"], t["shift"] = (_rand(device, *mod, dtype=dtype, seed=seed + 5 + i, std=0.3) for i in range(2))
        if affine:
            t["next_weight"], t["next_bias"] = (_rand(device, cols, dtype=dtype, seed=seed + 7 + i, std=0.3, mean=1.0 - i) for i in range(2))
    return t


def _call(op, t, kw):
    if op == "norm":
        return {"normed": norms.norm(t["x"], t.get("next_weight"), t.get("next_bias"), kind=kw["next_kind"], scale=t.get("scale"),
                                     shift=t.get("shift"), eps=kw.get("next_eps", 1e-5))}
    own = {k: kw[k] for k in ("kind", "residual_scale", "eps") if k in kw}
    own["gate"] = t["gate"] if t.get("gate") is not None else kw.get("gate", 1.0)
    if op == "gate_add":
        return {"stream": norms.gate_add(t["x"], t["residual"], t.get("weight"), t.get("bias"), **own)}
    stream, normed = norms.gate_add_norm(t["x"], t["residual"], t.get("weight"), t.get("bias"), t.get("next_weight"), t.get("next_bias"),
                                         next_kind=kw["next_kind"], scale=t.get("scale"), shift=t.get("shift"),
                                         next_eps=kw.get("next_eps", 1e-5), **own)
    return {"stream": stream, "normed": normed}


def _close(got, want, what):
    value, bound = want
    got = got.detach().cpu().double()
    assert got.shape == value.shape, f"{what}: {got.shape} for {value.shape}"
    off = (got - value).abs()
    assert bool((off <= bound).all()), f"{what}: {float((off - bound).max()):.3e} past its bound, off {float(off.max()):.3e}"


def _kw(op, kind, next_kind, **more):
    kw = dict(more)
    if op != "norm":
        kw["kind"] = kind
    if op != "gate_add":
        kw["next_kind"] = next_kind
    return kw


def _check(op, t, kw, dtype, what, dy=None):
    """Forward without and with gradients, and every gradient, against the oracle."""
    t = {k: v for k, v in t.items() if v is not None}
    if kw.get("kind") is None:
        t.pop("weight", None), t.pop("bias", None)
    leaves = {k: v.detach().requires_grad_(True) for k, v in t.items()}
    with torch.no_grad():
        quiet = _call(op, t, kw)
    out = _call(op, leaves, kw)
    names = list(out)
    dy = dy or {n: _rand(t["x"].device, *t["x"].shape, dtype=dtype, seed=90 + i, std=0.5) for i, n in enumerate(names)}
    want = bo.norms(t, dtype=dtype, **{"d" + n: g for n, g in dy.items()}, **kw)
    grads = torch.autograd.grad([out[n] for n in names if n in dy], list(leaves.values()), [dy[n] for n in names if n in dy])
    for n in names:
        assert torch.equal(quiet[n], out[n]), f"{what}: {n} differs where gradients are wanted"
        _close(out[n], want[n], f"{what} {n}")
    for n, g in zip(leaves, grads):
        _close(g, want["d" + n], f"{what} d{n}")
    return out, dict(zip(leaves, grads))


# ------------------------------------------------------------------------------------ the CPU


@pytest.mark.parametrize("op,kind,next_kind", [("norm", None, "layer"), ("norm", None, "rms"), ("gate_add", None, None), ("gate_add", "layer", None),
                                               ("gate_add", "rms", None), ("gate_add_norm", "layer", "rms"), ("gate_add_norm", "rms", "layer"),
                                               ("gate_add_norm", None, "layer")])
def test_oracle_gradients_against_differences(op, kind, next_kind):
    """Every gradient of the oracle's formulas against central differences of its own forward."""
    t = _tensors("cpu", (2, 3, 5), torch.float64, op=op, per=1)
    if kind is None:
        t.pop("weight", None), t.pop("bias", None)
    kw = _kw(op, kind, next_kind, eps=1e-3, next_eps=1e-2)
    if op != "norm":
        kw["residual_scale"] = 0.7
    outs = [n for n in ("stream", "normed") if (n == "stream" and op != "norm") or (n == "normed" and op != "gate_add")]
    dy = {"d" + n: _rand("cpu", 2, 3, 5, dtype=torch.float64, seed=80 + i) for i, n in enumerate(outs)}
    loss = lambda: sum(float((bo.norms(t, **kw)[n][0] * dy["d" + n]).sum()) for n in outs)  # noqa: E731
    want = bo.norms(t, **dy, **kw)
    for name, v in t.items():
        grad = want["d" + name][0].reshape(-1)
        flat = v.view(-1)
        for i in range(flat.numel()):
            old = float(flat[i])
            flat[i] = old + 1e-5
            up = loss()
            flat[i] = old - 1e-5
            down = loss()
            flat[i] = old
            assert abs((up - down) / 2e-5 - float(grad[i])) < 1e-7 * max(1.0, abs(float(grad[i]))), name


def test_oracle_sees_a_planted_mistake():
    """The bounds tell a missing mean, another sample's scale, an eps outside the root and a forgotten gate from the right result."""
    t = _tensors("cpu", (2, 4, 64), torch.bfloat16, op="gate_add_norm", per=1)
    kw = dict(kind="layer", next_kind="layer", dtype=torch.bfloat16)
    right = bo.norms(t, **kw)
    value, bound = right["normed"]
    wrong = [bo.norms(t, **{**kw, "next_kind": "rms"}), bo.norms({**t, "scale": t["scale"].flip(0)}, **kw),
             bo.norms(t, **{**kw, "next_eps": 0.3}), bo.norms({k: v for k, v in t.items() if k != "gate"}, **kw)]
    for w in wrong:
        assert bool(((w["normed"][0] - value).abs() > bound).any())


def test_refusals_without_a_gpu():
    x = torch.zeros(2, 8)
    for call in (lambda: norms.norm(x), lambda: norms.gate_add(x, x), lambda: norms.gate_add_norm(x, x)):
        with pytest.raises(RuntimeError, match="x must be a CUDA tensor"):
            call()
    with pytest.raises(ValueError, match="kind must be one of"):
        norms.norm(x, kind="batch")
    with pytest.raises(ValueError, match="kind must be one of"):
        norms.norm(x, kind=None)
    with pytest.raises(ValueError, match="next_kind must be one of"):
        norms.gate_add_norm(x, x, next_kind=None)
    with pytest.raises(ValueError, match="takes no weight"):
        norms.gate_add(x, x, torch.ones(8))
    with pytest.raises(TypeError, match="x must be a tensor"):
        norms.norm([1.0])
    with pytest.raises(TypeError, match="residual must be a tensor"):
        norms.gate_add(x, None)
    for eps in (-1e-5, math.nan, math.inf):
        with pytest.raises(ValueError, match="eps must be finite"):
            norms.norm(x, eps=eps)


def _args(**kw):
    a = N.GfNormArgs()
    base = dict(dtype=1, kind=1, next_kind=1, rows=6, cols=16, group_rows=3, eps=1e-5, next_eps=1e-5, gate_value=1.0, residual_scale=1.0, x=4096, ldx=16,
                residual=4096, ldr=16, weight=4096, gate=4096, ld_gate=16, next_weight=4096, scale=4096, ld_scale=16, stream=4096, normed=4096,
                dstream=4096, ld_dstream=16, dnormed=4096, ld_dnormed=16, dx=4096)
    for k, v in {**base, **kw}.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=3), "unknown dtype"), (dict(kind=3), "unknown norm"), (dict(next_kind=-1), "unknown norm"), (dict(rows=-6), "rows negative"),
    (dict(rows=2**31), "rows negative or too large"), (dict(cols=0), "cols must lie in"), (dict(cols=16385), "cols must lie in"),
    (dict(group_rows=0), "group_rows must divide"), (dict(group_rows=4), "group_rows must divide"), (dict(eps=math.nan), "eps must be finite"),
    (dict(next_eps=-1.0), "eps must be finite"), (dict(x=None), "x must not be NULL"), (dict(ldx=15), "x: row stride 15 is below its width 16"),
    (dict(ldr=15), "residual: row stride 15"), (dict(x=4097), "x is not aligned"), (dict(ldx=2**62), "x: too large"),
    (dict(ld_gate=8), "gate: row stride 8"), (dict(gate=4097), "gate is not aligned"), (dict(ld_scale=-16), "scale: row stride -16"),
    (dict(weight=4097), "weight is not aligned"), (dict(kind=0), "takes no weight"), (dict(next_kind=0), "without a next norm"),
    (dict(residual=None), "without a residual"), (dict(residual=None, kind=0, weight=None, gate=None, next_kind=0), "without a residual"),
])
@pytest.mark.parametrize("phase", ["forward", "backward"])
def test_abi_refuses_before_device_work(kw, msg, phase):
    lib = N.lib()
    a = _args(**kw)
    rc = lib.gf_norm_forward(ctypes.byref(a), None) if phase == "forward" else lib.gf_norm_backward(ctypes.byref(a), 4096, 2**40, None)
    assert rc == 1 and msg in lib.gf_last_error().decode(), lib.gf_last_error()


def test_abi_refuses_by_phase():
    lib = N.lib()
    err = lambda: lib.gf_last_error().decode()  # noqa: E731
    assert lib.gf_norm_forward(None, None) == 1 and lib.gf_norm_backward(None, None, 0, None) == 1 and lib.gf_norm_workspace_bytes(None) == 0
    assert lib.gf_norm_forward(ctypes.byref(_args(normed=None)), None) == 1 and "normed" in err()
    alone = dict(next_kind=0, next_weight=None, scale=None)
    assert lib.gf_norm_forward(ctypes.byref(_args(stream=None, **alone)), None) == 1 and "stream" in err()
    assert lib.gf_norm_forward(ctypes.byref(_args(residual=None, kind=0, weight=None, gate=None)), None) == 1 and "stream" in err()
    back = lambda a: lib.gf_norm_backward(ctypes.byref(a), 4096, 2**40, None)  # noqa: E731
    assert back(_args(rows=0)) == 1 and "needs rows" in err()
    assert back(_args(dnormed=None)) == 1 and "dnormed" in err()
    assert back(_args(dstream=None, **alone)) == 1 and "dstream" in err()
    assert back(_args(dbias=4096)) == 1 and "dbias without its parameter" in err()
    assert back(_args(dscale=4097)) == 1 and "dscale is not aligned" in err()
    assert back(_args(dshift=4096, **alone)) == 1 and "without a next norm" in err()
    assert lib.gf_norm_forward(ctypes.byref(_args(rows=0, x=None)), None) == 0


def test_abi_workspace():
    lib = N.lib()
    assert lib.gf_norm_workspace_bytes(ctypes.byref(_args())) == 0  # no parameter trains
    a = _args(dweight=4096)
    need = lib.gf_norm_workspace_bytes(ctypes.byref(a))
    assert need >= 2 * 4 * 16 * 4  # a chunk a group at least, four sums of its columns
    assert lib.gf_norm_backward(ctypes.byref(a), 4096, need - 1, None) == 2 and "workspace" in lib.gf_last_error().decode()
    assert lib.gf_norm_backward(ctypes.byref(a), None, need, None) == 2
    assert lib.gf_norm_backward(ctypes.byref(a), 4104, need, None) == 1 and "16-byte" in lib.gf_last_error().decode()
    for rows, cols, group in ((2**31 - 1, 8, 1), (2**31 - 1, 16384, 2**31 - 1), (2**30, 16384, 1), (1, 1, 1)):
        got = lib.gf_norm_workspace_bytes(ctypes.byref(_args(rows=rows, cols=cols, group_rows=group, ldx=cols, dweight=4096)))
        assert rows // group * 16 * cols <= got < 2**62


# ------------------------------------------------------------------------------------ the GPU

# a width on each side of every way of holding a row, odd ones among them
WIDTHS = [1, 7, 8, 64, 127, 128, 129, 320, 512, 513, 640, 1000, 1025, 1280, 1536, 1537, 2048, 2055, 4096, 4104, 6144, 6150, 8192, 8200, 12001, 16384]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("cols", WIDTHS)
@pytest.mark.parametrize("op", ["norm", "gate_add", "gate_add_norm"])
def test_widths(device, op, cols, dtype):
    _say("widths", op, cols, dtype)
    for kind, next_kind, shape, per in (("layer", "rms", (2, 5, cols), 1), ("rms", "layer", (11, cols), None)):
        t = _tensors(device, shape, dtype, op=op, per=per, seed=cols)
        _check(op, t, _kw(op, kind, next_kind), dtype, f"{op} {kind} {shape}")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 64, 300, 1025, 5000])
@pytest.mark.parametrize("op", ["norm", "gate_add", "gate_add_norm"])
def test_rows(device, op, rows, dtype):
    """Row counts on each side of every way of cutting them, with sums over all of them."""
    for cols in (24, 136):
        _say("rows", op, rows, cols, dtype)
        t = _tensors(device, (rows, cols), dtype, op=op, seed=rows)
        _check(op, t, _kw(op, "layer", "layer"), dtype, f"{op} {rows} x {cols}")


@pytest.mark.gpu
@pytest.mark.parametrize("shape,per", [((1, 7, 40), 1), ((3, 1, 40), 1), ((2, 3, 5, 40), 1), ((2, 3, 5, 40), 2), ((6, 40), 1), ((31, 3, 40), 1), ((40, 9, 40), 1),
                                       ((300, 2, 40), 1), ((9000, 40), 1), ((3, 700, 40), 1), ((4, 4, 40), 0), ((3, 33, 600), 1), ((70, 2, 2100), 1)])
@pytest.mark.parametrize("op", ["norm", "gate_add", "gate_add_norm"])
def test_samples(device, op, shape, per):
    """Gate, scale and shift of one row for all, of a row a sample, of a row for every row; few groups of many rows and many of few."""
    _say("samples", op, shape, per)
    for dtype in (torch.float32, torch.bfloat16):
        t = _tensors(device, shape, dtype, op=op, per=per, seed=sum(shape))
        _check(op, t, _kw(op, "layer", "layer"), dtype, f"{op} {shape} {per}")
    if op == "gate_add_norm":  # some shared by all rows, some a sample's
        t["gate"] = t["gate"].reshape(-1, shape[-1])[0].contiguous()
        _check(op, t, _kw(op, "layer", "layer"), dtype, "a gate for all")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["layer", "rms", None])
@pytest.mark.parametrize("next_kind", ["layer", "rms"])
def test_kinds_and_what_may_be_absent(device, kind, next_kind):
    """Every norm with every other, with and without each parameter, a number for a gate, a scaled residual, other eps."""
    _say("kinds", kind, next_kind)
    dtype = torch.bfloat16
    full = _tensors(device, (2, 9, 72), dtype, op="gate_add_norm", per=1)
    kw = _kw("gate_add_norm", kind, next_kind, residual_scale=1.7, eps=1e-3, next_eps=0.25)
    names = ("weight", "bias", "gate", "next_weight", "next_bias", "scale", "shift")
    for absent in ((), names, *((n,) for n in names), ("bias", "next_bias"), ("scale", "gate"), ("weight", "bias", "next_weight", "next_bias")):
        t = {k: v for k, v in full.items() if k not in absent}
        _check("gate_add_norm", t, {**kw, "gate": -0.4}, dtype, f"without {absent}")
        u = {k: v for k, v in t.items() if k not in ("residual", "weight", "bias", "gate")}
        _check("norm", u, {"next_kind": next_kind}, dtype, f"norm without {absent}")
        u = {k: v for k, v in t.items() if k not in ("next_weight", "next_bias", "scale", "shift")}
        _check("gate_add", u, {"kind": kind, "residual_scale": 0.0, "gate": 2.5}, dtype, f"gate_add without {absent}")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
def test_strides_and_alignment(device, dtype):
    """Rows of larger matrices, odd bases, a transposed x, slices of one modulation, gradients that are a broadcast number."""
    _say("strides", dtype)
    kw = _kw("gate_add_norm", "layer", "layer")
    t = _tensors(device, (3, 16, 72), dtype, op="gate_add_norm", per=1)
    want, grads = _check("gate_add_norm", t, kw, dtype, "plain")

    def wide(m, left, right):
        big = torch.full((*m.shape[:-1], left + m.shape[-1] + right), float("nan"), dtype=dtype, device=device)
        big[..., left:left + m.shape[-1]] = m
        return big[..., left:left + m.shape[-1]]

    for left, right in ((8, 8), (1, 2), (16, 3)):
        out, g = _check("gate_add_norm", {k: wide(v, left, right) for k, v in t.items()}, kw, dtype, f"strided {left},{right}")
        for n in want:
            assert torch.equal(out[n], want[n])
        for n in grads:
            assert torch.equal(g[n], grads[n]), n
    mods = torch.cat([t[n] for n in ("gate", "scale", "shift")], -1)
    u = dict(t, **dict(zip(("gate", "scale", "shift"), mods.chunk(3, dim=-1))))
    out, _ = _check("gate_add_norm", u, kw, dtype, "slices")
    assert torch.equal(out["normed"], want["normed"])
    u = {k: v.transpose(0, 1).contiguous().transpose(0, 1) if k in ("x", "residual") else v for k, v in t.items()}
    _check("gate_add_norm", u, kw, dtype, "transposed")
    u = dict(t, weight=torch.stack((t["weight"], t["bias"]), -1)[:, 0], gate=t["gate"][:1].expand(3, 1, 72), x=t["x"][:, :1].expand(3, 16, 72))
    _check("gate_add_norm", u, kw, dtype, "every second, expanded")
    dy = {n: torch.full((1, 1, 1), v, dtype=dtype, device=device).expand(3, 16, 72) for n, v in (("stream", 0.5), ("normed", -0.25))}
    _check("gate_add_norm", t, kw, dtype, "broadcast gradients", dy=dy)


@pytest.mark.gpu
def test_one_output_alone(device):
    """A backward from the stream alone, or from the norm alone."""
    t = _tensors(device, (2, 9, 72), torch.float32, op="gate_add_norm", per=1)
    for name in ("stream", "normed"):
        _say("one output", name)
        dy = {name: _rand(device, 2, 9, 72, dtype=torch.float32, seed=5)}
        _check("gate_add_norm", t, _kw("gate_add_norm", "layer", "rms"), torch.float32, name, dy=dy)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
def test_far_means_and_ranges(device, dtype):
    """Rows that lie far from zero against their spread, rows of one value, of zeros (also with eps 0, as the formula), tiny and large ones."""
    _say("ranges", dtype)
    cols = 200
    x = _rand(device, 8, cols, dtype=torch.float32, seed=3)
    x[0] += 100.0
    x[1] = x[1] * 0.01 - 50.0
    x[2] = 7.5
    x[3] = 0.0
    x[4] *= 1e-4
    x[5] *= 1e3
    x[6, 5] = 3e4
    t = {"x": x.to(dtype)}
    for kind in ("layer", "rms"):
        _check("norm", t, {"next_kind": kind}, dtype, kind)
    y = norms.norm(t["x"], kind="layer")
    assert bool((y[2:4] == 0).all()) and bool(torch.isfinite(y).all())
    assert bool(torch.isnan(norms.norm(torch.zeros(2, cols, dtype=dtype, device=device), kind="rms", eps=0.0)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_bad_row_stays_in_its_row(device, bad, dtype):
    """Infinities and NaN reach the outputs of their own row, the sums over it, and nothing else."""
    _say("bad rows", bad, dtype)
    for cols in (64, 1280, 2100):
        t = _tensors(device, (2, 5, cols), dtype, op="gate_add_norm", per=1)
        kw = _kw("gate_add_norm", "layer", "rms")
        clean, g0 = _check("gate_add_norm", t, kw, dtype, "clean")
        u = {k: v.clone() for k, v in t.items()}
        u["x"][1, 3, 17] = bad
        leaves = {k: v.requires_grad_(True) for k, v in u.items()}
        out = _call("gate_add_norm", leaves, kw)
        dy = [_rand(device, 2, 5, cols, dtype=dtype, seed=90 + i, std=0.5) for i in range(2)]
        g = dict(zip(leaves, torch.autograd.grad(list(out.values()), list(leaves.values()), dy)))
        keep = torch.ones(2, 5, dtype=torch.bool, device=device)
        keep[1, 3] = False
        for n in out:
            assert torch.equal(out[n][keep], clean[n][keep]) and bool(torch.isnan(out[n][1, 3]).all())
        for n in ("x", "residual"):
            assert torch.equal(g[n][keep], g0[n][keep]) and bool(torch.isnan(g[n][1, 3]).all())
        for n in ("gate", "scale"):
            assert torch.equal(g[n][0], g0[n][0]) and bool(torch.isnan(g[n][1]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["norm", "gate_add", "gate_add_norm"])
def test_no_rows(device, op):
    t = _tensors(device, (0, 3, 24), torch.float32, op=op)
    t["x"].requires_grad_(True)
    for v in t.values():
        v.requires_grad_(True)
    out = _call(op, t, _kw(op, "layer", "layer"))
    for g, v in zip(torch.autograd.grad([o.sum() for o in out.values()], list(t.values())), t.values()):
        assert g.shape == v.shape and not bool(g.any())


@pytest.mark.gpu
def test_refusals(device):
    x = torch.zeros(2, 3, 8, device=device)
    m = lambda *s, **k: torch.zeros(*s, device=device, **k)  # noqa: E731
    for call, msg in (
        (lambda: norms.norm(x, m(7)), "weight must have shape"), (lambda: norms.norm(x, m(8, dtype=torch.float16)), "weight must be torch.float32"),
        (lambda: norms.norm(x, m(8), torch.zeros(8)), "bias must be a CUDA tensor"), (lambda: norms.norm(x.double()), "x must be float32"),
        (lambda: norms.norm(m(2, 16385)), "cols must lie in"), (lambda: norms.norm(m(3, 0)), "cols must lie in"), (lambda: norms.norm(m(())), "at least one"),
        (lambda: norms.norm(x, scale=m(2, 8)), "scale must have shape"), (lambda: norms.norm(x, scale=m(1, 3, 8)), "scale must have shape"),
        (lambda: norms.norm(x, scale=m(3, 1, 8)), "scale must have shape"), (lambda: norms.norm(x, shift=m(2, 1, 1)), "shift must have shape"),
        (lambda: norms.norm(x, scale=m(2, 1, 8), shift=m(2, 3, 8)), "shared by the same rows"),
        (lambda: norms.gate_add(x, m(2, 3, 7)), "residual must have x's shape"), (lambda: norms.gate_add(x, m(6, 8)), "residual must have x's shape"),
    ):
        with pytest.raises(RuntimeError, match=msg):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["norm", "gate_add", "gate_add_norm"])
def test_the_same_bits_twice(device, op):
    """No sum depends on who comes first: two runs give the same bits, also while another stream works."""
    t = _tensors(device, (4, 600, 1280), torch.bfloat16, op=op, per=1)
    kw = _kw(op, "layer", "layer")
    runs = []
    side = torch.cuda.Stream()
    for k in range(3):
        leaves = {n: v.detach().requires_grad_(True) for n, v in t.items()}
        if k == 2:
            with torch.cuda.stream(side):
                for _ in range(20):
                    torch.relu(t["x"])
        out = _call(op, leaves, kw)
        dy = [_rand(device, 4, 600, 1280, dtype=torch.bfloat16, seed=90 + i) for i in range(len(out))]
        runs.append([*out.values(), *torch.autograd.grad(list(out.values()), list(leaves.values()), dy)])
    for other in runs[1:]:
        for a, b in zip(runs[0], other):
            assert torch.equal(a, b)
    side.synchronize()


@pytest.mark.gpu
def test_on_another_stream(device):
    """Work of a stream of its own, from tensors made there, with its workspace."""
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        t = _tensors(device, (2, 300, 320), torch.float32, op="gate_add_norm", per=1)
        side.synchronize()
        _check("gate_add_norm", t, _kw("gate_add_norm", "layer", "layer"), torch.float32, "stream")
    side.synchronize()


@pytest.mark.gpu
def test_captured_phases_replay(device):
    """Both phases in one graph, replayed with other inputs between eager work: every replay gives the eager results."""
    norms._ops()
    ops = torch.ops.guass_amd
    t = _tensors(device, (2, 200, 640), torch.bfloat16, op="gate_add_norm", per=1)
    dy = [_rand(device, 2, 200, 640, dtype=torch.bfloat16, seed=70 + i) for i in range(2)]
    args = lambda: (t["x"], t["residual"], t["weight"], t["bias"], t["gate"], 1.0, 1.0, 1, 1e-5, t["next_weight"], t["next_bias"],  # noqa: E731
                    t["scale"], t["shift"], 1, 1e-5)

    def step():
        return [*ops.block_norm_forward(*args(), True), *ops.block_norm_backward(*args(), *dy, 511)]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for k in range(4):
        for i, v in enumerate((*t.values(), *dy)):
            v.copy_(_rand(device, *v.shape, dtype=v.dtype, seed=1000 * k + i))
        graph.replay()
        torch.cuda.synchronize()
        got = [c.clone() for c in captured]
        for a, b in zip(got, step()):
            assert torch.equal(a, b), f"replay {k}"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
def test_dimensions(device, dtype):
    """One dimension, two, four; the same tensor as both inputs and as both weights."""
    _say("dimensions", dtype)
    for shape in ((72,), (5, 72), (2, 3, 4, 72)):
        t = _tensors(device, shape, dtype, op="gate_add_norm")
        _check("gate_add_norm", t, _kw("gate_add_norm", "layer", "rms"), dtype, f"{shape}")
        t["residual"], t["next_weight"] = t["x"], t["weight"]
        _check("gate_add_norm", t, _kw("gate_add_norm", "layer", "rms"), dtype, f"{shape} alike")
    x = _rand(device, 6, 72, dtype=torch.float32, seed=1).requires_grad_(True)
    dy = _rand(device, 6, 72, dtype=torch.float32, seed=2)
    both, = torch.autograd.grad(norms.gate_add(x, x, kind="rms"), x, dy)
    u, v = (x.detach().clone().requires_grad_(True) for _ in range(2))
    assert torch.equal(both, sum(torch.autograd.grad(norms.gate_add(u, v, kind="rms"), (u, v), dy)))


@pytest.mark.gpu
def test_more_elements_than_32_bits_count(device):
    """Rows behind the first 2^32 bytes and 2^31 elements: as the same rows by themselves."""
    _say("large")
    rows, cols = 2**31 // 6144 + 40, 6144
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device=device)
    x[-7:] = _rand(device, 7, cols, dtype=torch.bfloat16, seed=1)
    x[:-7] = x[-1]
    w = _rand(device, cols, dtype=torch.bfloat16, seed=2)
    stream, normed = norms.gate_add_norm(x, x, w, None, w, kind="rms")
    want = norms.gate_add_norm(x[-7:], x[-7:], w, None, w, kind="rms")
    assert torch.equal(stream[-7:], want[0]) and torch.equal(normed[-7:], want[1])
    del stream, normed
    norms._ops()
    back = torch.ops.guass_amd.block_norm_backward
    args = lambda x, g: (x, None, None, None, None, 1.0, 1.0, 0, 0.0, w, None, None, None, 1, 1e-5, None, g, 1)  # noqa: E731
    assert torch.equal(back(*args(x, x))[0][-7:], back(*args(x[-7:], x[-7:]))[0])


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [65, 300, 513, 1000, 1024, 1025, 1280, 1536, 1537])
@pytest.mark.parametrize("op", ["norm", "gate_add", "gate_add_norm"])
def test_many_rows(device, op, cols):
    """Rows enough for a wave to take one alone; with the parameters' sums and without, whose kernels hold a row otherwise."""
    for dtype, shape, per in ((torch.bfloat16, (3, 700, cols), 1), (torch.float32, (2053, cols), None), (torch.float16, (700, 3, cols), 1)):
        _say("many rows", op, cols, dtype)
        t = _tensors(device, shape, dtype, op=op, per=per, seed=cols)
        kw = _kw(op, "layer", "rms" if dtype == torch.float16 else "layer")
        _check(op, t, kw, dtype, f"{op} {shape}")
        some = {k: v.detach().requires_grad_(k in ("x", "residual")) for k, v in t.items()}
        out = _call(op, some, kw)
        dy = {n: _rand(device, *shape, dtype=dtype, seed=90 + i, std=0.5) for i, n in enumerate(out)}
        names = [n for n in ("x", "residual") if n in some]
        want = bo.norms(t, dtype=dtype, **{"d" + n: g for n, g in dy.items()}, **kw)
        for n, g in zip(names, torch.autograd.grad(list(out.values()), [some[n] for n in names], list(dy.values()))):
            _close(g, want["d" + n], f"{op} {shape} d{n} alone")
