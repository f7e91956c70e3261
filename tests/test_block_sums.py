"""The parameters' gradients of the norms around a block: the column sums that they are made of, and the memory that these take."""

from __future__ import annotations

import ctypes

import pytest
import torch

from guass_amd import _native as N
from guass_amd import norms


def _say(*what):
    print("[gpu-test] block sums", *what, flush=True)


def _args(**kw):
    a = N.GfNormArgs()
    base = dict(dtype=1, kind=1, next_kind=1, eps=1e-5, next_eps=1e-5, gate_value=1.0, residual_scale=1.0, x=4096, residual=4096, weight=4096,
                next_weight=4096, stream=4096, normed=4096, dstream=4096, dnormed=4096, dx=4096)
    for k, v in {**base, **kw}.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("rows,cols,group", [(2**20, 64, 1), (16384, 2560, 16384), (16384, 2560, 1024), (4096, 333, 1), (100000, 1280, 20), (2**31 - 1, 16384, 1)])
def test_a_half_alone_takes_no_memory_for_the_other(rows, cols, group):
    """Two sums a column and chunk for each half that is there (groups of one row: as many chunks as rows)."""
    need = lambda **kw: N.lib().gf_norm_workspace_bytes(ctypes.byref(_args(  # noqa: E731
        rows=rows, cols=cols, group_rows=group, ldx=cols, ldr=cols, **kw)))
    norm = need(residual=None, kind=0, weight=None, dnext_weight=4096)
    gate_add = need(next_kind=0, next_weight=None, dweight=4096)
    width = -(-cols // 8) * 8
    for got in (norm, gate_add):
        assert got % 256 == 0 and got >= rows // group * 2 * 4 * width
    if group == 1:  # and what several slabs of groups give to be joined, and both rounded up
        for got in (norm, gate_add):
            assert got <= rows * 2 * 4 * width + 64 * 4 * 4 * width + 512
    else:
        assert gate_add <= 2 * 768 * 2 * 4 * width + rows // group * 2 * 4 * width + 64 * 4 * 4 * width + 512


# ------------------------------------------------------------------------------------ the GPU


def _whole(device, *shape, seed, most=2):
    """Whole numbers, none of them zero: a row that is lost shows in every column."""
    g = torch.Generator().manual_seed(seed)
    return (torch.randint(1, most + 1, shape, generator=g) * (torch.randint(0, 2, shape, generator=g) * 2 - 1)).double().to(device)


def _signs(device, *shape, seed):
    """Rows of as many 1 as -1, of an even number of columns that is a power of two: mean 0 and mean square 1 exactly, so n(x) = x with eps 0."""
    g = torch.Generator().manual_seed(seed)
    order = torch.rand(*shape, generator=g).argsort(-1)
    return torch.where(order % 2 == 0, 1.0, -1.0).double().to(device)


def _sums(call, t, grads, names, dtype):
    leaves = {k: v.to(dtype).requires_grad_(True) for k, v in t.items()}
    out = call(leaves)
    return dict(zip(names, torch.autograd.grad(out, [leaves[n] for n in names], [g.to(dtype) for g in grads])))


def _exact(got, want, dtype, sums, what):
    """Equal to the exact sum rounded once; and the exact sum without any one row would not be (in the columns whose sum the type holds)."""
    for n, w in want.items():
        assert torch.equal(got[n].cpu(), w.to(dtype).cpu()), f"{what} d{n}: {int((got[n].cpu() != w.to(dtype).cpu()).sum())} of {w.numel()} columns"
    for row in (0, sums.shape[0] // 2, sums.shape[0] - 1):
        assert bool(((sums.sum(0) - sums[row]).to(dtype) != sums.sum(0).to(dtype)).any()), "a lost row would not show"


ROWS = [1, 2, 15, 16, 17, 63, 64, 300, 1025, 5000, 20011]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("rows", ROWS)
def test_a_gates_sums_are_exact(device, rows, dtype):
    """sum over the rows of ds x, whole numbers below 2^24: exact in 32 bits in whatever order; every way of holding a row, widths with a
    part of a group of columns among them, and rows in samples."""
    for cols in (24, 333, 640, 1285, 2100, 8200):
        if rows * cols > 2**23:
            continue
        _say("gate", rows, cols, dtype)
        x, dy, r = (_whole(device, rows, cols, seed=i) for i in range(3))
        got = _sums(lambda t: norms.gate_add(t["x"], t["r"], gate=t["gate"]), {"x": x, "r": r, "gate": torch.ones_like(x[0])}, [dy], ["gate"], dtype)
        _exact(got, {"gate": (dy * x).sum(0)}, dtype, dy * x, f"{rows} x {cols}")
        for samples in (2, 5):
            if rows % samples:
                continue
            v = lambda t: t.view(samples, rows // samples, cols)  # noqa: E731
            got = _sums(lambda t: norms.gate_add(t["x"], t["r"], gate=t["gate"]), {"x": v(x), "r": v(r), "gate": torch.ones_like(v(x)[:, :1])}, [v(dy)],
                        ["gate"], dtype)
            _exact(got, {"gate": (v(dy) * v(x)).sum(1, keepdim=True)}, dtype, dy * x, f"{samples} of {rows} x {cols}")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_the_norms_sums_are_exact(device, kind, rows, dtype):
    """Rows of as many 1 as -1 are their own norm, so all sums are of whole numbers: norm's, gate_add's and both halves' of gate_add_norm."""
    for cols in (32, 512, 1024, 2048):
        if rows * cols > 2**23:
            continue
        _say("norm", kind, rows, cols, dtype)
        x, dy, one = _signs(device, rows, cols, seed=1), _whole(device, rows, cols, seed=2), torch.ones(cols, dtype=torch.float64, device=device)
        s0, s1 = dy.sum(0), (dy * x).sum(0)
        zero = torch.zeros_like(one)
        t = {"x": x, "w": one, "b": zero, "scale": zero, "shift": zero}
        got = _sums(lambda t: norms.norm(t["x"], t["w"], t["b"], kind=kind, scale=t["scale"], shift=t["shift"], eps=0.0), t, [dy], ["w", "b", "scale", "shift"], dtype)
        _exact(got, {"w": s1, "b": s0, "scale": s1, "shift": s0}, dtype, dy, f"norm {rows} x {cols}")
        t = {"x": x, "r": dy, "w": one, "b": zero, "gate": one}
        got = _sums(lambda t: norms.gate_add(t["x"], t["r"], t["w"], t["b"], kind=kind, gate=t["gate"], eps=0.0), t, [dy], ["w", "b", "gate"], dtype)
        _exact(got, {"w": s1, "b": s0, "gate": s1}, dtype, dy, f"gate_add {rows} x {cols}")
        # both halves: s = x, so the next norm is x too; its sums from its gradient, the branch's from the stream's alone
        t = {"x": x, "r": torch.zeros_like(x), "w": one, "b": zero, "gate": one, "w2": one, "b2": zero, "scale": zero, "shift": zero}
        call = lambda t: norms.gate_add_norm(t["x"], t["r"], t["w"], t["b"], t["w2"], t["b2"], kind=kind, gate=t["gate"], next_kind=kind,  # noqa: E731
                                             scale=t["scale"], shift=t["shift"], eps=0.0, next_eps=0.0)
        names = ["w", "b", "gate", "w2", "b2", "scale", "shift"]
        got = _sums(call, t, [torch.zeros_like(dy), dy], names, dtype)
        _exact({n: got[n] for n in names[3:]}, {"w2": s1, "b2": s0, "scale": s1, "shift": s0}, dtype, dy, f"gate_add_norm's norm {rows} x {cols}")
        got = _sums(call, t, [dy, torch.zeros_like(dy)], names, dtype)
        _exact(got, {"w": s1, "b": s0, "gate": s1, **{n: zero for n in names[3:]}}, dtype, dy, f"gate_add_norm's branch {rows} x {cols}")


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [8, 130])
def test_more_groups_than_workgroups(device, cols):
    """A gate, scale and shift of each row's own, for more rows than a grid has workgroups (2^20): each row's gradient, and what all rows
    share, of whole numbers."""
    rows = 2**20 + 77
    _say("groups", rows, cols)
    x, dy = _whole(device, rows, cols, seed=1).float(), _whole(device, rows, cols, seed=2).float()
    gate = torch.ones_like(x).requires_grad_(True)
    x.requires_grad_(True)
    y = norms.gate_add(x, dy, gate=gate)
    assert torch.equal(y, x + dy)
    dx, dgate = torch.autograd.grad(y, (x, gate), dy)
    assert torch.equal(dx, dy) and torch.equal(dgate, dy * x)
    del y, dx, dgate, gate
    zero = torch.zeros(rows, cols, device=device)
    scale, shift, bias = (t.requires_grad_(True) for t in (zero.clone(), zero, torch.zeros(cols, device=device)))
    ds, db, dscale = torch.autograd.grad(norms.norm(x.detach(), None, bias, kind="rms", scale=scale, shift=shift), (shift, bias, scale), dy)
    assert torch.equal(ds, dy) and torch.equal(db.double(), dy.double().sum(0))
    want = dy.double() * (x.detach().double() / (x.detach().double().square().mean(-1, keepdim=True) + 1e-5).sqrt())
    # squares are exact; 1 / cols, their mean with eps, the root to within 3 units, the norm and the product: 8 roundings at most
    assert bool(((dscale.double() - want).abs() <= 8 * 2.0**-24 * want.abs()).all())
