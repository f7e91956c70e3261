"""The norms around a block (guass_amd/norms.py) where the formula's answer is an infinity, and a large pass again and again."""

from __future__ import annotations

import math

import pytest
import torch

from guass_amd import norms

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _say(*what):
    print("[gpu-test] norms' edges", *what, flush=True)


def _rand(device, *shape, dtype, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dtype).to(device)


def _n64(x, kind):
    x = x.double()
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    return x / (x.square().mean(-1, keepdim=True) + 1e-5).sqrt() if kind else x


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("kind", ["layer", "rms", None])
@pytest.mark.parametrize("cols", [40, 600, 2100])
def test_an_infinite_factor_without_a_bias(device, cols, kind, dtype):
    """gate * n(x) and n(x) (1 + scale) of an infinite gate or scale are infinite with n(x)'s sign; other columns are as without it."""
    _say("factor", cols, kind, dtype)
    x, r, gate = _rand(device, 6, cols, dtype=dtype, seed=1), _rand(device, 6, cols, dtype=dtype, seed=2), _rand(device, cols, dtype=dtype, seed=3)
    sign = torch.sign(_n64(x, kind))[:, 17]
    others = torch.arange(cols, device=device) != 17
    for bad in (math.inf, -math.inf):
        inf = gate.clone()
        inf[17] = bad
        y, want = norms.gate_add(x, r, kind=kind, gate=inf), norms.gate_add(x, r, kind=kind, gate=gate)
        assert torch.equal(y[:, 17].double(), sign * bad) and torch.equal(y[:, others], want[:, others])
        if kind is not None:
            for shift in (None, gate):
                y, want = norms.norm(x, kind=kind, scale=inf, shift=shift), norms.norm(x, kind=kind, scale=gate, shift=shift)
                assert torch.equal(y[:, 17].double(), sign * bad) and torch.equal(y[:, others], want[:, others])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_an_infinite_gradient_without_a_bias(device, dtype):
    """The factor's gradient, sum dy n(x) weight, is infinite in its column with that element's sign (as an overflowed loss scale leaves it)."""
    _say("gradient", dtype)
    x, r, w = _rand(device, 9, 40, dtype=dtype, seed=1), _rand(device, 9, 40, dtype=dtype, seed=2), _rand(device, 40, dtype=dtype, seed=3)
    dy = _rand(device, 9, 40, dtype=dtype, seed=4)
    dy[5, 17] = math.inf
    factor = torch.zeros(40, dtype=dtype, device=device)
    want = float(torch.sign(_n64(x, "layer")[5, 17] * w[17].double())) * math.inf
    for call in (lambda f: norms.gate_add(x, r, w, kind="layer", gate=f), lambda f: norms.norm(x, w, scale=f)):
        f = factor.clone().requires_grad_(True)
        g, = torch.autograd.grad(call(f), f, dy)
        assert float(g[17]) == want and int(torch.isfinite(g).sum()) == 39


@pytest.mark.gpu
@pytest.mark.parametrize("op,shape", [("gate_add", (16, 1024, 2560)), ("gate_add_norm", (32, 256, 1280)), ("norm", (4, 4096, 320)), ("gate_add", (3, 701, 1333))])
def test_pass_after_pass_the_same_bits(device, op, shape):
    """Training passes on two sets of inputs in turn that nothing waits between, as many workgroups' sums joined as a card has units: every
    output and gradient has the bits of a pass by itself."""
    _say("again", op, shape)
    cols, dtype = shape[-1], torch.bfloat16
    sets = []
    for k in range(2):
        t = {"x": _rand(device, *shape, dtype=dtype, seed=10 * k), "r": _rand(device, *shape, dtype=dtype, seed=10 * k + 1)}
        t.update({n: _rand(device, cols, dtype=dtype, seed=10 * k + 2 + i) for i, n in enumerate("wb")})
        t.update({n: _rand(device, shape[0], 1, cols, dtype=dtype, seed=10 * k + 4 + i) for i, n in enumerate(("g", "s"))})
        sets.append(({n: v.requires_grad_(True) for n, v in t.items()}, [_rand(device, *shape, dtype=dtype, seed=10 * k + 6 + i) for i in range(2)]))

    def step(k):
        t, dy = sets[k]
        if op == "norm":
            out, names = (norms.norm(t["x"], t["w"], t["b"], scale=t["g"], shift=t["s"]),), "xwbgs"
        elif op == "gate_add":
            out, names = (norms.gate_add(t["x"], t["r"], t["w"], t["b"], kind="layer", gate=t["g"]),), "xrwbg"
        else:
            out, names = norms.gate_add_norm(t["x"], t["r"], t["w"], t["b"], t["w"], t["b"], kind="layer", gate=t["g"], scale=t["s"]), "xrwbgs"
        return [*(o.detach() for o in out), *torch.autograd.grad(out, [t[n] for n in names], dy[:len(out)])]

    want = []
    for k in range(2):
        want.append(step(k))
        torch.cuda.synchronize()
    differ = torch.zeros((), dtype=torch.int64, device=device)
    for i in range(24):
        for a, b in zip(step(i % 2), want[i % 2]):
            differ += (a != b).sum()
    assert int(differ) == 0
