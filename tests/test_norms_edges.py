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
