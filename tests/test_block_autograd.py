"""What the norms around a block and the products with 4-bit weights keep for their backward, and which of their gradients can be
differentiated further.
"""

from __future__ import annotations

import pytest
import torch

from guass_amd import norms


def _say(*what):
    print("[gpu-test] block autograd", *what, flush=True)


def _rand(device, *shape, dtype=torch.float32, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dtype).to(device)


# gate_add: kind, gate (a tensor of one row a sample, a number), which inputs train, which of x and the residual a gradient is made of
KEPT = [("layer", "row", "xrwbg", "x"), ("rms", 1.0, "x", "x"), (None, "row", "xr", ""), (None, "row", "xrg", "x"), (None, 0.5, "xr", ""),
        (None, 1.0, "xr", ""), ("layer", 1.0, "r", ""), ("rms", 1.0, "w", "x"), ("layer", "row", "rb", ""), (None, "row", "g", "x")]


@pytest.mark.gpu
@pytest.mark.parametrize("kind,gate,train,kept", KEPT)
def test_gate_add_keeps_what_its_gradients_are_made_of(device, kind, gate, train, kept):
    """The others may be written between forward and backward, and their memory is given back; the gradients stay the same."""
    _say("kept", kind, gate, train)
    rows, cols = 512, 1024  # a tensor is 2 MB, the parameters a few KB
    base = {"x": _rand(device, 4, rows // 4, cols, seed=1), "r": _rand(device, 4, rows // 4, cols, seed=2)}
    if kind is not None:
        base.update(w=_rand(device, cols, seed=3), b=_rand(device, cols, seed=4))
    if gate == "row":
        base["g"] = _rand(device, 4, 1, cols, seed=5)
    leaves = {k: v.requires_grad_(k in train) for k, v in base.items()}
    dy = _rand(device, 4, rows // 4, cols, seed=6)
    wanted = [leaves[k] for k in train if k in leaves]

    def call(t):
        return norms.gate_add(t["x"], t["r"], t.get("w"), t.get("b"), kind=kind, gate=t["g"] if gate == "row" else gate, residual_scale=0.5)

    want = torch.autograd.grad(call(leaves), wanted, dy)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated(device)
    own = {**leaves, "x": leaves["x"] * 1, "r": leaves["r"] * 1}
    y = call(own)
    with torch.no_grad():
        for name in "xr":
            if name not in kept:
                own[name].zero_()
    del own
    size = dy.numel() * 4
    held = torch.cuda.memory_allocated(device) - before
    assert size * (1 + len(kept)) <= held < size * (1 + len(kept)) + size // 2, f"{held / size:.2f} activations"
    for a, b in zip(torch.autograd.grad(y, wanted, dy), want):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["x", "r"])
def test_what_a_gradient_is_made_of_may_not_be_written(device, name):
    """With a next norm both are read again."""
    t = {k: _rand(device, 3, 40, seed=i).requires_grad_(True) for i, k in enumerate("xr")}
    own = {k: v * 1 for k, v in t.items()}
    _, h = norms.gate_add_norm(own["x"], own["r"])
    with torch.no_grad():
        own[name].zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        h.sum().backward()
