"""What the norms around a block and the products with 4-bit weights keep for their backward, and which of their gradients can be
differentiated further.
"""

from __future__ import annotations

import pytest
import torch

from guass_amd import norms
from guass_amd import quantized as q4


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


LINEAR = {  # calls whose gradients depend on no input that trains
    "gate_add of a number": (lambda t: norms.gate_add(t["x"], t["r"], gate=0.5, residual_scale=0.25), "xr"),
    "gate_add, a frozen gate": (lambda t: norms.gate_add(t["x"], t["r"], gate=t["g"].detach()), "xr"),
    "gate_add's residual": (lambda t: norms.gate_add(t["x"].detach(), t["r"], t["w"], kind="layer", gate=t["g"], residual_scale=2.0), "r"),
    "norm's shift": (lambda t: norms.norm(t["x"], t["w"], shift=t["g"]), "g"),
    "norm's bias": (lambda t: norms.norm(t["x"], t["w"], t["b"]), "b"),
    "gate_add_norm's shift": (lambda t: norms.gate_add_norm(t["x"], t["r"], next_weight=t["w"], shift=t["g"])[1], "g"),
    "gate_add_norm's stream": (lambda t: norms.gate_add_norm(t["x"], t["r"], next_weight=t["w"], gate=0.5)[0], "xr"),
    "quantized_linear": (lambda t: q4.quantized_linear(t["x"], _weight(t["x"].device), t["b"], t["r"]), "xbr"),
}


def _weight(device):
    return q4.quantize(_rand(device, 40, 40, seed=50))


def _inputs(device):
    t = {k: _rand(device, 2, 5, 40, seed=i) for i, k in enumerate("xr")}
    t.update(w=_rand(device, 40, seed=3), b=_rand(device, 40, seed=4), g=_rand(device, 40, seed=5))
    return {k: v.requires_grad_(True) for k, v in t.items()}


@pytest.mark.gpu
@pytest.mark.parametrize("name", LINEAR)
def test_a_constant_gradient_is_no_second_derivative(device, name):
    """With create_graph such a gradient comes back as it is: a penalty on it, beside a loss, has a backward (and no say in it)."""
    _say("constant", name)
    call, train = LINEAR[name]
    t = _inputs(device)
    dy = _rand(device, 2, 5, 40, seed=9)
    leaves = [t[k] for k in train]
    want = torch.autograd.grad(call(t), leaves, dy)
    got = torch.autograd.grad(call(t), leaves, dy, create_graph=True)
    for a, b in zip(got, want):
        assert torch.equal(a, b) and not a.requires_grad
    loss = sum((g**2).sum() for g in got) + t["x"].sum()
    assert torch.equal(torch.autograd.grad(loss, t["x"])[0], torch.ones_like(t["x"]))


@pytest.mark.gpu
def test_an_unscaled_residuals_gradient_is_differentiable(device):
    """It is the stream's (the product's) gradient itself, with that one's graph, also where others refuse a second derivative."""
    for call in (lambda t: norms.gate_add(t["x"], t["r"], t["w"], kind="rms"), lambda t: q4.quantized_linear(t["x"], _weight(device), t["b"], t["r"])):
        t = _inputs(device)
        dy = _rand(device, 2, 5, 40, seed=9).requires_grad_(True)
        dx, dr = torch.autograd.grad(call(t), (t["x"], t["r"]), dy, create_graph=True)
        assert torch.equal(torch.autograd.grad((dr**2).sum(), dy)[0], 2 * dy)
        with pytest.raises(RuntimeError, match="differentiable once only"):
            (dx**2).sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("which,train", [("x", "xw"), ("x", "xg"), ("w", "xw"), ("w", "wg"), ("b", "bg"), ("g", "xg"), ("g", "wg"), ("g", "bg")])
def test_a_gradient_that_depends_refuses(device, which, train):
    """gate_add's, each by an input that it is made of and that trains; and of the next norm by the stream's."""
    t = {k: v.detach().requires_grad_(k in train) for k, v in _inputs(device).items()}
    dy = _rand(device, 2, 5, 40, seed=9)
    grad, = torch.autograd.grad(norms.gate_add(t["x"], t["r"], t["w"], t["b"], kind="layer", gate=t["g"]), t[which], dy, create_graph=True)
    with pytest.raises(RuntimeError, match="gate_add is differentiable once only"):
        (grad**2).sum().backward()
    t = _inputs(device)
    calls = {"x": t["r"], "w": t["w"], "b": t["b"], "g": t["g"]}
    _, h = norms.gate_add_norm(t["x"], t["r"], next_weight=t["w"], next_bias=t["b"], scale=t["g"])
    grad, = torch.autograd.grad(h, calls[which], dy, create_graph=True)
    with pytest.raises(RuntimeError, match="gate_add_norm is differentiable once only"):
        (grad**2).sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("kind,gate", [(None, 0.5), ("layer", 1.0)])
def test_a_broadcast_gradient_is_laid_out_once(device, kind, gate):
    """gate_add's backward takes the gradient's place for x and the residual where it reads neither, with no copies of its own for them."""
    _say("broadcast gradient", kind)
    x, r = (_rand(device, 512, 1024, seed=i).requires_grad_(True) for i in range(2))
    one = torch.full((1, 1), 3.0, device=device).expand(512, 1024)
    want = torch.autograd.grad(norms.gate_add(x, r, kind=kind, gate=gate, residual_scale=0.25), (x, r), one.contiguous())
    y = norms.gate_add(x, r * 1, kind=kind, gate=gate, residual_scale=0.25)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats(device)
    before = torch.cuda.memory_allocated(device)
    got = torch.autograd.grad(y, (x, r), one)
    size = 4 * x.numel()  # the gradient laid out, dx, the residual's, and that times 1 behind it
    assert torch.cuda.max_memory_allocated(device) - before < 4 * size + size // 2
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["gate_add of a number", "gate_add, a frozen gate", "gate_add's residual", "gate_add_norm's stream"])
def test_compiled_where_an_input_is_not_kept(device, name):
    _say("compiled", name)
    torch._dynamo.reset()
    norms._ops()
    call, train = LINEAR[name]
    compiled = torch.compile(lambda t: call(t) * 2, backend="aot_eager", fullgraph=True)
    t, dy = _inputs(device), _rand(device, 2, 5, 40, seed=9)
    leaves = [t[k] for k in train]
    want = torch.autograd.grad(call(t) * 2, leaves, dy)
    for a, b in zip(torch.autograd.grad(compiled(t), leaves, dy), want):
        assert torch.equal(a, b)
