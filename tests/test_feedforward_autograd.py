"""How the feed-forward operators take part in torch: derivatives that they do not have, gradients that nobody asks
for, autocast, tracing.
"""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest
import torch
import torch.autograd.forward_ad as fwd

from guass_amd import feedforward as ff


def _say(*what):
    print("[gpu-test] feedforward autograd", *what, flush=True)


def _rand(device, *shape, dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype).to(device)


def _inputs(device, rows=4, d=8, n=16, dtype=torch.float32):
    """x, a weight of 2 n rows, a bias of as many, a residual of the linear product's width."""
    return {"x": _rand(device, rows, d, dtype=dtype, seed=1), "w": _rand(device, 2 * n, d, dtype=dtype, seed=2),
            "b": _rand(device, 2 * n, dtype=dtype, seed=3), "r": _rand(device, rows, 2 * n, dtype=dtype, seed=4)}


CALLS = {
    "dropout_add": (lambda t: ff.dropout_add(t["x"], t["x2"], p=0.1, seed=1), ("x", "x2")),
    "gated_linear": (lambda t: ff.gated_linear(t["x"], t["w"], t["b"], p=0.1, seed=1), ("x", "w", "b")),
    "linear_dropout_add": (lambda t: ff.linear_dropout_add(t["x"], t["w"], t["b"], t["r"], p=0.1, seed=1), ("x", "w", "b", "r")),
}


@pytest.mark.gpu
@pytest.mark.parametrize("op", CALLS)
def test_forward_mode_raises(device, op):
    """A tangent on any input is refused, with gradients wanted, not wanted and switched off; not where forward mode is
    switched off."""
    _say("forward mode", op)
    call, names = CALLS[op]
    t = _inputs(device)
    t["x2"] = t["x"].clone()
    plain = call(t)
    for name in names:
        for grad in (False, True):
            with fwd.dual_level():
                dual = fwd.make_dual(t[name].clone().requires_grad_(grad), torch.ones_like(t[name]))
                with pytest.raises(NotImplementedError, match=f"{op} has no forward-mode derivative"):
                    call({**t, name: dual})
                with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                    call({**t, name: dual})
                with fwd._set_fwd_grad_enabled(False):
                    assert torch.equal(call({**t, name: dual}), plain)


@pytest.mark.gpu
@pytest.mark.parametrize("op,names", [
    ("dropout_add", ("x",)), ("linear_dropout_add", ("x", "w")), ("gated_linear", ("x",)), ("gated_linear", ("w",)),
    ("gated_linear", ("b",))])
def test_a_second_derivative_raises(device, op, names):
    """A gradient taken with a graph refuses to be differentiated, also where it depends on the bias alone."""
    _say("second derivative", op, names)
    t = _inputs(device)
    t["x2"] = None
    leaves = [t[n].requires_grad_(True) for n in names]
    y = CALLS[op][0](t)
    dy = torch.ones_like(y).requires_grad_(op == "dropout_add")
    grad = torch.autograd.grad(y, leaves, dy, create_graph=True)[0]
    with pytest.raises(RuntimeError, match=f"{op} is differentiable once only"):
        (grad**2).sum().backward()


@pytest.mark.gpu
def test_a_linear_bias_gradient_has_no_second_derivative(device):
    """The linear product's bias gradient is a sum of dy: nothing of it depends on an input, and nothing raises."""
    t = _inputs(device)
    t["b"].requires_grad_(True)
    y = ff.linear_dropout_add(t["x"], t["w"], t["b"])
    grad, = torch.autograd.grad(y.sum(), t["b"], create_graph=True)
    assert not grad.requires_grad and bool((grad == 4).all())


@pytest.mark.gpu
@pytest.mark.parametrize("with_bias", [True, False])
@pytest.mark.parametrize("op", CALLS)
def test_gradients_asked_for_are_the_full_ones(device, op, with_bias):
    """Every input alone, all of them training: the gradient that a full backward gives, with and without a bias."""
    _say("asked for", op, with_bias)
    call, names = CALLS[op]
    t = _inputs(device)
    t["x2"] = t["x"].clone()
    if not with_bias:
        t["b"] = None
        names = [n for n in names if n != "b"]
    leaves = {n: t[n].requires_grad_(True) for n in names}
    y = call(t)
    dy = _rand(device, *y.shape, seed=9)
    full = torch.autograd.grad(y, list(leaves.values()), dy, retain_graph=True)
    for (name, leaf), want in zip(leaves.items(), full):
        got, = torch.autograd.grad(y, leaf, dy, retain_graph=True)
        assert torch.equal(got, want), name


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["gated_linear", "linear_dropout_add"])
def test_gradients_not_asked_for_are_not_computed(device, op):
    """dx alone of a weight that trains too: the backward takes less memory than dweight would."""
    _say("not asked for", op)
    x, w = _rand(device, 65, 4096, dtype=torch.bfloat16), torch.zeros(16384, 4096, dtype=torch.bfloat16, device=device)
    x.requires_grad_(True), w.requires_grad_(True)
    y = ff.gated_linear(x, w) if op == "gated_linear" else ff.linear_dropout_add(x, w)
    dy = torch.ones_like(y)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    torch.autograd.grad(y, x, dy)
    assert torch.cuda.max_memory_allocated() - before < w.numel() * w.element_size()


def test_merged_layer_takes_a_parametrized_bias():
    """GaussianLinear's merged forward reads the bias as an attribute: a parametrization or an override makes it."""
    from torch.nn.utils import parametrize

    from guass_amd.layers import GaussianAdapterConfig, GaussianLinear

    class Twice(torch.nn.Module):
        def forward(self, v):
            return 2 * v

    layer = GaussianLinear(8, 6, adapter_config=GaussianAdapterConfig(init_num_gaussians=4, delta_apply="merged"))
    layer.compute_delta_weight = lambda: torch.ones(6, 8)  # the render needs a GPU
    layer.last_forward_metadata = {}
    bias = layer.bias.detach().clone()
    parametrize.register_parametrization(layer, "bias", Twice())
    x = torch.randn(3, 8)
    assert torch.equal(layer(x), torch.nn.functional.linear(x, layer.weight + 1, 2 * bias))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16], ids=str)
def test_autocast_takes_its_type(device, kind):
    """Under autocast: the same as casting by hand; a residual of another type is added after; float32 leaves get their
    gradients; dropout alone stays in its own type."""
    _say("autocast", kind)
    t = _inputs(device, rows=70, d=40, n=24)
    rng = dict(p=0.2, seed=5)
    leaves = [t[n].requires_grad_(True) for n in ("x", "w", "b", "r")]
    x, w, b, r = leaves
    low = lambda v: v.to(kind)  # noqa: E731
    cases = [(lambda: ff.gated_linear(x, w, b, **rng), lambda: ff.gated_linear(low(x), low(w), low(b), **rng), kind),
             (lambda: ff.gated_linear(low(x), w, None, **rng), lambda: ff.gated_linear(low(x), low(w), None, **rng), kind),
             (lambda: ff.linear_dropout_add(x, w, b, r, **rng), lambda: r + ff.linear_dropout_add(low(x), low(w), low(b), **rng), torch.float32),
             (lambda: ff.linear_dropout_add(low(x), w, b, low(r), **rng), lambda: ff.linear_dropout_add(low(x), low(w), low(b), low(r), **rng), kind),
             (lambda: ff.dropout_add(x, x, **rng), lambda: ff.dropout_add(x, x, **rng), torch.float32),
             (lambda: ff.dropout_add(low(x), x, **rng), lambda: x + ff.dropout_add(low(x), **rng), torch.float32)]
    for call, by_hand, want_type in cases:
        with torch.autocast("cuda", dtype=kind):
            y = call()
        want = by_hand()
        assert y.dtype == want.dtype == want_type and torch.equal(y, want)
        dy = _rand(device, *y.shape, dtype=y.dtype, seed=9)
        for got, ref in zip(torch.autograd.grad(y, leaves, dy, allow_unused=True), torch.autograd.grad(want, leaves, dy, allow_unused=True)):
            assert (got is None) == (ref is None)
            assert got is None or torch.equal(got, ref)
    with torch.autocast("cuda", dtype=kind), torch.autocast("cuda", enabled=False):
        assert ff.gated_linear(x, w, b).dtype == torch.float32


@pytest.mark.gpu
@pytest.mark.parametrize("input_type", [torch.float32, torch.bfloat16], ids=str)
def test_block_under_autocast(device, input_type):
    """The adapted block with float32 weights in bfloat16 autocast, as its parts by torch: types, output and the Gaussians'
    gradients (the composition rounds the inner activation and its parts, about eight roundings of 2^-9: 2% of
    the norm is beyond four times their sum)."""
    from guass_amd.layers import GaussianAdapterConfig, GaussianFeedForward, GaussianLinear

    _say("block autocast", input_type)
    torch.manual_seed(0)
    cfg = GaussianAdapterConfig(init_num_gaussians=48, init_amp_scale=0.05, tile_out=16, tile_in=16, delta_apply="merged")
    block = GaussianFeedForward(GaussianLinear(64, 192, adapter_config=cfg, device=device),
                                GaussianLinear(96, 64, adapter_config=cfg, device=device))
    x, r = _rand(device, 130, 64, dtype=input_type, seed=1), _rand(device, 130, 64, seed=2)
    params = [p for ly in (block.proj, block.out) for p in ly.get_gaussian_parameters().values()]
    dy = _rand(device, 130, 64, seed=3)
    results = []
    for fused in (True, False):
        with torch.autocast("cuda", dtype=torch.bfloat16):
            if fused:
                y = block(x, r)
            else:
                value, gate = block.proj(x).chunk(2, dim=-1)
                y = block.out(value * torch.nn.functional.gelu(gate)) + r
        results.append([y.detach(), *torch.autograd.grad(y, params, dy)])
    for a, b in zip(*results):
        assert a.dtype == b.dtype
        assert float((a.double() - b.double()).norm() / b.double().norm()) < 2e-2


@pytest.mark.parametrize("dtype,code", [(torch.float32, 0), (torch.bfloat16, 1), (torch.float16, 2)], ids=str)
def test_traced_size_of_what_is_saved(dtype, code):
    import ctypes

    from guass_amd import _native as N

    for rows, out in ((1, 1), (3, 8), (7, 9), (64, 5120), (1001, 777)):
        a = N.GfFfArgs()
        a.dtype, a.activation, a.rows, a.in_features, a.out_features = code, 1, rows, 16, out
        assert N.lib().gf_ff_saved_bytes(ctypes.byref(a)) == rows * ff._saved_bytes(dtype, out)


@pytest.mark.gpu
@pytest.mark.parametrize("op", CALLS)
def test_compiled_as_eager(device, op):
    """A compiled function that calls an operator: outputs and gradients as without, also with other sizes after."""
    _say("compiled", op)
    call, names = CALLS[op]
    torch._dynamo.reset()  # one code object, compiled for each operator anew
    ff._ops()  # loading the operators' library is not traced
    compiled = torch.compile(lambda t: call(t) * 2, backend="aot_eager", fullgraph=True)
    for rows in (4, 4, 9, 70):
        t = _inputs(device, rows=rows)
        t["x2"] = t["x"].clone()
        with torch.no_grad():
            assert torch.equal(compiled(t), call(t) * 2)
        leaves = [t[n].requires_grad_(True) for n in names]
        got, want = compiled(t), call(t) * 2
        assert torch.equal(got, want)
        dy = _rand(device, *want.shape, seed=9)
        for a, b in zip(torch.autograd.grad(got, leaves, dy), torch.autograd.grad(want, leaves, dy)):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_operators_hold_to_their_schemas(device):
    """torch's own check: no input is written, outputs have the traced shapes, types and strides."""
    _say("schemas")
    ops = torch.ops.guass_amd
    ff._ops()
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        t = _inputs(device, rows=5, dtype=dtype)
        seed = torch.ones(1, dtype=torch.int64, device=device)
        utils = ("test_schema", "test_faketensor")
        torch.library.opcheck(ops.dropout_forward, (t["x"], None, 0.1, 3, None, 0), test_utils=utils)
        torch.library.opcheck(ops.dropout_forward, (t["x"].t(), t["x"].t(), 0.1, 0, seed, 0), test_utils=utils)
        for act in (0, 1):
            torch.library.opcheck(ops.linear_forward, (t["x"], t["w"], t["b"], None, act, 0.1, 3, None, 0, True), test_utils=utils)
            y, saved = ops.linear_forward(t["x"], t["w"], t["b"], None, act, 0.1, 3, None, 0, True)
            for want in ((True, True, True), (False, True, False)):
                torch.library.opcheck(ops.linear_backward, (t["x"], t["w"], saved, y, act, 0.1, 3, None, 0, *want), test_utils=utils)


@pytest.mark.gpu
def test_phases_by_themselves_carry_no_gradient(device):
    t = _inputs(device)
    t["x"].requires_grad_(True)
    y, saved = ff._linear_forward(t["x"], t["w"], None, None, "gelu", 0.0, 0, 0, True)
    assert not y.requires_grad and not saved.requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("op", CALLS)
def test_compiled_without_rows(device, op):
    _say("compiled without rows", op)
    call, names = CALLS[op]
    torch._dynamo.reset()
    ff._ops()
    t = _inputs(device, rows=0)
    t["x2"] = t["x"].clone()
    leaves = [t[n].requires_grad_(True) for n in names]
    y = torch.compile(lambda t: call(t) * 2, backend="aot_eager", fullgraph=True)(t)
    assert y.shape[0] == 0
    for leaf, grad in zip(leaves, torch.autograd.grad(y.sum(), leaves)):
        assert grad.shape == leaf.shape and not bool(grad.any())


@pytest.mark.gpu
@pytest.mark.parametrize("op", CALLS)
def test_inference_mode(device, op):
    t = _inputs(device)
    t["x2"] = t["x"].clone()
    want = CALLS[op][0](t)
    with torch.inference_mode():
        u = {k: v * 1 for k, v in t.items()}
        assert torch.equal(CALLS[op][0](u), want)


FIRST_CALLS = """
import threading, time
import torch
from guass_amd import feedforward as ff
load, results = torch.ops.load_library, []
def slow(path):
    time.sleep(0.2)
    load(path)
torch.ops.load_library = slow
def call():
    try:
        results.append(ff._ops())
    except Exception as e:
        results.append(e)
threads = [threading.Thread(target=call) for _ in range(8)]
[t.start() for t in threads], [t.join() for t in threads]
assert len(results) == 8 and all(r is results[0] for r in results), results
"""


def test_first_calls_from_many_threads():
    """The operators are loaded and their shape functions registered once, whoever comes first."""
    proc = subprocess.run([sys.executable, "-c", FIRST_CALLS], cwd=Path(__file__).resolve().parent.parent, capture_output=True,
                          text=True, timeout=300)
    assert proc.returncode == 0, proc.stderr[-2000:]
