"""A block's second half run whole on its operators (guass_amd.layers: BlockNorm, FeedForwardBlock, QuantizedLinear,
QuantizedFeedForward), and how the norms and the 4-bit products take part in torch: derivatives that they do not have, gradients
that nobody asks for, autocast, traces, devices.
"""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch import nn

from guass_amd import feedforward as ff
from guass_amd import norms
from guass_amd import quantized as q4
from guass_amd.layers import (
    BlockNorm,
    FeedForwardBlock,
    GaussianAdapterConfig,
    GaussianFeedForward,
    GaussianFieldBatch,
    GaussianLinear,
    QuantizedFeedForward,
    QuantizedLinear,
)


def _say(*what):
    print("[gpu-test] block", *what, flush=True)


def _rand(device, *shape, dtype=torch.float32, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dtype).to(device)


# ------------------------------------------------------------------------------------ the CPU


def test_layers_check_what_they_are_given():
    cfg = GaussianAdapterConfig(init_num_gaussians=4)
    adapted = GaussianFeedForward(GaussianLinear(8, 24, adapter_config=cfg), GaussianLinear(12, 8, adapter_config=cfg))
    weight = lambda r, c: q4.QuantizedWeight(torch.zeros(r, 16 * -(-c // 32), dtype=torch.uint8), torch.zeros(r, -(-c // 32), dtype=torch.uint8), c)  # noqa: E731
    proj, out = QuantizedLinear(weight(24, 8)), QuantizedLinear(weight(8, 12), torch.zeros(8))
    assert (proj.out_features, proj.in_features) == (24, 8) and not out.bias.requires_grad and proj.weight.shape == (24, 8)
    FeedForwardBlock(BlockNorm(8), adapted, BlockNorm(8, kind="rms", bias=False))
    FeedForwardBlock(BlockNorm(8, affine=False), QuantizedFeedForward(proj, out))
    for error, msg, call in (
        (ValueError, "kind must be one of", lambda: BlockNorm(8, kind="batch")), (ValueError, "features must be positive", lambda: BlockNorm(0)),
        (TypeError, "must be BlockNorms", lambda: FeedForwardBlock(nn.LayerNorm(8), adapted)), (TypeError, "ff must be a", lambda: FeedForwardBlock(BlockNorm(8), nn.Linear(8, 8))),
        (TypeError, "weight must be a QuantizedWeight", lambda: QuantizedLinear(torch.zeros(4, 8))), (TypeError, "linear must be an nn.Linear", lambda: QuantizedLinear.from_linear(BlockNorm(8))),
        (TypeError, "out is not a QuantizedLinear", lambda: QuantizedFeedForward(proj, nn.Linear(12, 8))), (ValueError, "value and gate", lambda: QuantizedFeedForward(out, proj)),
        (ValueError, "activation", lambda: QuantizedFeedForward(proj, out, activation="relu")), (TypeError, "must be a LayerNorm", lambda: BlockNorm.from_norm(nn.BatchNorm1d(8))),
        (ValueError, "over the last dimension", lambda: BlockNorm.from_norm(nn.LayerNorm((4, 8)))), (ValueError, "must have an eps", lambda: BlockNorm.from_norm(nn.RMSNorm(8))),
    ):
        with pytest.raises(error, match=msg):
            call()


def test_norms_take_over_parameters():
    layer, rms = nn.LayerNorm(8, eps=1e-6), nn.RMSNorm(8, eps=1e-3)
    for norm, kind in ((layer, "layer"), (rms, "rms")):
        made = BlockNorm.from_norm(norm)
        assert made.weight is norm.weight and made.kind == kind and made.eps == norm.eps and made.features == 8
    assert BlockNorm.from_norm(layer).bias is layer.bias and BlockNorm.from_norm(rms).bias is None


def test_quantized_weight_round_trips_its_tiles():
    """Codes and scales come back as they were given, whatever the sizes; a state dict carries a layer."""
    g = torch.Generator().manual_seed(0)
    for rows, cols in ((1, 1), (16, 128), (17, 129), (5, 31), (40, 300), (0, 8)):
        groups = -(-cols // 32)
        codes, scales = (torch.randint(0, 256, (rows, n), generator=g, dtype=torch.uint8) for n in (16 * groups, groups))
        w = q4.QuantizedWeight(codes, scales, cols)
        assert torch.equal(w.codes, codes) and torch.equal(w.scales, scales)
        assert w.tile_codes.is_contiguous() and w.tile_codes.shape == (-(-rows // 16), -(-cols // 128), 1024)
        u = q4.QuantizedWeight.from_tiles(w.tile_codes, w.tile_scales, rows, cols).to("cpu")
        assert torch.equal(u.codes, codes) and torch.equal(u.scales, scales) and u.shape == (rows, cols)
    a = QuantizedLinear(q4.QuantizedWeight(torch.full((4, 16), 7, dtype=torch.uint8), torch.full((4, 1), 120, dtype=torch.uint8), 8))
    b = QuantizedLinear(q4.QuantizedWeight(torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.uint8), 8))
    b.load_state_dict(a.state_dict())
    assert torch.equal(b.weight.codes, a.weight.codes)
    with pytest.raises(ValueError, match="tile_codes of a weight"):
        q4.QuantizedWeight.from_tiles(w.tile_codes, w.tile_scales, 17, 8)


FIRST_CALLS = """
import threading
import torch
from guass_amd import norms, quantized
results = []
def call(f):
    try:
        results.append(f())
    except Exception as e:
        results.append(e)
threads = [threading.Thread(target=call, args=(f,)) for f in (norms._ops, quantized._ops) * 6]
[t.start() for t in threads], [t.join() for t in threads]
assert not any(isinstance(r, Exception) for r in results), results
assert len({id(r) for r in results}) == 2
"""


def test_first_calls_from_many_threads():
    proc = subprocess.run([sys.executable, "-c", FIRST_CALLS], cwd=Path(__file__).resolve().parent.parent, capture_output=True, text=True,
                          timeout=300)
    assert proc.returncode == 0, proc.stderr[-2000:]


# ------------------------------------------------------------------------------------ the GPU


def _norm64(x, module):
    x = x.double()
    if module.kind == "layer":
        x = (x - x.mean(-1, keepdim=True)) / (x.var(-1, correction=0, keepdim=True) + module.eps).sqrt()
    else:
        x = x / (x.square().mean(-1, keepdim=True) + module.eps).sqrt()
    x = x if module.weight is None else x * module.weight.double()
    return x if module.bias is None else x + module.bias.double()


@pytest.mark.gpu
@pytest.mark.parametrize("modulated", [False, True])
def test_adapted_block_trains(device, modulated):
    """A block on adapted layers, rendered in one batch, its norm modulated a sample, its way back normed and gated: output and every
    gradient, the Gaussians' among them, against the same block in 64 bits through torch (float32 kernels: each of about ten operations is off by
    less than 2^-15 of the norm)."""
    _say("adapted block", modulated)
    torch.manual_seed(0)
    cfg = GaussianAdapterConfig(init_num_gaussians=40, init_amp_scale=0.05, tile_out=16, tile_in=16, delta_apply="merged")
    adapted = GaussianFeedForward(GaussianLinear(64, 192, adapter_config=cfg, device=device), GaussianLinear(96, 64, adapter_config=cfg, device=device))
    block = FeedForwardBlock(BlockNorm(64, device=device), adapted, BlockNorm(64, kind="rms", device=device) if modulated else None)
    with torch.no_grad():
        for p in block.norm.parameters():
            p.add_(_rand(device, 64, seed=5, std=0.2))
    batch = GaussianFieldBatch([adapted.proj, adapted.out])
    x, dy = _rand(device, 3, 50, 64, seed=1).requires_grad_(True), _rand(device, 3, 50, 64, seed=2)
    mods = {n: _rand(device, 3, 1, 64, seed=10 + i, std=0.3).requires_grad_(True) for i, n in enumerate(("scale", "shift", "gate"))} if modulated else {}
    leaves = [x, *mods.values(), *(p for p in block.parameters() if p.requires_grad)]
    batch.render()
    y = block(x, **mods)
    got = torch.autograd.grad(y, leaves, dy)
    w1, w2 = (ly.merged_weight().double() for ly in (adapted.proj, adapted.out))
    m = {k: v.double() for k, v in mods.items()}
    h = _norm64(x, block.norm)
    h = h * (1 + m["scale"]) + m["shift"] if modulated else h
    value, gate = torch.nn.functional.linear(h, w1, adapted.proj.bias.double()).chunk(2, -1)
    z = torch.nn.functional.linear(value * torch.nn.functional.gelu(gate), w2, adapted.out.bias.double())
    ref = x.double() + (m["gate"] * _norm64(z, block.out_norm) if modulated else z)
    want = torch.autograd.grad(ref, leaves, dy.double())
    assert float((y.double() - ref).norm() / ref.norm()) < 2.0**-15
    for leaf, a, b in zip(leaves, got, want):
        assert a.shape == leaf.shape and float((a.double() - b.double()).norm() / b.double().norm()) < 2.0**-15


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("rows", [1, 7, 100])
def test_quantized_block_samples(device, rows, dtype):
    """Two blocks as a sampler runs them: the norm, the products with merged 4-bit weights, and the end of one block with the norm of the
    next in one pass; against 64 bits with the weights' values.  bfloat16: each block rounds its norm, inner activation, product and
    stream, 2^-9 of each at most: 8 roundings, amplified less than fourfold by a block of random weights, stay below 2^-4."""
    _say("quantized block", rows, dtype)
    torch.manual_seed(1)
    cfg = GaussianAdapterConfig(init_num_gaussians=24, init_amp_scale=0.05)
    parts = []
    for _ in range(2):
        adapted = GaussianFeedForward(GaussianLinear(72, 176, adapter_config=cfg, device=device), GaussianLinear(88, 72, adapter_config=cfg, device=device), activation="silu")
        made = QuantizedFeedForward.from_feed_forward(adapted)
        for ly, source in ((made.proj, adapted.proj), (made.out, adapted.out)):
            want = q4.quantize(source.merged_weight().detach())
            assert torch.equal(ly.weight.codes, want.codes) and torch.equal(ly.bias, source.bias)
        parts.append(made.to(dtype))
        assert made.proj.tile_codes.dtype == torch.uint8
    n1, n2 = BlockNorm(72, kind="rms", bias=False, device=device, dtype=dtype), BlockNorm(72, device=device, dtype=dtype)
    x = _rand(device, rows, 72, dtype=dtype, seed=3)
    with torch.no_grad():
        branch = parts[0](n1(x))
        stream, h = n2.after(branch, x, residual_scale=0.5)
        y = parts[1](h, stream)
        whole = FeedForwardBlock(n2, parts[1])(stream)

        def ff64(part, v):
            value, gate = torch.nn.functional.linear(v, part.proj.weight.dequantize().double(), part.proj.bias.double()).chunk(2, -1)
            return torch.nn.functional.linear(value * torch.nn.functional.silu(gate), part.out.weight.dequantize().double(), part.out.bias.double())

        s = 0.5 * x.double() + ff64(parts[0], _norm64(x, n1))
        ref = s + ff64(parts[1], _norm64(s, n2))
    limit = 2.0**-15 if dtype == torch.float32 else 2.0**-7 if dtype == torch.float16 else 2.0**-4
    assert float((y.double() - ref).norm() / ref.norm()) < limit
    assert float((whole.double() - ref).norm() / ref.norm()) < limit
    assert y.dtype == dtype


def _inputs(device, dtype=torch.float32, samples=2, rows=4, d=40):
    t = {n: _rand(device, samples, rows, d, dtype=dtype, seed=i) for i, n in enumerate(("x", "r"))}
    t.update({n: _rand(device, d, dtype=dtype, seed=10 + i) for i, n in enumerate(("w", "b", "w2", "b2"))})
    t.update({n: _rand(device, samples, 1, d, dtype=dtype, seed=20 + i) for i, n in enumerate(("gate", "scale", "shift"))})
    t["pb"], t["pr"] = _rand(device, 48, dtype=dtype, seed=30), _rand(device, samples, rows, 48, dtype=dtype, seed=31)
    return t


_W = {}


def _weight(device):
    if device not in _W:
        _W[device] = q4.quantize(_rand(device, 48, 40, seed=50))
    return _W[device]


CALLS = {
    "norm": (lambda t: norms.norm(t["x"], t["w2"], t["b2"], scale=t["scale"], shift=t["shift"]), ("x", "w2", "b2", "scale", "shift")),
    "gate_add": (lambda t: norms.gate_add(t["x"], t["r"], t["w"], t["b"], kind="rms", gate=t["gate"]), ("x", "r", "w", "b", "gate")),
    "gate_add_norm": (lambda t: torch.cat(norms.gate_add_norm(t["x"], t["r"], t["w"], t["b"], t["w2"], t["b2"], kind="layer", gate=t["gate"], scale=t["scale"],
                                                              shift=t["shift"], next_kind="rms"), -1), ("x", "r", "w", "b", "gate", "w2", "b2", "scale", "shift")),
    "quantized_linear": (lambda t: q4.quantized_linear(t["x"], _weight(t["x"].device), t["pb"], t["pr"]), ("x", "pb", "pr")),
    "quantized_gated_linear": (lambda t: q4.quantized_gated_linear(t["x"], _weight(t["x"].device), t["pb"]), ("x", "pb")),
}


@pytest.mark.gpu
@pytest.mark.parametrize("op", CALLS)
def test_forward_mode_raises(device, op):
    _say("forward mode", op)
    call, names = CALLS[op]
    t = _inputs(device)
    for name in names:
        for grad in (False, True):
            plain = call({**t, name: t[name].clone().requires_grad_(grad)})  # a gated product's training pass rounds elsewhere
            with fwd.dual_level():
                dual = fwd.make_dual(t[name].clone().requires_grad_(grad), torch.ones_like(t[name]))
                with pytest.raises(NotImplementedError, match=f"{op} has no forward-mode derivative"):
                    call({**t, name: dual})
                with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                    call({**t, name: dual})
                with fwd._set_fwd_grad_enabled(False):
                    assert torch.equal(call({**t, name: dual}), plain)


@pytest.mark.gpu
@pytest.mark.parametrize("op,name", [(op, n) for op in CALLS for n in CALLS[op][1] if (op, n) not in (
    ("quantized_linear", "x"), ("quantized_linear", "pb"), ("quantized_linear", "pr"))])
def test_a_second_derivative_raises(device, op, name):
    """Where a gradient depends on an input; a linear product's depend on none."""
    _say("second derivative", op, name)
    t = _inputs(device)
    t[name].requires_grad_(True)
    y = CALLS[op][0](t)
    dy = torch.ones_like(y).requires_grad_(True)
    grad, = torch.autograd.grad(y, t[name], dy, create_graph=True)
    if op == "gate_add" and name == "r":
        assert torch.equal(grad, dy)
        return
    with pytest.raises(RuntimeError, match=f"{op} is differentiable once only"):
        (grad**2).sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("op", CALLS)
def test_gradients_asked_for_are_the_full_ones(device, op):
    """Every input alone, all of them training, and every input alone training: the gradient that a full backward gives."""
    _say("asked for", op)
    call, names = CALLS[op]
    t = _inputs(device)
    plain = dict(t)
    leaves = {n: t[n].requires_grad_(True) for n in names}
    y = call(t)
    dy = _rand(device, *y.shape, seed=9)
    full = torch.autograd.grad(y, list(leaves.values()), dy, retain_graph=True)
    for (name, leaf), want in zip(leaves.items(), full):
        got, = torch.autograd.grad(y, leaf, dy, retain_graph=True)
        assert torch.equal(got, want), name
        alone = {k: v.detach() for k, v in plain.items()}
        alone[name].requires_grad_(True)
        z = call(alone)
        assert torch.equal(z, y)
        assert torch.equal(torch.autograd.grad(z, alone[name], dy)[0], want), name


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16], ids=str)
def test_autocast(device, kind):
    """The norms in float32, as torch's layer_norm; the products in autocast's type, as nn.Linear, a residual of another type after them."""
    _say("autocast", kind)
    t = _inputs(device)
    low = {k: v.to(kind) for k, v in t.items()}
    w = _weight(device)
    for op in ("norm", "gate_add", "gate_add_norm"):
        mixed = {**t, "x": low["x"], "w2": low["w2"]}
        with torch.autocast("cuda", dtype=kind):
            y = CALLS[op][0](mixed)
        assert y.dtype == torch.float32 and torch.equal(y, CALLS[op][0]({k: v.float() for k, v in mixed.items()}))
    with torch.autocast("cuda", dtype=kind):
        y = q4.quantized_linear(t["x"], w, t["pb"], t["pr"])
        z = q4.quantized_linear(low["x"], w, t["pb"], low["pr"])
        g = q4.quantized_gated_linear(t["x"], w, t["pb"])
    assert y.dtype == torch.float32 and torch.equal(y, t["pr"] + q4.quantized_linear(low["x"], w, low["pb"]))
    assert z.dtype == kind and torch.equal(z, q4.quantized_linear(low["x"], w, low["pb"], low["pr"]))
    assert g.dtype == kind and torch.equal(g, q4.quantized_gated_linear(low["x"], w, low["pb"]))
    x = t["x"].requires_grad_(True)
    with torch.autocast("cuda", dtype=kind):
        y = q4.quantized_linear(x, w, t["pb"])
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    assert dx.dtype == torch.float32
    with torch.autocast("cuda", dtype=kind), torch.autocast("cuda", enabled=False):
        assert q4.quantized_linear(t["x"], w).dtype == torch.float32


@pytest.mark.gpu
@pytest.mark.parametrize("op", CALLS)
def test_compiled_as_eager(device, op):
    """A compiled function that calls an operator: outputs and gradients as without, also with other sizes after, and without rows."""
    _say("compiled", op)
    call, names = CALLS[op]
    torch._dynamo.reset()
    norms._ops(), q4._ops(), _weight(device)
    compiled = torch.compile(lambda t: call(t) * 2, backend="aot_eager", fullgraph=True)
    for rows in (4, 4, 9, 70, 0):
        t = _inputs(device, rows=rows)
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
    """torch's own check: no input is written, none is an output, outputs have the traced shapes, types and strides."""
    _say("schemas")
    norms._ops(), q4._ops()
    ops = torch.ops.guass_amd
    utils = ("test_schema", "test_faketensor")
    for dtype in (torch.float32, torch.bfloat16):
        t = _inputs(device, dtype=dtype)
        both = (t["x"], t["r"], t["w"], t["b"], t["gate"], 1.0, 1.0, 1, 1e-5, t["w2"], t["b2"], t["scale"], t["shift"], 2, 1e-5)
        alone = (t["x"].transpose(0, 1).contiguous().transpose(0, 1), None, None, None, None, 1.0, 1.0, 0, 0.0, t["w2"], None, None, t["shift"], 1, 1e-5)
        torch.library.opcheck(ops.block_norm_forward, (*both, True), test_utils=utils)
        torch.library.opcheck(ops.block_norm_forward, (*both, False), test_utils=utils)
        torch.library.opcheck(ops.block_norm_forward, (*alone, True), test_utils=utils)
        for wants in (511, 1, 2 + 16 + 128, 0):
            torch.library.opcheck(ops.block_norm_backward, (*both, t["x"], t["r"], wants), test_utils=utils)
            torch.library.opcheck(ops.block_norm_backward, (*both, t["x"], None, wants), test_utils=utils)
        w = _rand(device, 48, 40, dtype=dtype, seed=1)
        torch.library.opcheck(ops.q4_quantize, (w,), test_utils=utils)
        codes, scales = ops.q4_quantize(w)
        torch.library.opcheck(ops.q4_dequantize, (codes, scales, 48, 40, dtype), test_utils=utils)
        for act in (0, 1):
            for save in (True, False):
                torch.library.opcheck(ops.q4_forward, (t["x"], codes, scales, t["pb"], None if act else t["pr"], 48, 40, act, save), test_utils=utils)
            y, saved = ops.q4_forward(t["x"], codes, scales, t["pb"], None, 48, 40, act, True)
            for want in ((True, True), (False, True), (True, False)):
                torch.library.opcheck(ops.q4_backward, (y, codes, scales, saved, 48, 40, act, *want), test_utils=utils)


@pytest.mark.gpu
@pytest.mark.parametrize("op", CALLS)
def test_inference_mode(device, op):
    t = _inputs(device)
    want = CALLS[op][0](t)
    with torch.inference_mode():
        assert torch.equal(CALLS[op][0]({k: v * 1 for k, v in t.items()}), want)


@pytest.mark.gpu
def test_two_streams_at_once(device):
    """The same calls on two streams, each with its own inputs, interleaved: the results of one at a time."""
    _say("two streams")
    t = [_inputs(device, samples=8, rows=300), {k: v * 0.5 for k, v in _inputs(device, samples=8, rows=300).items()}]
    for u in t:
        for v in u.values():
            v.requires_grad_(True)
    step = lambda op, u: [CALLS[op][0](u)]  # noqa: E731

    def full(op, u):
        y = CALLS[op][0](u)
        return [y, *torch.autograd.grad(y, [u[n] for n in CALLS[op][1]], torch.ones_like(y))]

    want = {op: [full(op, u) for u in t] for op in CALLS}
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = {op: [[], []] for op in CALLS}
    for op in CALLS:
        for _ in range(3):
            for i, s in enumerate(streams):
                with torch.cuda.stream(s):
                    got[op][i] = full(op, t[i])
    torch.cuda.synchronize()
    for op in CALLS:
        for i in range(2):
            for a, b in zip(got[op][i], want[op][i]):
                assert torch.equal(a, b), (op, i)


@pytest.mark.gpu
def test_operators_beside_the_feed_forward_ones(device):
    """gate_add without norm and gate is dropout_add without dropout, and a product with a weight's 4-bit values is the dense one's."""
    x, r = (_rand(device, 30, 64, dtype=torch.bfloat16, seed=i) for i in range(2))
    assert torch.equal(norms.gate_add(x, r), ff.dropout_add(x, r, p=0.0, seed=0))
    w = q4.quantize(_rand(device, 48, 64, seed=3))
    for rows in (30, 200):
        x = _rand(device, rows, 64, dtype=torch.bfloat16, seed=4)
        assert torch.equal(q4.quantized_linear(x, w), ff.linear_dropout_add(x, w.dequantize(torch.bfloat16)))
