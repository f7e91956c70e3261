"""The layers on the norms around a block and on 4-bit weights (guass_amd.layers): what they are made of."""

from __future__ import annotations

import pytest
import torch
from torch import nn

from guass_amd.layers import BlockNorm, QuantizedFeedForward, QuantizedLinear
from guass_amd.quantized import QuantizedWeight


def test_a_norm_without_an_eps_takes_a_given_one():
    rms = nn.RMSNorm(8)
    assert rms.eps is None
    eps = torch.finfo(torch.float32).eps
    made = BlockNorm.from_norm(rms, eps=eps)
    assert made.eps == eps and made.kind == "rms" and made.weight is rms.weight and made.bias is None
    assert BlockNorm.from_norm(nn.LayerNorm(8, eps=1e-3), eps=0.0).eps == 0.0
    with pytest.raises(ValueError, match="must have an eps, or eps be given"):
        BlockNorm.from_norm(rms)


def _quantized(rows, cols, value, bias=False):
    groups = -(-cols // 32)
    weight = QuantizedWeight(torch.full((rows, 16 * groups), value, dtype=torch.uint8), torch.full((rows, groups), 120, dtype=torch.uint8), cols)
    return QuantizedLinear(weight, torch.full((rows,), float(value)) if bias else None)


def test_a_state_dict_of_another_size_is_refused():
    """Also where the tiles, of 16 rows and 128 columns, are alike; the layer stays as it was."""
    for rows, cols in ((20, 40), (24, 33), (17, 128)):
        layer, other = _quantized(24, 40, 1), _quantized(rows, cols, 2)
        assert layer.tile_codes.shape == other.tile_codes.shape
        with pytest.raises(RuntimeError, match=rf"size mismatch for weight: \[{rows}, {cols}\] in the checkpoint, the layer's is \[24, 40\]"):
            layer.load_state_dict(other.state_dict())
        assert torch.equal(layer.weight.codes, _quantized(24, 40, 1).weight.codes)
    ff, other = (QuantizedFeedForward(_quantized(2 * n, 40, n), _quantized(40, n, n)) for n in (20, 18))
    with pytest.raises(RuntimeError, match="size mismatch for proj.weight"):
        ff.load_state_dict(other.state_dict())


def test_a_state_dict_loads():
    """As saved and read back, without the size, and not strictly; what is missing or too much is said as ever."""
    import io

    whole = _quantized(24, 40, 2, bias=True)
    file = io.BytesIO()
    torch.save(whole.state_dict(), file)
    file.seek(0)
    state = torch.load(file, weights_only=True)
    old = {k: v for k, v in state.items() if k != "_extra_state"}
    for given in (state, old):
        layer = _quantized(24, 40, 1, bias=True)
        assert layer.load_state_dict(given) == ([], [])
        assert torch.equal(layer.weight.codes, whole.weight.codes) and torch.equal(layer.weight.scales, whole.weight.scales)
        assert torch.equal(layer.bias, whole.bias)
    layer = _quantized(24, 40, 1)
    with pytest.raises(RuntimeError, match="Unexpected key"):
        layer.load_state_dict(state)
    keys = layer.load_state_dict({"tile_codes": state["tile_codes"]}, strict=False)
    assert keys.missing_keys == ["tile_scales"] and torch.equal(layer.tile_codes, whole.tile_codes)


@pytest.mark.gpu
def test_a_given_eps_is_torchs_default(device):
    """On rows so small that eps counts: torch's own RMSNorm without an eps, in 64 bits with float32's."""
    x = torch.randn(5, 40, generator=torch.Generator().manual_seed(1)).to(device) * 1e-3
    rms = nn.RMSNorm(40, device=device)
    eps = torch.finfo(torch.float32).eps
    y = BlockNorm.from_norm(rms, eps=eps)(x)
    want = x.double() / (x.double().square().mean(-1, keepdim=True) + eps).sqrt()
    # squares and their sum, 1 / sqrt, two products: at most 40 + 8 roundings of 2^-24
    assert float(((y.double() - want).abs() / want.abs()).max()) < 48 * 2.0**-24
    assert torch.allclose(y, rms(x), rtol=1e-5, atol=0)
