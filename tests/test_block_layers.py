"""The layers on the norms around a block and on 4-bit weights (guass_amd.layers): what they are made of."""

from __future__ import annotations

import pytest
import torch
from torch import nn

from guass_amd.layers import BlockNorm


def test_a_norm_without_an_eps_takes_a_given_one():
    rms = nn.RMSNorm(8)
    assert rms.eps is None
    eps = torch.finfo(torch.float32).eps
    made = BlockNorm.from_norm(rms, eps=eps)
    assert made.eps == eps and made.kind == "rms" and made.weight is rms.weight and made.bias is None
    assert BlockNorm.from_norm(nn.LayerNorm(8, eps=1e-3), eps=0.0).eps == 0.0
    with pytest.raises(ValueError, match="must have an eps, or eps be given"):
        BlockNorm.from_norm(rms)


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
