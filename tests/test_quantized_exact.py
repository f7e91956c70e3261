"""Products with 4-bit weights (guass_amd/quantized.py) whose every sum is exact: whatever is lost, taken twice or taken from another
row, tile or lane shows.
"""

from __future__ import annotations

import math

import pytest
import torch

from guass_amd import quantized as q4
from oracle import block_oracle as bo

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
ids = lambda v: str(v).replace("torch.", "") if isinstance(v, torch.dtype) else None  # noqa: E731


def _say(*what):
    print("[gpu-test] quantized exact", *what, flush=True)


def _whole(rows, cols, seed, most=3):
    return torch.randint(-most, most + 1, (rows, cols), generator=torch.Generator().manual_seed(seed)).double()


def _weight(device, rows, cols, seed):
    """Any codes at the scale 1: multiples of a half, of 6 at most."""
    groups = -(-cols // 32)
    codes = torch.randint(0, 256, (rows, 16 * groups), generator=torch.Generator().manual_seed(seed), dtype=torch.uint8)
    scales = torch.full((rows, groups), 127, dtype=torch.uint8)
    return q4.QuantizedWeight(codes.to(device), scales.to(device), cols), bo.dequantize(codes, scales, cols)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("rows", [1, 4, 5, 16, 17, 32, 33, 64, 65, 128, 129])
def test_sums_of_whole_numbers(device, rows, dtype):
    """x of whole numbers up to 3 by multiples of a half up to 6: a sum of 20000 stays below 2^20 and a half is its step, so 32 bits hold
    every partial one in whatever order, and the output is the exact one rounded once.  Several tiles for each wave, a part of one, more
    columns than a workgroup's, and enough of them for the wide form."""
    for d, n in ((128, 48), (2056, 40), (19999, 24), (700, 8200)):
        _say(rows, d, n, dtype)
        w, values = _weight(device, n, d, seed=d)
        x = _whole(rows, d, seed=rows)
        got, want = q4.quantized_linear(x.to(dtype).to(device), w).cpu(), (x @ values.t()).to(dtype)
        if dtype == torch.float32 and rows > 128:
            # The dense products split 32 bits into three planes, and 2^-126 stands in an empty one: a sum's parts are no whole numbers
            # then, and each of its 6 d additions may round by 2^-24, 16 more at its end (oracle/feedforward_oracle.py).
            bound = (6 * d + 16) * 2.0**-24 * (x.abs() @ values.abs().t())
            assert bool(((got.double() - want).abs() <= bound).all()), f"{rows} x {d} -> {n}"
            continue
        assert torch.equal(got, want), f"{rows} x {d} -> {n}"
