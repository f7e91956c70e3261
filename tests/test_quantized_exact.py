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


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=ids)
@pytest.mark.parametrize("rows", [3, 32, 100])
def test_every_scale_whose_values_the_type_holds(device, rows, dtype):
    """All 16 codes at 2^-125 to 2^125, picked out by a row of x with a single 1: exact, as the type has them (0.5 * 2^-125 is its smallest
    normal number, 6 * 2^125 below its largest)."""
    _say("scales", rows, dtype)
    codes = torch.tensor([[2 * i | (2 * i + 1) << 4 for i in range(8)] * 2], dtype=torch.uint8).expand(251, 16).contiguous()
    scales = torch.arange(2, 253, dtype=torch.uint8)[:, None].contiguous()
    values = bo.dequantize(codes, scales, 32)
    w = q4.QuantizedWeight(codes.to(device), scales.to(device), 32)
    assert torch.equal(w.dequantize(dtype).cpu().double(), values)
    for first in range(0, 32, rows):
        x = torch.zeros(rows, 32, dtype=dtype)
        at = torch.arange(rows)
        x[at, (first + at) % 32] = 1.0
        got = q4.quantized_linear(x.to(device), w).cpu().double()
        assert torch.equal(got, values[:, (first + at) % 32].t())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("rows", [64, 128, 129, 200])
def test_an_infinity_at_every_number_of_rows(device, rows, dtype):
    """In x at a column of any code: infinite of the code's sign, a NaN where the code is zero, the other rows as without."""
    _say("infinity", rows, dtype)
    w, values = _weight(device, 48, 50, seed=4)
    x = _whole(rows, 50, seed=5).to(dtype).to(device)
    want = q4.quantized_linear(x, w)
    at = rows - 1 - rows // 3
    for bad in (math.inf, -math.inf):
        x[at, 49] = bad
        got = q4.quantized_linear(x, w)
        keep = torch.arange(rows, device=device) != at
        assert torch.equal(got[keep], want[keep])
        exact = values[:, 49] * bad
        assert bool(torch.isnan(exact).any()) and torch.equal(got[at].cpu().double().nan_to_num(0.5, 1.0, -1.0), exact.nan_to_num(0.5, 1.0, -1.0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("rows", [5, 80, 150])
def test_rows_of_larger_matrices_give_the_same_bits(device, rows, dtype):
    """Strides and odd bases change no sum, in float32 neither."""
    w, _ = _weight(device, 40, 72, seed=3)
    g = torch.Generator().manual_seed(6)
    x, b, r = (torch.randn(*s, generator=g).to(dtype).to(device) for s in ((rows, 72), (40,), (rows, 40)))
    want = q4.quantized_linear(x, w, b, r)
    for left, right in ((8, 8), (1, 2), (16, 3)):
        wide = []
        for m in (x, r):
            big = torch.full((rows + 1, left + m.shape[1] + right), math.nan, dtype=dtype, device=device)
            big[:-1, left:left + m.shape[1]] = m
            wide.append(big[:-1, left:left + m.shape[1]])
        assert torch.equal(q4.quantized_linear(wide[0], w, b, wide[1]), want)
