"""The parameters' gradients of the norms around a block: the column sums that they are made of, and the memory that these take."""

from __future__ import annotations

import ctypes

import pytest

from guass_amd import _native as N


def _args(**kw):
    a = N.GfNormArgs()
    base = dict(dtype=1, kind=1, next_kind=1, eps=1e-5, next_eps=1e-5, gate_value=1.0, residual_scale=1.0, x=4096, residual=4096, weight=4096,
                next_weight=4096, stream=4096, normed=4096, dstream=4096, dnormed=4096, dx=4096)
    for k, v in {**base, **kw}.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("rows,cols,group", [(2**20, 64, 1), (16384, 2560, 16384), (16384, 2560, 1024), (4096, 333, 1), (100000, 1280, 20), (2**31 - 1, 16384, 1)])
def test_a_half_alone_takes_no_memory_for_the_other(rows, cols, group):
    """Two sums a column and chunk for each half that is there (groups of one row: as many chunks as rows)."""
    need = lambda **kw: N.lib().gf_norm_workspace_bytes(ctypes.byref(_args(  # noqa: E731
        rows=rows, cols=cols, group_rows=group, ldx=cols, ldr=cols, **kw)))
    norm = need(residual=None, kind=0, weight=None, dnext_weight=4096)
    gate_add = need(next_kind=0, next_weight=None, dweight=4096)
    width = -(-cols // 8) * 8
    for got in (norm, gate_add):
        assert got % 256 == 0 and got >= rows // group * 2 * 4 * width
    if group == 1:  # and what several slabs of groups give to be joined, and both rounded up
        for got in (norm, gate_add):
            assert got <= rows * 2 * 4 * width + 64 * 4 * 4 * width + 512
    else:
        assert gate_add <= 2 * 768 * 2 * 4 * width + rows // group * 2 * 4 * width + 64 * 4 * 4 * width + 512
