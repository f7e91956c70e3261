"""The feed-forward entries' size arithmetic over the whole range of their arguments, without a GPU.

Run under AddressSanitizer and UndefinedBehaviorSanitizer as well (tests/test_sanitized_host.py).
"""

from __future__ import annotations

import ctypes

import pytest

from guass_amd import _native as N

LIMIT = 2**48  # elements of a matrix


def _args(**kw):
    a = N.GfFfArgs()
    base = dict(dtype=1, activation=1, rows=4, in_features=16, out_features=8, x=4096, ldx=16, weight=4096, ldw=16, y=4096,
                dy=4096, lddy=8, saved=4096, dx=4096, dweight=4096, dbias=4096)
    for k, v in {**base, **kw}.items():
        setattr(a, k, v)
    return a


def _queries(a):
    lib = N.lib()
    return (lib.gf_ff_saved_bytes(ctypes.byref(a)), lib.gf_ff_workspace_bytes(ctypes.byref(a), 0),
            lib.gf_ff_workspace_bytes(ctypes.byref(a), 1))


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("kw", [
    dict(rows=2**31 - 1, out_features=2**29 - 1),              # the saved values' bytes pass 63 bits
    dict(rows=2**31 - 1, in_features=2**30 - 1, ldx=2**30 - 1, ldw=2**30 - 1),
    dict(in_features=2**30 - 1, out_features=2**29 - 1, ldx=2**30 - 1, ldw=2**30 - 1),
    dict(ldx=2**62), dict(ldw=2**62), dict(lddy=2**62), dict(ldx=-2**62), dict(residual=4096, ldr=2**62),
])
def test_sizes_past_every_memory_are_refused(kw, dtype):
    lib = N.lib()
    a = _args(dtype=dtype, **kw)
    assert _queries(a) == (0, 0, 0)
    assert "too large" in lib.gf_last_error().decode()
    for phase in (lib.gf_ff_forward, lib.gf_ff_backward):
        assert phase(ctypes.byref(a), None, 0, None) == 1
        assert "too large" in lib.gf_last_error().decode()


def test_row_strides_are_bounded_by_the_rows():
    """A stride that is fine by itself, times the rows, is not."""
    lib = N.lib()
    a = _args(rows=2**20, ldx=2**29)
    assert lib.gf_ff_forward(ctypes.byref(a), None, 0, None) == 1 and "x: too large" in lib.gf_last_error().decode()
    d = N.GfDropout(0.5, 1, None, 0)
    assert lib.gf_dropout_add(0, ctypes.byref(d), 2**20, 8, 4096, 2**29, None, 0, 4096, 8, None) == 1
    assert "x: too large" in lib.gf_last_error().decode()


@pytest.mark.parametrize("dtype,element", [(0, 8), (1, 5), (2, 6)])
def test_saved_bytes_up_to_the_limit(dtype, element):
    a = _args(dtype=dtype, rows=2**31 - 1, out_features=2**16 - 3, in_features=8)
    assert _queries(a)[0] == (2**31 - 1) * 2**16 * element


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("rows,d,n", [(1, 1, 1), (64, 8, 8), (65, 8, 8), (2**31 - 1, 8, 2**10), (1, 2**21, 2**20), (2**20, 2**21, 2**19)])
def test_workspaces_over_the_range(dtype, rows, d, n):
    """Both phases count without overflow, and for the packed operands at least."""
    for act in (0, 1):
        a = _args(dtype=dtype, activation=act, rows=rows, in_features=d, out_features=n, ldx=d, ldw=d, lddy=n)
        saved, forward, backward = _queries(a)
        w_rows = n * (1 + act)
        elements = (rows * d + w_rows * d) * 6
        assert forward < 2**62 and backward < 2**62
        if dtype == 0:
            assert forward >= (elements if rows > 64 else 0) and backward >= elements + rows * w_rows * 6
