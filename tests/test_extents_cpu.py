"""Extents and positions that the operators of attention between cells refuse before they work anything out: no GPU."""
import ctypes

import pytest

from dihydrogen_b200 import _abi
from test_attention_cpu import attention, desc, nd, rotary, status


@pytest.mark.parametrize("dims", [(1 << 32, 1 << 32), (1 << 16, 1 << 31, 1 << 31), (1 << 62, 4), (3, 1 << 62, 1 << 62),
                                  (1 << 15, 1 << 15)])
def test_cells_whose_number_wraps(dims):
    few = nd(1, 8, 4, 7)
    assert attention(desc(), nd(1, 16, *dims), few) == _abi.UNSUPPORTED
    assert attention(desc(), nd(1, 16, 4, 7), nd(1, 8, *dims)) == _abi.UNSUPPORTED
    assert status("dcb_attention_workspace_bytes", desc(), nd(1, 16, *dims), few, 0) == -1


@pytest.mark.parametrize("dims", [(0, 1 << 62, 1), (1 << 62, 0, 1), (0, 1 << 31, 4), (0, 1 << 61, 0)])
def test_rotary_tables_of_an_empty_tensor_with_a_long_axis(dims):
    assert rotary(xd=nd(1, 24, *dims), nsd=3, axis=(2, 4, 2)) == _abi.UNSUPPORTED


def test_rotary_tables_that_no_memory_holds():
    assert rotary(xd=nd(1, 1 << 16, 0, (1 << 31) - 1, 0), nsd=3, head_dim=1 << 16, rotated_heads=1,
                  axis=(0, 1 << 16, 0)) == _abi.BAD_ARG
    assert b"memory" in _abi.lib().dcb_last_error()


@pytest.mark.parametrize("kw", [dict(base=1e-320), dict(step=1e308), dict(step=-1e308), dict(base=1e-300, step=1e100)])
def test_rotary_angles_that_are_not_finite(kw):
    """base^(-2j / a) or step times a position passes what a double holds: the table would be NaN."""
    rd = _abi.RotaryDesc()
    rd.nsd, rd.head_dim, rd.rotated_heads, rd.base = 2, 256, 1, kw.get("base", 100.0)
    rd.axis_channels[1], rd.axis_channels[2] = 0, 256
    for i in range(3):
        rd.step[i] = kw.get("step", 1.0)
    assert status("dcb_rotary_plan_create", rd, nd(1, 256, 3, 500), ctypes.byref(ctypes.c_void_p())) == _abi.BAD_ARG
    assert b"finite" in _abi.lib().dcb_last_error()


@pytest.mark.parametrize("scale", [2.4e38, 2.9e38, 3.4e38])
def test_attention_scales_that_overflow_in_powers_of_two(scale):
    few = nd(1, 8, 4, 7)
    assert attention(desc(scale=scale), nd(1, 16, 4, 7), few) == _abi.BAD_ARG
    assert b"scale" in _abi.lib().dcb_last_error()
    assert status("dcb_attention_workspace_bytes", desc(scale=2.3e38), nd(1, 16, 4, 7), few, 0) >= 0
