"""Gradients over their own inputs: refused by address, however the start is given.  Host arithmetic, no GPU."""
import ctypes

import pytest

from dlf_amd import hip_backend

OTHER = ctypes.c_void_p(0x900000)
INVALID = -1


@pytest.mark.parametrize("dtype,size", [(0, 4), (4, 2), (9, 2)])
@pytest.mark.parametrize("x_offset,dx_offset", [(8, 0), (0, 8), (8, 8), (-3, 5)])
def test_one_start_as_two_pointers(dtype, size, x_offset, dx_offset):
    lib = hip_backend.load_library()
    x, dx = (ctypes.c_void_p(0x10000 - size * o) for o in (x_offset, dx_offset))
    assert lib.dlfx_route_grad(None, b"sigmoid", dtype, 4, 64, x, x_offset, 64, 2, OTHER, OTHER, 0, 1.0, dx, dx_offset, 65) == INVALID
    assert lib.dlfx_cross_entropy_grad(None, dtype, 2, 4, 100, x, x_offset, 100, OTHER, None, 0.0, None, dx, dx_offset, 101, None, 0) == INVALID
    assert lib.dlfx_cross_entropy_piece_grad(None, dtype, 2, 4, 100, x, x_offset, 100, OTHER, 0, OTHER, None, 0.0, dx, dx_offset, 101) == INVALID
