"""Limits and aliases that the sequence-model operators' C entry points refuse: host arithmetic, no GPU."""
import ctypes

from dlf_amd import hip_backend

FAKE, OTHER = ctypes.c_void_p(0x1000), ctypes.c_void_p(0x900000)
INVALID, LARGE = -1, -7


def i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


def test_more_threads_than_a_launch_counts():
    lib = hip_backend.load_library()

    def scan(m, n, strides, dtype=0):
        d, s = i64(m, n), i64(*strides)
        return lib.dlfx_gated_scan(None, b"gated", dtype, m, n, 2, d, FAKE, 0, s, FAKE, 0, s, None, 0, None, OTHER, 0, s, None, 0, None, None, 0)

    def grad(m, n, strides, dtype=0):
        d, s = i64(m, n), i64(*strides)
        return lib.dlfx_gated_scan_grad(None, b"gated", dtype, m, n, 2, d, FAKE, 0, s, None, 0, None, None, 0, None, FAKE, 0, s, FAKE, 0, s, None, 0, None,
                                        OTHER, 0, s, OTHER, 0, s, None, 0, None, None, 0)
    for call in (scan, grad):
        for dtype in (0, 4, 9):
            assert call(1 << 33, 4, (4, 1), dtype) == LARGE                   # a lane per row
            assert call(1 << 33, 20, (20, 1), dtype) == LARGE                 # lanes along the row
            assert call(1 << 33, 2000, (2000, 1), dtype) == LARGE
            assert call(1 << 31, 40, (1, 1 << 31), dtype) == LARGE            # rows side by side
            assert call(1 << 34, 400, (1, 1 << 34), dtype) == LARGE
            assert call(1 << 30, 400, (2, 1 << 32), dtype) == LARGE           # ... far apart
    m = (1 << 26) - 3
    assert lib.dlfx_route(None, b"softmax", 0, m, 8, FAKE, 0, 8, None, 1, 1, 1, 2, 0, 1.0, OTHER, OTHER, None) == LARGE
    assert lib.dlfx_route_grad(None, b"softmax", 0, m, 8, FAKE, 0, 8, 2, FAKE, FAKE, 0, 1.0, OTHER, 0, 8) == LARGE
    assert lib.dlfx_cross_entropy_piece_grad(None, 0, 2, 1 << 20, 1 << 24, FAKE, 0, 1 << 24, FAKE, 0, FAKE, None, 0.0, OTHER, 0, 1 << 24) == LARGE


def test_a_gradient_over_its_input_keeps_the_stride():
    lib = hip_backend.load_library()
    assert lib.dlfx_route_grad(None, b"sigmoid", 0, 4, 64, FAKE, 8, 64, 2, OTHER, OTHER, 0, 1.0, FAKE, 8, 65) == INVALID
    assert lib.dlfx_cross_entropy_grad(None, 0, 2, 4, 100, FAKE, 8, 100, OTHER, None, 0.0, None, FAKE, 8, 101, None, 0) == INVALID
    assert lib.dlfx_cross_entropy_piece_grad(None, 0, 2, 4, 100, FAKE, 8, 100, OTHER, 0, OTHER, None, 0.0, FAKE, 8, 101) == INVALID
