"""ctypes binding of libdlfx.so (the C ABI in include/dlfx.h) plus the backend
object the front-ends call.  PyTorch is used only to own device memory and to
name the HIP stream work is enqueued on.

There is no fallback: if the library is missing or a call fails, this raises.
"""
from __future__ import annotations

import ctypes
import functools
import math
import os
from ctypes import c_char_p, c_float, c_int, c_int64, c_size_t, c_void_p, POINTER

import numpy as np

from .frontend import BFLOAT16, Tensor, to_bfloat16
from .shape import Shape, ShapeError

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "lib", "libdlfx.so")

_I64P = POINTER(c_int64)


class DlfxError(RuntimeError):
    def __init__(self, status: int, text: str, where: str):
        super().__init__("%s: %s (status %d)" % (where, text, status))
        self.status = status


def _declare(lib):
    view = [c_int, _I64P, _I64P]
    lib.dlfx_version.restype = c_int
    lib.dlfx_status_string.restype = c_char_p
    lib.dlfx_status_string.argtypes = [c_int]
    lib.dlfx_last_hip_error.restype = c_int
    lib.dlfx_set_tuning.restype = c_int
    lib.dlfx_set_tuning.argtypes = [c_char_p, c_int64]

    lib.dlfx_reduce_scratch_bytes.restype = c_size_t
    lib.dlfx_reduce_scratch_bytes.argtypes = [c_int, c_int64, c_int64]
    lib.dlfx_reduce.restype = c_int
    lib.dlfx_reduce.argtypes = ([c_void_p, c_char_p, c_int, c_int64, c_int64] + view + [c_void_p, c_int64]
                                + view + [c_void_p, c_int64, c_void_p, c_size_t])

    lib.dlfx_reduce_static.restype = c_int
    lib.dlfx_reduce_static.argtypes = ([c_void_p, c_char_p, c_int, c_int64, c_int64] + view + [c_void_p, c_int64]
                                       + view + [c_void_p, c_int64])

    lib.dlfx_logits_head.restype = c_int
    lib.dlfx_logits_head.argtypes = [c_void_p, c_int, c_int64, c_int64, c_void_p, c_int64, c_int64,
                                     c_void_p, c_void_p, c_void_p, c_void_p, c_int64, c_void_p, c_void_p]

    lib.dlfx_arg_reduce_scratch_bytes.restype = c_size_t
    lib.dlfx_arg_reduce_scratch_bytes.argtypes = [c_int, c_int64, c_int64]
    lib.dlfx_arg_reduce.restype = c_int
    lib.dlfx_arg_reduce.argtypes = ([c_void_p, c_char_p, c_int, c_int, c_int64, c_int64] + view
                                    + [c_void_p, c_int64] + view + [c_void_p, c_int64, c_void_p, c_size_t])

    lib.dlfx_scan_scratch_bytes.restype = c_size_t
    lib.dlfx_scan_scratch_bytes.argtypes = [c_int, c_int64, c_int64]
    lib.dlfx_scan.restype = c_int
    lib.dlfx_scan.argtypes = [c_void_p, c_char_p, c_int, c_int64, c_int64, c_int, c_int, _I64P,
                              c_void_p, c_int64, _I64P, c_void_p, c_int64, _I64P, c_void_p, c_size_t]

    lib.dlfx_sort_scratch_bytes.restype = c_size_t
    lib.dlfx_sort_scratch_bytes.argtypes = [c_int, c_int64, c_int64]
    lib.dlfx_sort.restype = c_int
    lib.dlfx_sort.argtypes = [c_void_p, c_int, c_int, c_int, _I64P, c_void_p, c_int64, _I64P,
                              c_void_p, c_int64, _I64P, c_void_p, c_size_t]

    lib.dlfx_argsort_scratch_bytes.restype = c_size_t
    lib.dlfx_argsort_scratch_bytes.argtypes = [c_int, c_int64, c_int64]
    lib.dlfx_argsort.restype = c_int
    lib.dlfx_argsort.argtypes = [c_void_p, c_int, c_int, c_int, c_int, _I64P, c_void_p, c_int64, _I64P,
                                 c_void_p, c_int64, _I64P, c_void_p, c_int64, _I64P, c_void_p, c_size_t]

    lib.dlfx_top_k_scratch_bytes.restype = c_size_t
    lib.dlfx_top_k_scratch_bytes.argtypes = [c_int, c_int64, c_int64, c_int64]
    lib.dlfx_top_k.restype = c_int
    lib.dlfx_top_k.argtypes = [c_void_p, c_int64, c_int, c_int, c_int, c_int, _I64P, _I64P,
                               c_void_p, c_int64, _I64P, c_void_p, c_int64, _I64P,
                               c_void_p, c_int64, _I64P, c_void_p, c_size_t]
    lib.dlfx_count_scratch_bytes.restype = c_size_t
    lib.dlfx_count_scratch_bytes.argtypes = [c_int, c_int64, c_int64]
    lib.dlfx_count.restype = c_int
    lib.dlfx_count.argtypes = ([c_void_p, c_int, c_int64, c_int64, c_void_p] + view + [c_void_p, c_int64]
                               + view + [c_void_p, c_int64, c_void_p, c_size_t])

    lib.dlfx_scan_nonzero_scratch_bytes.restype = c_size_t
    lib.dlfx_scan_nonzero_scratch_bytes.argtypes = [c_int, c_int64, c_int64]
    lib.dlfx_scan_nonzero.restype = c_int
    lib.dlfx_scan_nonzero.argtypes = [c_void_p, c_int, c_int64, c_int64, c_int, c_int, _I64P,
                                      c_void_p, c_int64, _I64P, c_void_p, c_int64, _I64P, c_void_p, c_size_t]

    lib.dlfx_softmax.restype = c_int
    lib.dlfx_softmax.argtypes = [c_void_p, c_char_p, c_int, c_int64, c_int64, c_void_p, c_int64, c_void_p, c_int64, c_void_p, c_size_t]
    lib.dlfx_softmax_scratch_bytes.restype = c_size_t
    lib.dlfx_softmax_scratch_bytes.argtypes = [c_int, c_int64, c_int64]

    lib.dlfx_merge_scratch_bytes.restype = c_size_t
    lib.dlfx_merge_scratch_bytes.argtypes = [c_int, c_int64, c_int64]
    lib.dlfx_merge.restype = c_int
    lib.dlfx_merge.argtypes = [c_void_p, c_int, c_int, c_int, _I64P, _I64P, c_void_p, c_int64,
                               _I64P, _I64P, c_void_p, c_int64, _I64P, _I64P, c_void_p, c_int64, c_void_p, c_size_t]

    lib.dlfx_gather_indices.restype = c_int
    lib.dlfx_gather_indices.argtypes = [c_void_p, c_int64, c_int64, c_int, c_int, _I64P,
                                        c_void_p, c_int64, c_void_p, c_int64]
    lib.dlfx_copy.restype = c_int
    lib.dlfx_copy.argtypes = [c_void_p, c_int, c_int, _I64P, c_void_p, c_int64, _I64P, c_void_p, c_int64, _I64P]
    lib.dlfx_fill.restype = c_int
    lib.dlfx_fill.argtypes = [c_void_p, c_int, c_int, _I64P, _I64P, c_void_p, c_int64, c_void_p]

    part, scratch, rows = [c_void_p, c_int64, _I64P], [c_void_p, c_size_t], [c_void_p, c_int64, c_int64]
    lib.dlfx_gated_scan_scratch_bytes.restype = c_size_t
    lib.dlfx_gated_scan_scratch_bytes.argtypes = [c_int, c_int64, c_int64]
    lib.dlfx_gated_scan.restype = c_int
    lib.dlfx_gated_scan.argtypes = [c_void_p, c_char_p, c_int, c_int64, c_int64, c_int, _I64P] + part * 5 + scratch
    lib.dlfx_gated_scan_grad.restype = c_int
    lib.dlfx_gated_scan_grad.argtypes = [c_void_p, c_char_p, c_int, c_int64, c_int64, c_int, _I64P] + part * 9 + scratch
    lib.dlfx_route.restype = c_int
    lib.dlfx_route.argtypes = ([c_void_p, c_char_p, c_int, c_int64, c_int64] + rows + [c_void_p, c_int64, c_int64, c_int, c_int64, c_int, c_float]
                               + [c_void_p] * 3)
    lib.dlfx_route_grad.restype = c_int
    lib.dlfx_route_grad.argtypes = ([c_void_p, c_char_p, c_int, c_int64, c_int64] + rows + [c_int64, c_void_p, c_void_p, c_int, c_float] + rows)
    lib.dlfx_cross_entropy_scratch_bytes.restype = c_size_t
    lib.dlfx_cross_entropy_scratch_bytes.argtypes = [c_int, c_int64, c_int64]
    matrix = [c_void_p, c_int, c_int, c_int64, c_int64] + rows + [c_void_p]
    lib.dlfx_cross_entropy.restype = c_int
    lib.dlfx_cross_entropy.argtypes = matrix + [c_float, c_void_p] + scratch
    lib.dlfx_cross_entropy_grad.restype = c_int
    lib.dlfx_cross_entropy_grad.argtypes = matrix + [c_void_p, c_float, c_void_p] + rows + scratch
    lib.dlfx_cross_entropy_piece.restype = c_int
    lib.dlfx_cross_entropy_piece.argtypes = matrix + [c_int64, c_int, c_void_p] + scratch
    lib.dlfx_cross_entropy_join.restype = c_int
    lib.dlfx_cross_entropy_join.argtypes = [c_void_p, c_int, c_int64, c_void_p, c_void_p, c_float, c_void_p]
    lib.dlfx_cross_entropy_piece_grad.restype = c_int
    lib.dlfx_cross_entropy_piece_grad.argtypes = matrix + [c_int64, c_void_p, c_void_p, c_float] + rows
    return lib


_lib = None

# Every symbol include/dlfx.h declares.
EXPORTS = ("dlfx_version", "dlfx_status_string", "dlfx_last_hip_error", "dlfx_set_tuning",
           "dlfx_reduce_scratch_bytes", "dlfx_reduce", "dlfx_reduce_static", "dlfx_logits_head",
           "dlfx_arg_reduce_scratch_bytes", "dlfx_arg_reduce",
           "dlfx_scan_scratch_bytes", "dlfx_scan",
           "dlfx_sort_scratch_bytes", "dlfx_sort",
           "dlfx_argsort_scratch_bytes", "dlfx_argsort",
           "dlfx_top_k_scratch_bytes", "dlfx_top_k",
           "dlfx_count_scratch_bytes", "dlfx_count",
           "dlfx_scan_nonzero_scratch_bytes", "dlfx_scan_nonzero", "dlfx_gather_indices",
           "dlfx_merge_scratch_bytes", "dlfx_merge", "dlfx_softmax_scratch_bytes", "dlfx_softmax",
           "dlfx_copy", "dlfx_fill",
           "dlfx_gated_scan_scratch_bytes", "dlfx_gated_scan", "dlfx_gated_scan_grad", "dlfx_route", "dlfx_route_grad",
           "dlfx_cross_entropy_scratch_bytes", "dlfx_cross_entropy", "dlfx_cross_entropy_grad", "dlfx_cross_entropy_piece",
           "dlfx_cross_entropy_join", "dlfx_cross_entropy_piece_grad")


def load_library():
    """Loads libdlfx.so; raises when it has not been built (no fallback exists)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError("libdlfx.so is not built: run `python -m dlf_amd.build` "
                               "(or __graft_entry__.build()) first; expected at " + LIB_PATH)
        _lib = _declare(ctypes.CDLL(LIB_PATH))
    return _lib


def _arr(values):
    values = list(values)
    return (c_int64 * max(1, len(values)))(*values)


@functools.lru_cache(maxsize=4096)
def _const(values: tuple):
    """A C array of extents or strides that a call only reads."""
    return (c_int64 * max(1, len(values)))(*values)


def _check(status: int, where: str):
    if status != 0:
        lib = load_library()
        text = lib.dlfx_status_string(status).decode()
        if status == -6:
            text += " (hipError %d)" % lib.dlfx_last_hip_error()
        raise DlfxError(status, text, where)


_NP_TO_TORCH = None


def _torch_dtype(np_dtype):
    global _NP_TO_TORCH
    if _NP_TO_TORCH is None:
        import torch
        _NP_TO_TORCH = {np.dtype(np.float32): torch.float32, np.dtype(np.float64): torch.float64,
                        np.dtype(np.int32): torch.int32, np.dtype(np.int64): torch.int64,
                        np.dtype(np.float16): torch.float16, np.dtype(np.int16): torch.int16,
                        np.dtype(np.bool_): torch.bool,
                        np.dtype(np.complex64): torch.complex64, np.dtype(np.complex128): torch.complex128,
                        BFLOAT16: torch.bfloat16}
    return _NP_TO_TORCH[np.dtype(np_dtype)]


def _dtype_code_of(torch_dtype, torch):
    return {torch.float32: 0, torch.float64: 1, torch.int32: 2, torch.int64: 3, torch.float16: 4, torch.int16: 5,
            torch.bool: 6, torch.complex64: 7, torch.complex128: 8, torch.bfloat16: 9}[torch_dtype]


class HipBackend:
    """Backend whose six boundary calls go through the C ABI onto the current HIP stream."""

    name = "hip"

    def __init__(self, device: str = "cuda:0"):
        import torch
        if not torch.cuda.is_available():
            raise RuntimeError("no HIP device visible to PyTorch")
        self.torch = torch
        self.device = torch.device(device)
        if self.device.index is None:            # "cuda": the current one, from here on
            self.device = torch.device(self.device.type, torch.cuda.current_device())
        self.lib = load_library()
        self._scratch = None
        self._retired = []
        self._from_torch_dtype = None

    # -- storage ------------------------------------------------------------
    def alloc(self, dtype, count: int):
        return self.torch.empty(count or 1, dtype=_torch_dtype(dtype), device=self.device)

    def upload(self, flat: np.ndarray):
        if flat.dtype == BFLOAT16:
            return self.torch.from_numpy(np.ascontiguousarray(flat).view(np.int16)).to(self.device).view(self.torch.bfloat16)
        return self.torch.from_numpy(np.ascontiguousarray(flat)).to(self.device)

    @staticmethod
    def _flat(storage):
        """A storage's memory in one row: from_torch and new leave a tensor's own shape on it."""
        if storage.is_contiguous():
            return storage.view(-1)
        return storage.as_strided((1 + sum((e - 1) * s for e, s in zip(storage.shape, storage.stride())),), (1,))

    def download(self, storage) -> np.ndarray:
        storage = self._flat(storage)
        if storage.dtype == self.torch.bfloat16:
            return storage.view(self.torch.int16).cpu().numpy().view(BFLOAT16)
        return storage.cpu().numpy()

    def copy_view(self, storage, shape):
        """Row-major device copy of a strided view (dlfx_copy: the reference's reorder(X, Y))."""
        out = self.torch.empty(max(1, shape.size), dtype=storage.dtype, device=self.device)
        if shape.size == 0:              # an empty slice: nothing to move
            return out
        dense = []
        size = 1
        for e in reversed(shape.extents):
            dense.insert(0, size)
            size *= e
        self._call(self.lib.dlfx_copy, "dlfx_copy", _dtype_code_of(storage.dtype, self.torch), len(shape.extents), _arr(shape.extents),
                   storage.data_ptr(), shape.offset, _arr(shape.strides), out.data_ptr(), 0, _arr(dense))
        return out

    def copy(self, dtype, extents, x, x_offset, x_strides, y, y_offset, y_strides, defer=False):
        return self._issue(self.lib.dlfx_copy, "dlfx_copy", (dtype, len(extents), _arr(extents)),
                           (x.data_ptr(), x_offset, _arr(x_strides), y.data_ptr(), y_offset, _arr(y_strides)), defer, (x, y))

    def fill(self, dtype, extents, strides, x, x_offset, value, defer=False):
        host_types = {0: np.float32, 1: np.float64, 2: np.int32, 3: np.int64, 4: np.float16, 5: np.int16,
                      6: np.bool_, 7: np.complex64, 8: np.complex128}
        v = to_bfloat16([value]) if dtype == 9 else np.array([value], dtype=host_types[dtype])
        call = self._issue(self.lib.dlfx_fill, "dlfx_fill", (dtype, len(extents), _arr(extents), _arr(strides)),
                           (x.data_ptr(), x_offset, v.ctypes.data_as(c_void_p)), defer, (x,))
        if call is None:
            return None
        return lambda v=v: call()

    def wrap(self, tensor):
        """Use an existing contiguous 1-D device tensor as storage."""
        return tensor

    def from_torch(self, tensor) -> Tensor:
        """A Tensor over the memory of a torch tensor of this backend's device (no copy; any strides).

        What is computed from it has no history: torch's autograd neither sees these calls nor their gradients, which
        are calls of their own.  A tensor that requires a gradient is therefore refused while torch records (detach it,
        or call inside torch.no_grad() or an autograd function)."""
        if tensor.device != self.device:
            raise ValueError("the tensor is on %s, this backend on %s" % (tensor.device, self.device))
        if tensor.is_conj() or tensor.is_neg():
            raise ValueError("a view that torch conjugates or negates when it is read: resolve it first")
        if tensor.requires_grad:
            if self.torch.is_grad_enabled():
                raise ValueError("the tensor requires a gradient, which torch would not get through these calls: detach() it first")
            tensor = tensor.detach()
        extents = tuple(tensor.shape)
        if 0 in extents:
            raise ShapeError("extent must be positive")
        return Tensor(self, Shape.of(extents, tensor.stride()), tensor, self._np_dtype(tensor.dtype))

    def new(self, extents: tuple, dtype) -> Tensor:
        """A Tensor of its own memory, not initialised."""
        return Tensor(self, Shape.dense(extents), self.torch.empty(extents, dtype=_torch_dtype(dtype), device=self.device), dtype)

    def to_torch(self, T: Tensor):
        """The torch view of a Tensor's memory (no copy; torch has no negative strides)."""
        sh, storage = T.shape, T.storage
        if sh.offset == 0 and storage.shape == sh.extents and storage.stride() == sh.strides:
            return storage
        if sh.strides and min(sh.strides) < 0:
            raise ShapeError("to_torch: a flipped view has no torch form; take contiguous() first")
        return storage.as_strided(sh.extents, sh.strides, storage.storage_offset() + sh.offset)

    def _np_dtype(self, torch_dtype):
        if self._from_torch_dtype is None:
            _torch_dtype(np.float32)
            self._from_torch_dtype = {v: k for k, v in _NP_TO_TORCH.items()}
        try:
            return self._from_torch_dtype[torch_dtype]
        except KeyError:
            raise TypeError("unsupported element type %r" % (torch_dtype,))

    def scratch(self, nbytes: int):
        if nbytes == 0:
            return None, 0
        if self._scratch is None or self._scratch.numel() < nbytes:
            # deferred calls keep pointers into earlier buffers: retire, do not free
            if self._scratch is not None:
                self._retired.append(self._scratch)
            self._scratch = self.torch.empty(nbytes, dtype=self.torch.uint8, device=self.device)
        return self._scratch.data_ptr(), nbytes

    def _stream(self):
        return self.torch.cuda.current_stream(self.device).cuda_stream

    # -- boundary calls -----------------------------------------------------
    # Each method marshals its arguments once and either issues the call or, with
    # defer=True, returns a closure that re-issues it (used by the benchmark so
    # that the timed region holds the C-ABI call and nothing else).
    def _issue(self, fn, where, head, tail, defer, keep=()):
        torch, device = self.torch, self.device

        def call(_keep=keep):        # the closure owns the buffers whose addresses it passes
            _check(fn(torch.cuda.current_stream(device).cuda_stream, *head, *tail), where)
        if defer:
            return call
        call()
        return None

    def reduce(self, name, dtype, m, n, xs, x, ys, y, defer=False):
        sp, sb = self.scratch(self.lib.dlfx_reduce_scratch_bytes(dtype, m, n))
        return self._issue(self.lib.dlfx_reduce, "dlfx_reduce(%s)" % name,
                           (name.encode(), dtype, m, n),
                           (xs.rank, _arr(xs.extents), _arr(xs.strides), x.data_ptr(), xs.offset,
                            ys.rank, _arr(ys.extents), _arr(ys.strides), y.data_ptr(), ys.offset, sp, sb), defer, (x, y))

    def reduce_static(self, name, dtype, m, n, xs, x, ys, y, defer=False):
        """dlfx_reduce_static: the same reduction with the library's own static device scratch."""
        return self._issue(self.lib.dlfx_reduce_static, "dlfx_reduce_static(%s)" % name,
                           (name.encode(), dtype, m, n),
                           (xs.rank, _arr(xs.extents), _arr(xs.strides), x.data_ptr(), xs.offset,
                            ys.rank, _arr(ys.extents), _arr(ys.strides), y.data_ptr(), ys.offset), defer, (x, y))

    def logits_head(self, dtype, m, n, x, x_offset, row_stride, sums, maxs, argmaxs, lses, k, best_values, best_indices,
                    defer=False):
        """dlfx_logits_head: sum, max, argmax, log-sum-exp and the k best of every row in one launch;
        any output (a device tensor) may be None."""
        def ptr(t):
            return None if t is None else t.data_ptr()
        return self._issue(self.lib.dlfx_logits_head, "dlfx_logits_head", (dtype, m, n),
                           (x.data_ptr(), x_offset, row_stride, ptr(sums), ptr(maxs), ptr(argmaxs), ptr(lses), k,
                            ptr(best_values), ptr(best_indices)), defer,
                           (x, sums, maxs, argmaxs, lses, best_values, best_indices))

    def arg_reduce(self, name, dtype, index_dtype, rows, k, xs, x, ys, y, defer=False):
        sp, sb = self.scratch(self.lib.dlfx_arg_reduce_scratch_bytes(dtype, rows, k))
        return self._issue(self.lib.dlfx_arg_reduce, "dlfx_arg_reduce(%s)" % name,
                           (name.encode(), dtype, index_dtype, rows, k),
                           (xs.rank, _arr(xs.extents), _arr(xs.strides), x.data_ptr(), xs.offset,
                            ys.rank, _arr(ys.extents), _arr(ys.strides), y.data_ptr(), ys.offset, sp, sb), defer, (x, y))

    def scan(self, name, dtype, m, n, exclusive, xs, x, ys, y, defer=False):
        sp, sb = self.scratch(self.lib.dlfx_scan_scratch_bytes(dtype, m, n))
        return self._issue(self.lib.dlfx_scan, "dlfx_scan(%s)" % name,
                           (name.encode(), dtype, m, n, int(bool(exclusive))),
                           (xs.rank, _arr(xs.extents), x.data_ptr(), xs.offset, _arr(xs.strides),
                            y.data_ptr(), ys.offset, _arr(ys.strides), sp, sb), defer, (x, y))

    def sort(self, direction, dtype, xs, x, ys, y, defer=False):
        n = xs.extents[-1]
        sp, sb = self.scratch(self.lib.dlfx_sort_scratch_bytes(dtype, xs.size // n, n))
        return self._issue(self.lib.dlfx_sort, "dlfx_sort", (direction, dtype),
                           (xs.rank, _arr(xs.extents), x.data_ptr(), xs.offset, _arr(xs.strides),
                            y.data_ptr(), ys.offset, _arr(ys.strides), sp, sb), defer, (x, y))

    def argsort(self, direction, dtype, index_dtype, xs, x, ys, y, is_, i, defer=False):
        n = xs.extents[-1]
        sp, sb = self.scratch(self.lib.dlfx_argsort_scratch_bytes(dtype, xs.size // n, n))
        return self._issue(self.lib.dlfx_argsort, "dlfx_argsort", (direction, dtype, index_dtype),
                           (xs.rank, _arr(xs.extents), x.data_ptr(), xs.offset, _arr(xs.strides),
                            y.data_ptr() if y is not None else None,
                            ys.offset if ys is not None else 0,
                            _arr(ys.strides) if ys is not None else None,
                            i.data_ptr(), is_.offset, _arr(is_.strides), sp, sb), defer, (x, y, i))

    def top_k(self, limit, direction, dtype, index_dtype, xs, x, ys, y, is_, i, defer=False):
        n = xs.extents[-1]
        sp, sb = self.scratch(self.lib.dlfx_top_k_scratch_bytes(dtype, xs.size // n, n, limit))
        return self._issue(self.lib.dlfx_top_k, "dlfx_top_k", (limit, direction, dtype, index_dtype),
                           (xs.rank, _arr(xs.extents), _arr(ys.extents),
                            x.data_ptr(), xs.offset, _arr(xs.strides),
                            y.data_ptr(), ys.offset, _arr(ys.strides),
                            i.data_ptr(), is_.offset, _arr(is_.strides), sp, sb), defer, (x, y, i))

    def count(self, dtype, m, n, value, xs, x, ys, y, defer=False):
        sp, sb = self.scratch(self.lib.dlfx_count_scratch_bytes(dtype, m, n))
        host_types = {0: np.float32, 1: np.float64, 2: np.int32, 3: np.int64, 4: np.float16, 5: np.int16,
                      7: np.complex64, 8: np.complex128}
        v = np.array([value], dtype=host_types[dtype])       # one host element of the input's type
        keep = v.ctypes.data_as(c_void_p)
        call = self._issue(self.lib.dlfx_count, "dlfx_count", (dtype, m, n, keep),
                           (xs.rank, _arr(xs.extents), _arr(xs.strides), x.data_ptr(), xs.offset,
                            ys.rank, _arr(ys.extents), _arr(ys.strides), y.data_ptr(), ys.offset, sp, sb), defer, (x, y))
        if call is None:
            return None
        return lambda v=v: call()      # the closure keeps the host value alive

    def scan_nonzero(self, dtype, m, n, exclusive, xs, x, ys, y, defer=False):
        sp, sb = self.scratch(self.lib.dlfx_scan_nonzero_scratch_bytes(dtype, m, n))
        return self._issue(self.lib.dlfx_scan_nonzero, "dlfx_scan_nonzero", (dtype, m, n, int(bool(exclusive))),
                           (xs.rank, _arr(xs.extents), x.data_ptr(), xs.offset, _arr(xs.strides),
                            y.data_ptr(), ys.offset, _arr(ys.strides), sp, sb), defer, (x, y))

    def gather_indices(self, m, n, row_major, dims, counts, out, defer=False):
        return self._issue(self.lib.dlfx_gather_indices, "dlfx_gather_indices", (m, n, int(bool(row_major))),
                           (len(dims), _arr(dims), counts.data_ptr(), 0, out.data_ptr(), 0), defer, (counts, out))

    def softmax(self, name, dtype, m, n, x, x_offset, y, y_offset, defer=False):
        sp, sb = self.scratch(self.lib.dlfx_softmax_scratch_bytes(dtype, m, n))
        return self._issue(self.lib.dlfx_softmax, "dlfx_softmax(%s)" % name, (name.encode(), dtype, m, n),
                           (x.data_ptr(), x_offset, y.data_ptr(), y_offset, sp, sb), defer, (x, y))

    def merge(self, direction, dtype, xs, x, ys, y, zs, z, defer=False):
        n = zs.extents[-1]
        sp, sb = self.scratch(self.lib.dlfx_merge_scratch_bytes(dtype, zs.size // n, n))
        return self._issue(self.lib.dlfx_merge, "dlfx_merge", (direction, dtype, zs.rank),
                           (_arr(xs.extents), _arr(xs.strides), x.data_ptr(), xs.offset,
                            _arr(ys.extents), _arr(ys.strides), y.data_ptr(), ys.offset,
                            _arr(zs.extents), _arr(zs.strides), z.data_ptr(), zs.offset, sp, sb), defer, (x, y, z))

    # -- sequence-model operators ---------------------------------------------
    # Scratch is allocated call by call from torch's stream-ordered allocator, so calls on different
    # streams and recorded graphs never share it.
    def _call(self, fn, where, *args):
        torch = self.torch
        device = self.device.index or 0
        if torch.cuda.current_device() != device:
            with torch.cuda.device(self.device):
                return self._call(fn, where, *args)
        # (current_stream(device).cuda_stream makes two Python objects for the same handle: 2.7 us, this 0.1)
        _check(fn(torch._C._cuda_getCurrentRawStream(device), *args), where)

    def _call_scratch(self, nbytes):
        if nbytes == 0:
            return None, 0, None
        buffer = self.torch.empty(nbytes, dtype=self.torch.uint8, device=self.device)
        return buffer.data_ptr(), nbytes, buffer

    @staticmethod
    def _part(part):
        """Pointer, offset and strides of a (storage, offset, strides), or nothing."""
        return (None, 0, None) if part is None else (part[0].data_ptr(), part[1], _const(part[2]))

    @staticmethod
    def _state(T):
        """The same of a tensor of one value per row."""
        return (None, 0, None) if T is None else (T.storage.data_ptr(), T.shape.offset, _const(T.shape.strides))

    @staticmethod
    def _start(T):
        return None if T is None else T.storage.data_ptr() + T.shape.offset * T.storage.element_size()

    def gated_scan(self, kind, dtype, dims, g, x, initial, y, last):
        """g, x, y: (storage, offset, strides) of views with the scanned axis last; initial (or None) and last: tensors."""
        n, m = dims[-1], math.prod(dims[:-1])
        sp, sb, keep = self._call_scratch(self.lib.dlfx_gated_scan_scratch_bytes(dtype, m, n))
        self._call(self.lib.dlfx_gated_scan, "dlfx_gated_scan", kind.encode(), dtype, m, n, len(dims), _const(dims),
                   *self._part(g), *self._part(x), *self._state(initial), *self._part(y), *self._state(last), sp, sb)

    def gated_scan_grad(self, kind, dtype, dims, g, x, y, dy, dg, dx, initial, dlast, dinitial):
        n, m = dims[-1], math.prod(dims[:-1])
        sp, sb, keep = self._call_scratch(self.lib.dlfx_gated_scan_scratch_bytes(dtype, m, n))
        self._call(self.lib.dlfx_gated_scan_grad, "dlfx_gated_scan_grad", kind.encode(), dtype, m, n, len(dims), _const(dims),
                   *self._part(g), *self._part(x), *self._state(initial), *self._part(y), *self._part(dy), *self._state(dlast),
                   *self._part(dg), *self._part(dx), *self._state(dinitial), sp, sb)

    def route(self, score, dtype, m, n, x, stride, bias, groups, kept_groups, group_best, k, renormalise, scale, weights, indices, loads):
        self._call(self.lib.dlfx_route, "dlfx_route", score.encode(), dtype, m, n, x.storage.data_ptr(), x.shape.offset, stride, self._start(bias),
                   groups, kept_groups, group_best, k, int(renormalise), scale, self._start(weights), self._start(indices), self._start(loads))

    def route_grad(self, score, dtype, m, n, x, stride, k, indices, dweights, renormalise, scale, dx, dx_stride):
        self._call(self.lib.dlfx_route_grad, "dlfx_route_grad", score.encode(), dtype, m, n, x.storage.data_ptr(), x.shape.offset, stride, k,
                   self._start(indices), self._start(dweights), int(renormalise), scale, dx.storage.data_ptr(), dx.shape.offset, dx_stride)

    def cross_entropy(self, dtype, index_dtype, m, n, x, stride, targets, z_loss, loss):
        sp, sb, keep = self._call_scratch(self.lib.dlfx_cross_entropy_scratch_bytes(dtype, m, n))
        self._call(self.lib.dlfx_cross_entropy, "dlfx_cross_entropy", dtype, index_dtype, m, n, x.storage.data_ptr(), x.shape.offset, stride,
                   self._start(targets), z_loss, self._start(loss), sp, sb)

    def cross_entropy_grad(self, dtype, index_dtype, m, n, x, stride, targets, weights, z_loss, loss, dx, dx_stride):
        sp, sb, keep = self._call_scratch(self.lib.dlfx_cross_entropy_scratch_bytes(dtype, m, n))
        self._call(self.lib.dlfx_cross_entropy_grad, "dlfx_cross_entropy_grad", dtype, index_dtype, m, n, x.storage.data_ptr(), x.shape.offset,
                   stride, self._start(targets), self._start(weights), z_loss, self._start(loss), dx.storage.data_ptr(), dx.shape.offset,
                   dx_stride, sp, sb)

    def cross_entropy_piece(self, dtype, index_dtype, m, n, x, stride, targets, first, resume, state):
        sp, sb, keep = self._call_scratch(self.lib.dlfx_cross_entropy_scratch_bytes(dtype, m, n))
        self._call(self.lib.dlfx_cross_entropy_piece, "dlfx_cross_entropy_piece", dtype, index_dtype, m, n, x.storage.data_ptr(), x.shape.offset,
                   stride, self._start(targets), first, int(resume), self._start(state), sp, sb)

    def cross_entropy_join(self, index_dtype, m, targets, state, z_loss, loss):
        self._call(self.lib.dlfx_cross_entropy_join, "dlfx_cross_entropy_join", index_dtype, m, self._start(targets), self._start(state), z_loss,
                   self._start(loss))

    def cross_entropy_piece_grad(self, dtype, index_dtype, m, n, x, stride, targets, first, state, weights, z_loss, dx, dx_stride):
        self._call(self.lib.dlfx_cross_entropy_piece_grad, "dlfx_cross_entropy_piece_grad", dtype, index_dtype, m, n, x.storage.data_ptr(),
                   x.shape.offset, stride, self._start(targets), first, self._start(state), self._start(weights), z_loss,
                   dx.storage.data_ptr(), dx.shape.offset, dx_stride)

    def read_element(self, storage, index):
        """One element of a device buffer on the host (synchronises the stream)."""
        return self._flat(storage)[index].item()

    def set_tuning(self, key: str, value: int):
        _check(self.lib.dlfx_set_tuning(key.encode(), value), "dlfx_set_tuning(%s)" % key)

    def synchronize(self):
        self.torch.cuda.synchronize(self.device)


_default = {}


def default_backend() -> HipBackend:
    """The backend of torch's current device, one per device and process."""
    import torch
    device = torch.cuda.current_device()
    if device not in _default:
        _default[device] = HipBackend("cuda:%d" % device)
    return _default[device]
