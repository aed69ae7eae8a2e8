"""Host front-ends of the axis primitives, mirroring dlf's tensor API.

These functions do what dlf's header front-ends do before they reach the
``gpgpu::dnn`` boundary: normalise axes, build the moved-axis / transposed
strided view, size the output, then hand extents, strides, offsets and buffers
to a backend.  Reference: dlf/include/tensor/reduce.h:68-377,
reduce_detail.h:9-38,149-165, reorder.h:1120-1300.

A backend provides storage allocation and the six boundary calls; the shipped
backend is the HIP library (``dlf_amd.hip_backend``).
"""
from __future__ import annotations

from typing import List, Optional, Sequence, Tuple

import numpy as np

from .shape import Shape, ShapeError, norm_axes, norm_axis

# numpy has no bfloat16: its arrays are held as the bits, under a type of their own
BFLOAT16 = np.dtype([("bfloat16", np.uint16)])

DTYPE_CODES = {np.dtype(np.float32): 0, np.dtype(np.float64): 1,
               np.dtype(np.int32): 2, np.dtype(np.int64): 3,
               np.dtype(np.float16): 4, np.dtype(np.int16): 5, np.dtype(np.bool_): 6,
               np.dtype(np.complex64): 7, np.dtype(np.complex128): 8, BFLOAT16: 9}

REDUCE_NAMES = ("reduce_sum", "reduce_mean", "reduce_max", "reduce_min", "reduce_log_sum_exp",
                "reduce_sum_exp", "reduce_log_sum", "reduce_prod", "reduce_asum",
                "reduce_sum_square", "reduce_nrm2", "reduce_amax", "reduce_amin")
SCAN_NAMES = ("cumsum", "cumprod", "cummax", "cummin")


def dtype_code(dtype) -> int:
    try:
        return DTYPE_CODES[np.dtype(dtype)]
    except KeyError:
        raise TypeError("unsupported element type %r" % (dtype,))


def to_bfloat16(array) -> np.ndarray:
    """A float array as BFLOAT16, rounded to nearest, ties to even (a NaN stays one)."""
    bits = np.ascontiguousarray(array, dtype=np.float32).view(np.uint32)
    rounded = ((bits + np.uint32(0x7fff) + ((bits >> np.uint32(16)) & np.uint32(1))) >> np.uint32(16)).astype(np.uint16)
    quiet = ((bits >> np.uint32(16)) | np.uint32(0x40)).astype(np.uint16)
    nan = (bits & np.uint32(0x7fffffff)) > np.uint32(0x7f800000)
    return np.ascontiguousarray(np.where(nan, quiet, rounded)).view(BFLOAT16)


def from_bfloat16(array: np.ndarray) -> np.ndarray:
    """A BFLOAT16 array as float32 (exact)."""
    return (np.ascontiguousarray(array).view(np.uint16).astype(np.uint32) << np.uint32(16)).view(np.float32)


class Tensor:
    """A shape plus backend storage; views share storage (TensorView / DevTensorView)."""

    def __init__(self, backend, shape: Shape, storage, dtype):
        self.backend = backend
        self.shape = shape
        self.storage = storage
        self.dtype = np.dtype(dtype)

    # -- construction -------------------------------------------------------
    @classmethod
    def empty(cls, backend, extents: Sequence[int], dtype) -> "Tensor":
        shape = Shape(extents)
        return cls(backend, shape, backend.alloc(np.dtype(dtype), shape.size), dtype)

    @classmethod
    def from_numpy(cls, backend, array: np.ndarray) -> "Tensor":
        array = np.ascontiguousarray(array)
        shape = Shape(array.shape if array.ndim else ())
        return cls(backend, shape, backend.upload(array.reshape(-1)), array.dtype)

    # -- queries ------------------------------------------------------------
    @property
    def rank(self) -> int:
        return self.shape.rank

    @property
    def size(self) -> int:
        return self.shape.size

    def extent(self, i: int) -> int:
        return self.shape.extents[i]

    def numpy(self) -> np.ndarray:
        """Host copy of the viewed elements (``DevTensor::read``)."""
        flat = self.backend.download(self.storage)
        sh = self.shape
        item = flat.dtype.itemsize
        view = np.lib.stride_tricks.as_strided(
            flat[sh.offset:], shape=sh.extents, strides=[s * item for s in sh.strides], writeable=False)
        return np.array(view)

    # -- views --------------------------------------------------------------
    def view(self, shape: Shape) -> "Tensor":
        return Tensor(self.backend, shape, self.storage, self.dtype)

    def transpose(self, perm: Optional[Sequence[int]] = None) -> "Tensor":
        return self.view(self.shape.transpose(perm))

    def slice(self, starts, ends, axes=None, steps=None) -> "Tensor":
        return self.view(self.shape.slice(starts, ends, axes, steps))

    def moveaxis(self, source: int, destination: int) -> "Tensor":
        return self.view(self.shape.moveaxis(source, destination))

    def flip(self, axes=None) -> "Tensor":
        return self.view(self.shape.flip(axes))

    def contiguous(self) -> "Tensor":
        """The viewed elements in row-major order in storage of their own (the reference's
        reorder(X, Y)); on the device when the backend can copy a strided view there."""
        copy = getattr(self.backend, "copy_view", None)
        if copy is not None:
            return Tensor(self.backend, Shape(list(self.shape.extents)), copy(self.storage, self.shape), self.dtype)
        return Tensor.from_numpy(self.backend, self.numpy())


# ---------------------------------------------------------------------------
# reduce (reduce.h:68-129, reduce_detail.h:9-38,91-101)

def prepare_reduce(x_shape: Shape, axes: Sequence[int], keepdims: bool) -> Tuple[Shape, List[int], int, int]:
    """Returns (transposed view, output extents, m, n)."""
    rank = x_shape.rank
    axes = norm_axes(rank, axes, True)
    reduced = set(range(rank)) if not axes else set(axes)
    out_dims, perm = [], []
    m = n = 1
    for i in range(rank):
        if i not in reduced:
            out_dims.append(x_shape.extents[i])
            perm.append(i)
        elif keepdims:
            out_dims.append(1)
    for i in range(rank):
        if i in reduced:
            perm.append(i)
            n *= x_shape.extents[i]
        else:
            m *= x_shape.extents[i]
    return x_shape.transpose(perm), out_dims, m, n


def reduce(name: str, X: Tensor, axes: Sequence[int] = (), keepdims: bool = False) -> Tensor:
    if isinstance(axes, int):
        axes = [axes]
    view, out_dims, m, n = prepare_reduce(X.shape, list(axes), keepdims)
    Y = Tensor.empty(X.backend, out_dims, X.dtype)
    X.backend.reduce(name, dtype_code(X.dtype), m, n, view, X.storage, Y.shape, Y.storage)
    return Y


def count(X: Tensor, value, axes: Sequence[int] = (), keepdims: bool = False) -> Tensor:
    """Number of elements equal to `value` over `axes` (reduce.h:160-198); int32 result."""
    if isinstance(axes, int):
        axes = [axes]
    view, out_dims, m, n = prepare_reduce(X.shape, list(axes), keepdims)
    Y = Tensor.empty(X.backend, out_dims, np.int32)
    X.backend.count(dtype_code(X.dtype), m, n, value, view, X.storage, Y.shape, Y.storage)
    return Y


def nonzero(X: Tensor, row_major: bool = False) -> Optional[Tensor]:
    """Coordinates of the non-zero elements (reduce.h:419-450): an [n, rank] int32 tensor, or
    [rank, n] when row_major; None when there is none (the reference clears the output)."""
    size = X.size
    counts = Tensor.empty(X.backend, [size], np.int32)
    counts_shape = Shape(X.shape.extents)           # contiguous, the input's extents
    X.backend.scan_nonzero(dtype_code(X.dtype), 1, size, False,
                           _as_row(X.shape), X.storage, _as_row(counts_shape), counts.storage)
    n = int(X.backend.read_element(counts.storage, size - 1))
    if n == 0:
        return None
    rank = X.rank
    Y = Tensor.empty(X.backend, [rank, n] if row_major else [n, rank], np.int32)
    X.backend.gather_indices(size, n, row_major, list(X.shape.extents), counts.storage, Y.storage)
    return Y


def _as_row(shape: Shape) -> Shape:
    """The view itself: scan_nonzero(1, size, ...) walks all of it as one row, in row-major
    order of the extents, which is how the reference passes it (reduce.h:426-429)."""
    return shape


def _make_reduce(name):
    def f(X: Tensor, axes: Sequence[int] = (), keepdims: bool = False) -> Tensor:
        return reduce(name, X, axes, keepdims)
    f.__name__ = name
    f.__doc__ = "dlf::%s (reduce.h:84-129)" % name
    return f


for _n in REDUCE_NAMES:
    globals()[_n] = _make_reduce(_n)


# ---------------------------------------------------------------------------
# argmax / argmin (reduce.h:204-234, reduce_detail.h:149-165)

def arg_reduce(name: str, X: Tensor, axis: int, keepdims: bool = True, index_dtype=np.int32) -> Tensor:
    axis = norm_axis(X.rank, axis)
    y_dims = list(X.shape.extents)
    if keepdims:
        y_dims[axis] = 1
    else:
        del y_dims[axis]
    view = X.shape.moveaxis(axis, -1)
    Y = Tensor.empty(X.backend, y_dims, index_dtype)
    k = view.extents[-1]
    X.backend.arg_reduce(name, dtype_code(X.dtype), dtype_code(index_dtype), view.size // k, k,
                         view, X.storage, Y.shape, Y.storage)
    return Y


def argmax(X: Tensor, axis: int, keepdims: bool = True, index_dtype=np.int32) -> Tensor:
    return arg_reduce("argmax", X, axis, keepdims, index_dtype)


def argmin(X: Tensor, axis: int, keepdims: bool = True, index_dtype=np.int32) -> Tensor:
    return arg_reduce("argmin", X, axis, keepdims, index_dtype)


# ---------------------------------------------------------------------------
# scan (reduce.h:240-377)

def scan(name: str, X: Tensor, axis: int = -1, exclusive: bool = False, reverse: bool = False,
         out: Optional[Tensor] = None) -> Tensor:
    axis = norm_axis(X.rank, axis)
    n = X.shape.extents[axis]
    m = X.size // n
    Y = out if out is not None else Tensor.empty(X.backend, X.shape.extents, X.dtype)
    if Y.shape.extents != X.shape.extents or Y.dtype != X.dtype:
        raise ShapeError("scan: output does not match input")
    xs = X.shape.moveaxis(axis, -1)
    ys = Y.shape.moveaxis(axis, -1)
    if reverse:
        xs = xs.flip([-1])
        ys = ys.flip([-1])
    X.backend.scan(name, dtype_code(X.dtype), m, n, exclusive, xs, X.storage, ys, Y.storage)
    return Y


def cumsum(X, axis=-1, exclusive=False, reverse=False, out=None):
    return scan("cumsum", X, axis, exclusive, reverse, out)


def cumprod(X, axis=-1, exclusive=False, reverse=False, out=None):
    return scan("cumprod", X, axis, exclusive, reverse, out)


def cummax(X, axis=-1, reverse=False, out=None):
    return scan("cummax", X, axis, False, reverse, out)


def cummin(X, axis=-1, reverse=False, out=None):
    return scan("cummin", X, axis, False, reverse, out)


# ---------------------------------------------------------------------------
# sort / argsort / top_k (reorder.h:1120-1300)

def _copy_into(X: Tensor, Y: Tensor) -> None:
    Y.storage = X.backend.upload(X.numpy().reshape(-1))
    Y.shape = Shape(X.shape.extents)


def sort(X: Tensor, axis: int = -1, descending: bool = False, out: Optional[Tensor] = None) -> Tensor:
    axis = norm_axis(X.rank, axis)
    Y = out if out is not None else Tensor.empty(X.backend, X.shape.extents, X.dtype)
    if X.shape.extents[axis] > 1:
        xs, ys = X.shape.moveaxis(axis, -1), Y.shape.moveaxis(axis, -1)
        X.backend.sort(int(descending), dtype_code(X.dtype), xs, X.storage, ys, Y.storage)
    elif Y is not X:
        _copy_into(X, Y)
    return Y


def argsort(X: Tensor, axis: int = -1, descending: bool = False, values: Optional[Tensor] = None,
            index_dtype=np.int32, with_values: bool = False):
    """Index-only argsort returns I; with ``values`` (or with_values) returns (Y, I)."""
    axis = norm_axis(X.rank, axis)
    I = Tensor.empty(X.backend, X.shape.extents, index_dtype)
    Y = values
    if Y is None and with_values:
        Y = Tensor.empty(X.backend, X.shape.extents, X.dtype)
    if X.shape.extents[axis] > 1:
        xs, is_ = X.shape.moveaxis(axis, -1), I.shape.moveaxis(axis, -1)
        ys = Y.shape.moveaxis(axis, -1) if Y is not None else None
        X.backend.argsort(int(descending), dtype_code(X.dtype), dtype_code(index_dtype), xs, X.storage,
                          ys, Y.storage if Y is not None else None, is_, I.storage)
    else:
        if Y is not None and Y is not X:
            _copy_into(X, Y)
        I.storage = X.backend.upload(np.zeros(I.size, dtype=index_dtype))
    return (Y, I) if Y is not None else I


def top_k(X: Tensor, k: int, axis: int = -1, largest: bool = True, index_dtype=np.int32):
    axis = norm_axis(X.rank, axis)
    k = min(int(k), X.shape.extents[axis])
    out_dims = list(X.shape.extents)
    out_dims[axis] = k
    Y = Tensor.empty(X.backend, out_dims, X.dtype)
    I = Tensor.empty(X.backend, out_dims, index_dtype)
    xs, ys, is_ = X.shape.moveaxis(axis, -1), Y.shape.moveaxis(axis, -1), I.shape.moveaxis(axis, -1)
    X.backend.top_k(k, int(largest), dtype_code(X.dtype), dtype_code(index_dtype),
                    xs, X.storage, ys, Y.storage, is_, I.storage)
    return Y, I


def merge(A: Tensor, B: Tensor, axis: int = -1, descending: bool = False, out: Optional[Tensor] = None) -> Tensor:
    """Merges two tensors sorted along `axis` into one sorted tensor (reorder.h:1061-1114):
    the other extents must agree; equal elements keep A's before B's."""
    rank = A.rank
    if B.rank != rank:
        raise ShapeError("merge: incompatible shape")
    axis = norm_axis(rank, axis)
    dims = []
    for i in range(rank):
        if i == axis:
            dims.append(A.extent(i) + B.extent(i))
        elif A.extent(i) != B.extent(i):
            raise ShapeError("merge: incompatible shape")
        else:
            dims.append(A.extent(i))
    C = out if out is not None else Tensor.empty(A.backend, dims, A.dtype)
    if list(C.shape.extents) != dims:
        raise ShapeError("merge: output shape")
    a, b, c = A.shape.moveaxis(axis, -1), B.shape.moveaxis(axis, -1), C.shape.moveaxis(axis, -1)
    A.backend.merge(1 if descending else 0, dtype_code(A.dtype), a, A.storage, b, B.storage, c, C.storage)
    return C


def _softmax_family(name: str, X: Tensor, axis: int) -> Tensor:
    """dlf/include/tensor/dnn.h:447-531: the tensor is flattened to [m, n] with m the product
    of the extents before `axis` (default 1) and each row is normalised.  A non-contiguous
    input is copied first, as the reference's reorder(X, Y) does."""
    axis = norm_axis(X.rank, axis)
    m = 1
    for i in range(axis):
        m *= X.extent(i)
    n = X.size // m
    src = X if X.shape.is_contiguous() else X.contiguous()
    Y = Tensor.empty(X.backend, list(X.shape.extents), X.dtype)
    X.backend.softmax(name, dtype_code(X.dtype), m, n, src.storage, src.shape.offset, Y.storage, 0)
    return Y


def softmax(X: Tensor, axis: int = 1) -> Tensor:
    return _softmax_family("softmax", X, axis)


def logsoftmax(X: Tensor, axis: int = 1) -> Tensor:
    return _softmax_family("logsoftmax", X, axis)


def hardmax(X: Tensor, axis: int = 1) -> Tensor:
    return _softmax_family("hardmax", X, axis)


def gather_elements(X: np.ndarray, I: np.ndarray, axis: int) -> np.ndarray:
    """Host helper of the reference's property tests (reorder_detail.h:190-207)."""
    return np.take_along_axis(X, I.astype(np.int64), axis=axis)


# ---------------------------------------------------------------------------
# sequence-model operators (no counterpart in the reference)

GATE_KINDS = ("gated", "gated_exp", "gated_sigmoid", "gated_blend")
SCORE_KINDS = ("softmax", "sigmoid")
SEQUENCE_DTYPES = (np.dtype(np.float32), np.dtype(np.float16), BFLOAT16)


def _sequence_dtype(where: str, X: Tensor) -> int:
    if X.dtype not in SEQUENCE_DTYPES:
        raise TypeError("%s: float32, float16 or bfloat16 elements, not %r" % (where, X.dtype))
    return DTYPE_CODES[X.dtype]


def _together(where: str, *tensors: Optional[Tensor]) -> None:
    for T in tensors[1:]:
        if T is not None and T.backend is not tensors[0].backend:
            raise ValueError("%s: tensors of different backends" % where)


def _like(where: str, what: str, T: Tensor, extents: tuple, dtype) -> Tensor:
    if T.shape.extents != extents:
        raise ShapeError("%s: %s has extents %s, not %s" % (where, what, list(T.shape.extents), list(extents)))
    if T.dtype != dtype:
        raise TypeError("%s: %s has element type %r, not %r" % (where, what, T.dtype, np.dtype(dtype)))
    return T


def _along(T: Tensor, axis: int, reverse: bool):
    """(storage, offset, strides) of the view with `axis` last, from its other end when reverse."""
    sh = T.shape
    st, step = sh.strides, sh.strides[axis]
    offset = sh.offset
    if reverse:
        offset += (sh.extents[axis] - 1) * step
        step = -step
    return T.storage, offset, st[:axis] + st[axis + 1:] + (step,)


def _new(like: Tensor, extents: tuple, dtype) -> Tensor:
    if extents and min(extents) <= 0:
        raise ShapeError("extent must be positive")
    return like.backend.new(extents, dtype)


def gated_scan(G: Tensor, X: Tensor, axis: int = -1, kind: str = "gated", reverse: bool = False,
               initial: Optional[Tensor] = None, last: Optional[Tensor] = None, out: Optional[Tensor] = None):
    """The gated linear recurrence along `axis` (reverse: from its last element): returns (Y, last).

    kind "gated": h = g h + x; "gated_exp": h = exp(g) h + x; "gated_sigmoid": h = s(g) h + x;
    "gated_blend": h = s(g) h + (1 - s(g)) x, s the logistic function.  The state is fp32: `initial`
    (None: zeros) and `last` have X's extents without `axis`; `last` may be the tensor given as
    `initial` (a decoding step updates its state in place).  G may share gates through strides of 0;
    `out` may be X or G."""
    where = "gated_scan(%s)" % kind
    if kind not in GATE_KINDS:
        raise ValueError("%s: kind is one of %s" % (where, ", ".join(GATE_KINDS)))
    code = _sequence_dtype(where, X)
    _together(where, X, G, initial, last, out)
    axis = norm_axis(X.rank, axis)
    extents = X.shape.extents
    kept = extents[:axis] + extents[axis + 1:]
    _like(where, "the gate", G, extents, X.dtype)
    Y = _like(where, "out", out, extents, X.dtype) if out is not None else _new(X, extents, X.dtype)
    if initial is not None:
        _like(where, "initial", initial, kept, np.float32)
    L = _like(where, "last", last, kept, np.float32) if last is not None else _new(X, kept, np.float32)
    X.backend.gated_scan(kind, code, kept + (extents[axis],), _along(G, axis, reverse), _along(X, axis, reverse), initial,
                         _along(Y, axis, reverse), L)
    return Y, L


def gated_scan_grad(G: Tensor, X: Optional[Tensor], Y: Tensor, dY: Tensor, axis: int = -1, kind: str = "gated", reverse: bool = False,
                    initial: Optional[Tensor] = None, dlast: Optional[Tensor] = None):
    """Gradients (dG, dX, dinitial) of gated_scan for dY and dlast (None: zeros), from the Y that it
    returned.  Only "gated_blend" reads X (None otherwise will do).  dG has every element of X's
    extents: where G shares a gate, sum it over the shared axes (reduce_sum; for bfloat16, which that does
    not take, the last state of gated_scan(one, dG, axis) with gates of 1, a single one under strides of
    0 will do, is the sum in fp32)."""
    where = "gated_scan_grad(%s)" % kind
    if kind not in GATE_KINDS:
        raise ValueError("%s: kind is one of %s" % (where, ", ".join(GATE_KINDS)))
    code = _sequence_dtype(where, Y)
    _together(where, Y, G, X, dY, initial, dlast)
    axis = norm_axis(Y.rank, axis)
    extents = Y.shape.extents
    kept = extents[:axis] + extents[axis + 1:]
    _like(where, "the gate", G, extents, Y.dtype)
    _like(where, "dY", dY, extents, Y.dtype)
    if X is not None:
        _like(where, "X", X, extents, Y.dtype)
    elif kind == "gated_blend":
        raise ValueError("%s: X is needed" % where)
    for what, T in (("initial", initial), ("dlast", dlast)):
        if T is not None:
            _like(where, what, T, kept, np.float32)
    dG, dX = _new(Y, extents, Y.dtype), _new(Y, extents, Y.dtype)
    dI = _new(Y, kept, np.float32)
    views = [_along(T, axis, reverse) if T is not None else None for T in (G, X, Y, dY, dG, dX)]
    Y.backend.gated_scan_grad(kind, code, kept + (extents[axis],), *views, initial, dlast, dI)
    return dG, dX, dI


def _rows(X: Tensor):
    """(tensor, m, n, row stride) with the last axis contiguous and every other axis merged into
    rows at one stride; a view that has no such form is copied first."""
    sh = X.shape
    if sh.rank == 0:
        raise ShapeError("rows along the last axis: the tensor has none")
    n = sh.extents[-1]
    m = sh.size // n
    if sh.strides[-1] == 1 or n == 1:
        stride = size = None
        for e, s in zip(reversed(sh.extents[:-1]), reversed(sh.strides[:-1])):
            if e == 1:
                continue
            if stride is None:
                stride, size = s, e
            elif s == stride * size:
                size *= e
            else:
                break
        else:
            if stride is None:
                return X, m, n, n
            if stride >= n:
                return X, m, n, stride
    return X.contiguous(), m, n, n


def _rows_of_output(where: str, X: Tensor, out: Optional[Tensor]):
    if out is None:
        out = _new(X, X.shape.extents, X.dtype)
    _like(where, "out", out, X.shape.extents, X.dtype)
    direct, _, _, stride = _rows(out)
    if direct is not out:
        raise ShapeError("%s: out must have a contiguous last axis and rows at one stride" % where)
    return out, stride


def _dense(T: Optional[Tensor]) -> Optional[Tensor]:
    return T if T is None or T.shape.is_contiguous() else T.contiguous()


def _score_kind(where: str, score: str) -> None:
    if score not in SCORE_KINDS:
        raise ValueError("%s: score is one of %s" % (where, ", ".join(SCORE_KINDS)))


def route(X: Tensor, k: int, score: str = "softmax", bias: Optional[Tensor] = None, groups: int = 1, kept_groups: Optional[int] = None,
          group_best: int = 1, renormalise: bool = False, scale: float = 1.0, loads: Optional[Tensor] = None):
    """The k experts of every row of router logits (experts on the last axis): (weights fp32, indices int32),
    both with k in place of the experts, best first.

    The score is the row's softmax or logistic function; experts are chosen by score + bias (fp32, one per
    expert), weighed by scale * score, renormalised over the chosen ones on request.  With groups > 1 only the
    kept_groups groups (neighbouring experts) with the largest sums of their group_best (1 or 2) best choices
    take part.  loads (int32, one per expert): the number of rows that took each expert is added to it.
    -inf or the type's lowest value masks an expert."""
    where = "route(%s)" % score
    _score_kind(where, score)
    code = _sequence_dtype(where, X)
    _together(where, X, bias, loads)
    rows, m, n, stride = _rows(X)
    if bias is not None:
        _like(where, "bias", bias, (n,), np.float32)
    if loads is not None:
        _like(where, "loads", loads, (n,), np.int32)
        if not loads.shape.is_contiguous():
            raise ShapeError("%s: loads must be contiguous" % where)
    k = int(k)
    dims = X.shape.extents[:-1] + (k,)
    W, I = _new(X, dims, np.float32), _new(X, dims, np.int32)
    X.backend.route(score, code, m, n, rows, stride, _dense(bias), int(groups), int(groups if kept_groups is None else kept_groups),
                    int(group_best), k, bool(renormalise), float(scale), W, I, loads)
    return W, I


def route_grad(X: Tensor, indices: Tensor, dweights: Tensor, score: str = "softmax", renormalise: bool = False, scale: float = 1.0,
               out: Optional[Tensor] = None) -> Tensor:
    """Gradient of the logits X for the gradient of route's weights, at the choice `indices` (both with k on the
    last axis).  out may be X."""
    where = "route_grad(%s)" % score
    _score_kind(where, score)
    code = _sequence_dtype(where, X)
    _together(where, X, indices, dweights, out)
    rows, m, n, stride = _rows(X)
    if indices.rank < 1:
        raise ShapeError("%s: indices have no axis of choices" % where)
    dims = X.shape.extents[:-1] + (indices.shape.extents[-1],)
    _like(where, "indices", indices, dims, np.int32)
    _like(where, "dweights", dweights, dims, np.float32)
    dX, dx_stride = _rows_of_output(where, X, out)
    X.backend.route_grad(score, code, m, n, rows, stride, dims[-1], _dense(indices), _dense(dweights), bool(renormalise), float(scale),
                         dX, dx_stride)
    return dX


def _targets_of(where: str, X: Tensor, targets: Tensor) -> Tensor:
    if targets.dtype not in (np.dtype(np.int32), np.dtype(np.int64)):
        raise TypeError("%s: targets are int32 or int64, not %r" % (where, targets.dtype))
    return _dense(_like(where, "targets", targets, X.shape.extents[:-1], targets.dtype))


def _weights_of(where: str, X: Tensor, weights: Optional[Tensor]) -> Optional[Tensor]:
    return _dense(_like(where, "weights", weights, X.shape.extents[:-1], np.float32)) if weights is not None else None


def cross_entropy(X: Tensor, targets: Tensor, z_loss: float = 0.0) -> Tensor:
    """Softmax cross entropy (fp32) of every row of logits against its target column: lse - x[target] +
    z_loss lse^2, lse the logarithm of the row's sum of exponentials.  The last axis is the vocabulary;
    targets (int32, int64) have the other extents, a negative one takes its row out (loss 0)."""
    where = "cross_entropy"
    code = _sequence_dtype(where, X)
    _together(where, X, targets)
    rows, m, n, stride = _rows(X)
    t = _targets_of(where, X, targets)
    loss = _new(X, X.shape.extents[:-1], np.float32)
    X.backend.cross_entropy(code, dtype_code(t.dtype), m, n, rows, stride, t, float(z_loss), loss)
    return loss


def cross_entropy_grad(X: Tensor, targets: Tensor, weights: Optional[Tensor] = None, z_loss: float = 0.0, out: Optional[Tensor] = None):
    """(loss, gradient of the logits) of the sum of weights * loss over the rows (weights fp32, None: ones), from one
    call.  out may be X."""
    where = "cross_entropy_grad"
    code = _sequence_dtype(where, X)
    _together(where, X, targets, weights, out)
    rows, m, n, stride = _rows(X)
    t, w = _targets_of(where, X, targets), _weights_of(where, X, weights)
    loss = _new(X, X.shape.extents[:-1], np.float32)
    dX, dx_stride = _rows_of_output(where, X, out)
    X.backend.cross_entropy_grad(code, dtype_code(t.dtype), m, n, rows, stride, t, w, float(z_loss), loss, dX, dx_stride)
    return loss, dX


def cross_entropy_piece(X: Tensor, targets: Tensor, first: int, state: Optional[Tensor] = None) -> Tensor:
    """Folds the logits of columns first, first + 1, ... of a larger vocabulary into the rows' state (None: a new
    one): [3, rows] fp32, the maxima, the sums of exp(x - maximum), the targets' logits.  Returns the state."""
    where = "cross_entropy_piece"
    code = _sequence_dtype(where, X)
    _together(where, X, targets, state)
    rows, m, n, stride = _rows(X)
    t = _targets_of(where, X, targets)
    resume = state is not None
    state = _state_of(where, m, state) if resume else _new(X, (3, m), np.float32)
    X.backend.cross_entropy_piece(code, dtype_code(t.dtype), m, n, rows, stride, t, int(first), resume, state)
    return state


def _state_of(where: str, m: int, state: Tensor) -> Tensor:
    _like(where, "the state", state, (3, m), np.float32)
    if not state.shape.is_contiguous():
        raise ShapeError("%s: the state must be contiguous" % where)
    return state


def cross_entropy_join(state: Tensor, targets: Tensor, z_loss: float = 0.0) -> Tensor:
    """The rows' losses from the state, once every piece of the vocabulary has gone by."""
    where = "cross_entropy_join"
    _together(where, state, targets)
    if targets.dtype not in (np.dtype(np.int32), np.dtype(np.int64)):
        raise TypeError("%s: targets are int32 or int64, not %r" % (where, targets.dtype))
    t = _dense(targets)
    _state_of(where, t.size, state)
    loss = _new(state, targets.shape.extents, np.float32)
    state.backend.cross_entropy_join(dtype_code(t.dtype), t.size, t, state, float(z_loss), loss)
    return loss


def cross_entropy_piece_grad(X: Tensor, targets: Tensor, first: int, state: Tensor, weights: Optional[Tensor] = None, z_loss: float = 0.0,
                             out: Optional[Tensor] = None) -> Tensor:
    """Gradient of a piece's logits from the finished state; see cross_entropy_grad.  out may be X."""
    where = "cross_entropy_piece_grad"
    code = _sequence_dtype(where, X)
    _together(where, X, targets, state, weights, out)
    rows, m, n, stride = _rows(X)
    t, w = _targets_of(where, X, targets), _weights_of(where, X, weights)
    _state_of(where, m, state)
    dX, dx_stride = _rows_of_output(where, X, out)
    X.backend.cross_entropy_piece_grad(code, dtype_code(t.dtype), m, n, rows, stride, t, int(first), state, w, float(z_loss), dX, dx_stride)
    return dX
