"""Operators of language models over libdcopy: rows moved and summed by index.

  embedding_lookup / embedding_grad     token ids -> rows of a table, and its gradient
  expert_sort                           a router's choices in expert order
  expert_dispatch / expert_combine      tokens to their experts' rows and back, weighted
  expert_combine_grad                   the gradient of the way back
  GradList, clip_grad_norm              global gradient norm and clipping

They take CUDA tensors and write into tensors the caller gives; shapes, types and row
pitches are read from the tensors (the last dimension must be dense).  Every buffer is
checked before a launch; launches go to ``stream``, by default torch's current stream of
the tensors' device.  A workspace that is not given is taken from torch's allocator.
``dcopy.torch_ops`` has the same as differentiable ``torch.ops.dcopy`` operators.
"""
from __future__ import annotations

import ctypes
from typing import Sequence

from . import DATA_TYPE, DcopyError, DcopyGrad, DcopyGradList, DcopyMatrix, _check, lib

__all__ = ["embedding_lookup", "embedding_grad", "embedding_grad_workspace", "expert_rows",
           "expert_sort", "expert_sort_workspace", "expert_dispatch", "expert_combine",
           "expert_combine_grad", "GradList", "grad_sum_squares", "grad_clip", "clip_grad_norm"]

_codes = {}


def _code(dtype) -> int:
    """The GE DataType of a torch dtype; -1 (refused by the library) for others."""
    if not _codes:
        import torch
        _codes.update({torch.float32: DATA_TYPE["FLOAT"], torch.float16: DATA_TYPE["FLOAT16"],
                       torch.bfloat16: DATA_TYPE["BF16"], torch.int32: DATA_TYPE["INT32"],
                       torch.int64: DATA_TYPE["INT64"], torch.int8: DATA_TYPE["INT8"],
                       torch.uint8: DATA_TYPE["UINT8"], torch.float8_e4m3fn: DATA_TYPE["UINT8"],
                       torch.float8_e5m2: DATA_TYPE["UINT8"]})
    return _codes.get(dtype, -1)


def _matrix(t, name: str) -> DcopyMatrix:
    """A tensor as rows of its last dimension; the other dimensions must step evenly."""
    if not t.is_cuda:
        raise ValueError(f"{name}: expected a CUDA tensor")
    shape, stride = t.shape, t.stride()
    if len(shape) == 2:
        rows, cols = shape
        pitch, unit = stride
    elif len(shape) < 2:
        rows, cols, pitch, unit = 1, t.numel(), 0, stride[0] if stride else 1
        if unit > 1:  # a strided vector: rows of one element
            rows, cols, pitch, unit = cols, 1, unit, 1
    else:
        cols, unit, pitch = shape[-1], stride[-1], stride[-2]
        rows = 1
        for n, step in zip(reversed(shape[:-1]), reversed(stride[:-1])):
            if n > 1 and rows > 1 and step != rows * pitch:
                raise ValueError(f"{name}: rows of shape {tuple(shape)} and strides {stride} do "
                                 "not lie at one pitch")
            if rows == 1 and n > 1:
                pitch = step
            rows *= n
    if unit != 1 and cols > 1:
        raise ValueError(f"{name}: the last dimension must be dense, its stride is {unit}")
    return DcopyMatrix(t.data_ptr(), rows, cols, pitch, _code(t.dtype), 0)


def _vector(t, name: str, dtype_name: str = "INT32"):
    """Address of a dense CUDA tensor of one type, or None."""
    if t is None:
        return None
    if not t.is_cuda or not t.is_contiguous() or _code(t.dtype) != DATA_TYPE[dtype_name]:
        raise ValueError(f"{name}: expected a contiguous CUDA tensor of type {dtype_name}")
    return t.data_ptr()


class _On:
    """The stream of a call: the given one or torch's current stream of the tensor's
    device, which is made current for the call when it is not."""
    __slots__ = ("stream", "raw", "guard", "device")

    def __init__(self, tensor, stream, others=()):
        import torch
        device = tensor.get_device()
        for t in others:
            if t is not None and t.get_device() != device:
                raise ValueError("tensors are on different devices")
        self.device = device
        self.stream = stream
        if stream is None:
            self.raw = torch._C._cuda_getCurrentRawStream(device) or None
        else:
            self.raw = (stream if isinstance(stream, int) else stream.cuda_stream) or None
        self.guard = None
        if torch._C._cuda_getDevice() != device:
            self.guard = torch.cuda.device(device)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()
        return self.raw

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)

    def scratch(self, nbytes: int):
        """Workspace from torch's allocator, kept from reuse until this call's stream is done."""
        import torch
        t = torch.empty(nbytes, dtype=torch.uint8, device=torch.device("cuda", self.device))
        if self.stream is not None:
            s = self.stream
            if isinstance(s, int):
                s = torch.cuda.ExternalStream(s, device=self.device)
            t.record_stream(s)
        return t


# ---- embedding ----------------------------------------------------------------------------


def embedding_lookup(out, table, ids, scale: float = 1.0, first_id: int = 0, stream=None) -> None:
    """out[i,:] = scale * table[ids[i] - first_id,:]; zero for ids outside the table."""
    o, t, i = _matrix(out, "out"), _matrix(table, "table"), _matrix(ids, "ids")
    with _On(out, stream, (table, ids)) as s:
        _check(lib().dcopy_embedding_lookup(ctypes.byref(o), ctypes.byref(t), ctypes.byref(i),
                                            first_id, scale, s), "dcopy_embedding_lookup")


def embedding_grad_workspace(tokens: int, vocab: int, width: int) -> int:
    """Bytes of embedding_grad's workspace."""
    n = ctypes.c_uint64(0)
    _check(lib().dcopy_embedding_grad_workspace(tokens, vocab, width, ctypes.byref(n)),
           "dcopy_embedding_grad_workspace")
    return n.value


def embedding_grad(grad, dout, ids, scale: float = 1.0, first_id: int = 0,
                   accumulate: bool = False, workspace=None, stream=None) -> None:
    """grad[v,:] = scale * sum of dout[i,:] over ids[i] - first_id == v, in the order of i
    (added to grad with accumulate); the same bits on every run."""
    g, d, i = _matrix(grad, "grad"), _matrix(dout, "dout"), _matrix(ids, "ids")
    on = _On(grad, stream, (dout, ids, workspace))
    with on as s:
        if workspace is None:
            workspace = on.scratch(embedding_grad_workspace(i.rows * i.cols, g.rows, g.cols))
        _check(lib().dcopy_embedding_grad(ctypes.byref(g), ctypes.byref(d), ctypes.byref(i),
                                          first_id, scale, 1 if accumulate else 0,
                                          workspace.data_ptr(), _bytes(workspace), s),
               "dcopy_embedding_grad")


def _bytes(t) -> int:
    if not t.is_contiguous():
        raise ValueError("workspace: expected a contiguous tensor")
    return t.numel() * t.element_size()


# ---- experts ------------------------------------------------------------------------------


def expert_rows(entries: int, experts: int, align: int = 1) -> int:
    """Rows that hold any routing of `entries` choices with segments padded to `align`."""
    n = ctypes.c_int64(0)
    _check(lib().dcopy_expert_rows(entries, experts, align, ctypes.byref(n)), "dcopy_expert_rows")
    return n.value


def expert_sort_workspace(entries: int, experts: int) -> int:
    """Bytes of expert_sort's workspace."""
    n = ctypes.c_uint64(0)
    _check(lib().dcopy_expert_sort_workspace(entries, experts, ctypes.byref(n)),
           "dcopy_expert_sort_workspace")
    return n.value


def expert_sort(dest, source, offsets, expert_ids, align: int = 1, workspace=None,
                stream=None) -> None:
    """dest (a row for each choice, -1 for ids outside the experts), source (the choice of
    each row, -1 for padding) and offsets (experts + 1 row numbers) of a router's choices."""
    i = _matrix(expert_ids, "expert_ids")
    n = i.rows * i.cols
    experts = offsets.numel() - 1
    d, so, of = _vector(dest, "dest"), _vector(source, "source"), _vector(offsets, "offsets")
    if dest.numel() != n:
        raise DcopyError(-2, f"dest has {dest.numel()} values for {n} choices", "dcopy_expert_sort")
    on = _On(dest, stream, (source, offsets, expert_ids, workspace))
    with on as s:
        if workspace is None:
            workspace = on.scratch(expert_sort_workspace(n, experts))
        _check(lib().dcopy_expert_sort(d, so, source.numel(), of, ctypes.byref(i), experts, align,
                                       workspace.data_ptr(), _bytes(workspace), s),
               "dcopy_expert_sort")


def _slots(dest, tokens: int, func: str) -> int:
    n = dest.numel()
    slots = dest.shape[-1] if dest.dim() > 1 else (n // tokens if tokens else 0)
    if slots * tokens != n:
        raise DcopyError(-2, f"dest has {n} values for {tokens} tokens", func)
    return slots


def _rows_source(source, rows: int, func: str):
    if source is not None and source.numel() != rows:
        raise DcopyError(-2, f"source has {source.numel()} values for {rows} rows", func)
    return _vector(source, "source")


def _weights(weights):
    return None if weights is None else ctypes.byref(_matrix(weights, "weights"))


def expert_dispatch(out, x, dest, source=None, weights=None, stream=None) -> None:
    """out[dest[i,j],:] = x[i,:] (times weights[i,j]); with source, other rows are zeroed."""
    o, m = _matrix(out, "out"), _matrix(x, "x")
    name = "dcopy_expert_dispatch"
    slots, d, so = _slots(dest, m.rows, name), _vector(dest, "dest"), _rows_source(source, o.rows, name)
    with _On(out, stream, (x, dest, source, weights)) as s:
        _check(lib().dcopy_expert_dispatch(ctypes.byref(o), ctypes.byref(m), d, slots, so,
                                           _weights(weights), s), name)


def expert_combine(out, y, dest, weights=None, stream=None) -> None:
    """out[i,:] = sum over j of (weights[i,j] *) y[dest[i,j],:]."""
    o, m = _matrix(out, "out"), _matrix(y, "y")
    name = "dcopy_expert_combine"
    slots, d = _slots(dest, o.rows, name), _vector(dest, "dest")
    with _On(out, stream, (y, dest, weights)) as s:
        _check(lib().dcopy_expert_combine(ctypes.byref(o), ctypes.byref(m), d, slots,
                                          _weights(weights), s), name)


def expert_combine_grad(dy, dweights, dout, y, dest, weights, source=None, stream=None) -> None:
    """dy[dest[i,j],:] = weights[i,j] * dout[i,:]; dweights[i,j] = <dout[i,:], y[dest[i,j],:]>."""
    gy, gw = _matrix(dy, "dy"), _matrix(dweights, "dweights")
    go, m, w = _matrix(dout, "dout"), _matrix(y, "y"), _matrix(weights, "weights")
    name = "dcopy_expert_combine_grad"
    slots, d, so = _slots(dest, go.rows, name), _vector(dest, "dest"), _rows_source(source, gy.rows, name)
    with _On(dy, stream, (dweights, dout, y, dest, weights, source)) as s:
        _check(lib().dcopy_expert_combine_grad(ctypes.byref(gy), ctypes.byref(gw), ctypes.byref(go),
                                               ctypes.byref(m), d, slots, so, ctypes.byref(w), s),
               name)


# ---- gradient norm and clipping -------------------------------------------------------------


class GradList:
    """Gradients laid out once for the norm and clipping kernels.

    ``grads`` are dense CUDA tensors (FLOAT, FLOAT16 or BF16, mixed as they come); clipped
    values go to ``out`` (same sizes, any of the types), by default in place.  The list keeps
    the tensors alive; gradients that move to other buffers need a new list.  Uses of one list
    follow one another on a stream.  Building it synchronises."""

    def __init__(self, grads: Sequence, out: Sequence = None, stream=None):
        import torch
        self._grads = list(grads)
        self._out = self._grads if out is None else list(out)
        if len(self._grads) != len(self._out):
            raise ValueError("out needs a tensor for each gradient")
        if not self._grads:
            raise ValueError("no gradients")
        arr = (DcopyGrad * len(self._grads))()
        for k, (g, o) in enumerate(zip(self._grads, self._out)):
            if not (g.is_cuda and o.is_cuda and g.is_contiguous() and o.is_contiguous()):
                raise ValueError(f"gradient {k}: expected contiguous CUDA tensors")
            if g.numel() != o.numel():
                raise ValueError(f"gradient {k}: {g.numel()} elements for {o.numel()}")
            arr[k] = DcopyGrad(g.data_ptr(), o.data_ptr(), g.numel(), _code(g.dtype), _code(o.dtype))
        n = ctypes.c_uint64(0)
        _check(lib().dcopy_grad_list_workspace(arr, len(arr), ctypes.byref(n)),
               "dcopy_grad_list_workspace")
        self._anchor = self._grads[0]
        self._space = torch.empty(n.value, dtype=torch.uint8, device=self._anchor.device)
        self._list = DcopyGradList()
        with _On(self._anchor, stream, self._grads + self._out) as s:
            _check(lib().dcopy_grad_list_build(ctypes.byref(self._list), arr, len(arr),
                                               self._space.data_ptr(), n.value, s),
                   "dcopy_grad_list_build")


def grad_sum_squares(total, grads: GradList, stream=None) -> None:
    """total[0] (fp64, CUDA) = the sum of squares over the list."""
    with _On(grads._anchor, stream, (total,)) as s:
        _check(lib().dcopy_grad_sum_squares(ctypes.byref(grads._list), _double(total), s),
               "dcopy_grad_sum_squares")


def grad_clip(grads: GradList, total, max_norm: float, norm=None, eps: float = 1e-6,
              stream=None) -> None:
    """Clips the list by the norm sqrt(total[0]); norm[0] (fp32, CUDA) gets it."""
    with _On(grads._anchor, stream, (total, norm)) as s:
        _check(lib().dcopy_grad_clip(ctypes.byref(grads._list), _double(total), max_norm, eps,
                                     _vector(norm, "norm", "FLOAT"), s), "dcopy_grad_clip")


def clip_grad_norm(grads: GradList, max_norm: float, norm=None, eps: float = 1e-6,
                   stream=None) -> None:
    """The list times min(1, max_norm / (norm + eps)); norm[0] (fp32, CUDA) gets the norm."""
    with _On(grads._anchor, stream, (norm,)) as s:
        _check(lib().dcopy_clip_grad_norm(ctypes.byref(grads._list), max_norm, eps,
                                          _vector(norm, "norm", "FLOAT"), s),
               "dcopy_clip_grad_norm")


def _double(t):
    import torch
    if not t.is_cuda or t.dtype != torch.float64 or t.numel() < 1:
        raise ValueError("total: expected a CUDA tensor of type float64")
    return t.data_ptr()
