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

The calls go through the extension module ``_tensor_calls`` (binding/tensor_calls.cpp),
which the build makes beside libdcopy.so.  Refusals raise ``DcopyError`` with the
library's status, tensors of the wrong kind or layout ``ValueError``.
"""
from __future__ import annotations

import ctypes
from typing import Sequence

from . import DcopyError, DcopyGrad, DcopyGradList, DcopyUnavailable, _check, lib

__all__ = ["embedding_lookup", "embedding_grad", "embedding_grad_workspace", "expert_rows",
           "expert_sort", "expert_sort_workspace", "expert_dispatch", "expert_combine",
           "expert_combine_grad", "GradList", "grad_sum_squares", "grad_clip", "clip_grad_norm"]


class _Loader:
    """Stands for the extension module until the first call: torch is loaded only then."""

    def __getattr__(self, name):
        global _calls
        import torch  # noqa: F401  (the module's symbols come from torch's libraries)
        try:
            from . import _tensor_calls as module
        except ImportError as exc:
            raise DcopyUnavailable(f"dcopy._tensor_calls is not built ({exc}); run "
                                   "__graft_entry__.build()") from exc
        handle = lib()
        names = ("dcopy_last_error_message", "dcopy_embedding_lookup", "dcopy_embedding_grad",
                 "dcopy_embedding_grad_workspace", "dcopy_expert_sort",
                 "dcopy_expert_sort_workspace", "dcopy_expert_dispatch", "dcopy_expert_combine",
                 "dcopy_expert_combine_grad", "dcopy_grad_sum_squares", "dcopy_grad_clip",
                 "dcopy_clip_grad_norm")
        module.bind({n: ctypes.cast(getattr(handle, n), ctypes.c_void_p).value for n in names},
                    DcopyError)
        _calls = module
        return getattr(module, name)


_calls = _Loader()


# ---- embedding ----------------------------------------------------------------------------


def embedding_lookup(out, table, ids, scale: float = 1.0, first_id: int = 0, stream=None) -> None:
    """out[i,:] = scale * table[ids[i] - first_id,:]; zero for ids outside the table."""
    _calls.embedding_lookup(out, table, ids, scale, first_id, stream)


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
    _calls.embedding_grad(grad, dout, ids, scale, first_id, accumulate, workspace, stream)


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
    _calls.expert_sort(dest, source, offsets, expert_ids, align, workspace, stream)


def expert_dispatch(out, x, dest, source=None, weights=None, stream=None) -> None:
    """out[dest[i,j],:] = x[i,:] (times weights[i,j]); with source, other rows are zeroed."""
    _calls.expert_dispatch(out, x, dest, source, weights, stream)


def expert_combine(out, y, dest, weights=None, stream=None) -> None:
    """out[i,:] = sum over j of (weights[i,j] *) y[dest[i,j],:]."""
    _calls.expert_combine(out, y, dest, weights, stream)


def expert_combine_grad(dy, dweights, dout, y, dest, weights, source=None, stream=None) -> None:
    """dy[dest[i,j],:] = weights[i,j] * dout[i,:]; dweights[i,j] = <dout[i,:], y[dest[i,j],:]>."""
    _calls.expert_combine_grad(dy, dweights, dout, y, dest, weights, source, stream)


# ---- gradient norm and clipping -------------------------------------------------------------


class GradList:
    """Gradients laid out once for the norm and clipping kernels.

    ``grads`` are dense CUDA tensors (FLOAT, FLOAT16 or BF16, mixed as they come); clipped
    values go to ``out`` (same sizes, any of the types), by default in place.  The list keeps
    the tensors alive; gradients that move to other buffers need a new list.  Uses of one list
    follow one another on a stream.  Building it synchronises.

    A list may be dropped while its last use still runs, on any stream: the memory that it
    held is not handed out before the streams it was used on are done with it."""

    def __init__(self, grads: Sequence, out: Sequence = None, stream=None):
        import torch
        grads = list(grads)
        out = grads if out is None else list(out)
        if not grads:
            raise ValueError("no gradients")
        arr = (DcopyGrad * len(grads))()
        device = _calls.fill_grads(ctypes.addressof(arr), grads, out)
        n = ctypes.c_uint64(0)
        _check(lib().dcopy_grad_list_workspace(arr, len(arr), ctypes.byref(n)),
               "dcopy_grad_list_workspace")
        self._list = DcopyGradList()
        self._space, handle = _calls.scratch(n.value, device, stream)
        with torch.cuda.device(device):
            _check(lib().dcopy_grad_list_build(ctypes.byref(self._list), arr, len(arr),
                                               self._space.data_ptr(), n.value, handle),
                   "dcopy_grad_list_build")
        kept = [self._space] + grads + (out if out is not grads else [])
        self._record = (ctypes.addressof(self._list), device, kept, {handle})


def grad_sum_squares(total, grads: GradList, stream=None) -> None:
    """total[0] (fp64, CUDA) = the sum of squares over the list."""
    _calls.grad_sum_squares(grads._record, total, stream)


def grad_clip(grads: GradList, total, max_norm: float, norm=None, eps: float = 1e-6,
              stream=None) -> None:
    """Clips the list by the norm sqrt(total[0]); norm[0] (fp32, CUDA) gets it."""
    _calls.grad_clip(grads._record, total, max_norm, eps, norm, stream)


def clip_grad_norm(grads: GradList, max_norm: float, norm=None, eps: float = 1e-6,
                   stream=None) -> None:
    """The list times min(1, max_norm / (norm + eps)); norm[0] (fp32, CUDA) gets the norm."""
    _calls.clip_grad_norm(grads._record, max_norm, eps, norm, stream)
