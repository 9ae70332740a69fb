"""PyTorch operators over libdcopy, registered with torch.library.

The reference exposes its Ascend C kernels to PyTorch as custom operators
(ge/examples/custom_op/ascendc_add_custom registers add_custom with
TORCH_LIBRARY_FRAGMENT).  These are the data-movement kernels of this library
as operators in the ``dcopy`` namespace, on CUDA tensors:

  torch.ops.dcopy.nd_to_nz(x, c0)                     ND -> FRACTAL_NZ
  torch.ops.dcopy.nz_to_nd(x_nz, nd_shape, c0)        FRACTAL_NZ -> ND
  torch.ops.dcopy.transpose(x, perm)                  GE Transpose (contiguous result)
  torch.ops.dcopy.datacopy_transpose(x)               standalone datacopy: int32 [r, c] -> [c, r]
  torch.ops.dcopy.strided_gather(x, count, block_len, src_gap)
                                                      DataCopyExt gather into a packed tensor
  torch.ops.dcopy.copy_ext_(dst, src, count, block_len, src_gap, dst_gap)
                                                      DataCopyExt in place (mutates dst)
  torch.ops.dcopy.box(x, sizes, strides, offset)      DataCopyNddma: the strided box of x
                                                      (element strides/offset) packed
  torch.ops.dcopy.nd_to_zz(x, c0) / zz_to_nd(x_zz, nd_shape, c0)
                                                      ND <-> FRACTAL_ZZ
  torch.ops.dcopy.to_fractal_z(w, src_format, c0)     NCHW / NHWC / HWCN / ND weight -> FRACTAL_Z
  torch.ops.dcopy.from_fractal_z(w_fz, dst_format, dst_shape, c0)
                                                      FRACTAL_Z -> NCHW / NHWC / HWCN
  torch.ops.dcopy.embedding(table, ids, scale, first_id)
                                                      rows of a table by token id
  torch.ops.dcopy.expert_sort(expert_ids, experts, align)
                                                      (dest, source, offsets) of a router's choices
  torch.ops.dcopy.expert_dispatch(x, dest, source)    tokens to their experts' rows
  torch.ops.dcopy.expert_combine(y, dest, source, weights)
                                                      and back, weighted and summed

The last four differentiate through embedding_backward and expert_combine_backward, which
are operators too; the gradients are those of dcopy.embedding_grad, dcopy.expert_combine_grad
and, for the moves, each other.

Lengths and gaps of the DataCopyExt operators count ELEMENTS of the tensors'
dtype (as DataCopyPadExtend's arguments do, datacopy.h:14-40).  Each operator
has a fake implementation, so shapes propagate under FakeTensor / torch.compile
tracing without a GPU.  Every call runs on torch's current CUDA stream.
"""
from __future__ import annotations

from typing import List, Optional

import torch
from torch.library import custom_op

import dcopy

# A GE data type of each element width, for the dtype-agnostic Transpose.
_GE_TYPE_OF_WIDTH = {1: dcopy.DATA_TYPE["UINT8"], 2: dcopy.DATA_TYPE["FLOAT16"],
                     4: dcopy.DATA_TYPE["FLOAT"], 8: dcopy.DATA_TYPE["INT64"],
                     16: dcopy.DATA_TYPE["COMPLEX128"]}


def _require_cuda(*ts):
    for t in ts:
        if not t.is_cuda:
            raise ValueError("dcopy operators take CUDA tensors")


@custom_op("dcopy::nd_to_nz", mutates_args=(), device_types="cuda")
def nd_to_nz(x: torch.Tensor, c0: int = 16) -> torch.Tensor:
    _require_cuda(x)
    x = x.contiguous()
    nz, _ = dcopy.nz_shape(list(x.shape), c0)
    out = torch.empty(nz, dtype=x.dtype, device=x.device)
    dcopy.nd_to_nz(out, x, list(x.shape), x.element_size(), c0)
    return out


@nd_to_nz.register_fake
def _nd_to_nz_fake(x, c0=16):
    nz, _ = dcopy.nz_shape(list(x.shape), c0)
    return x.new_empty(nz)


@custom_op("dcopy::nz_to_nd", mutates_args=(), device_types="cuda")
def nz_to_nd(x: torch.Tensor, nd_shape: List[int], c0: int = 16) -> torch.Tensor:
    _require_cuda(x)
    nz, _ = dcopy.nz_shape(list(nd_shape), c0)
    if list(x.shape) != nz:
        raise ValueError(f"NZ tensor shape {list(x.shape)} is not the NZ shape {nz} of {nd_shape}")
    x = x.contiguous()
    out = torch.empty(list(nd_shape), dtype=x.dtype, device=x.device)
    dcopy.nz_to_nd(out, x, list(nd_shape), x.element_size(), c0)
    return out


@nz_to_nd.register_fake
def _nz_to_nd_fake(x, nd_shape, c0=16):
    return x.new_empty(list(nd_shape))


@custom_op("dcopy::transpose", mutates_args=(), device_types="cuda")
def transpose(x: torch.Tensor, perm: List[int]) -> torch.Tensor:
    _require_cuda(x)
    x = x.contiguous()
    out = torch.empty([x.shape[p] for p in perm], dtype=x.dtype, device=x.device)
    dcopy.transpose(out, x, list(x.shape), list(perm), _GE_TYPE_OF_WIDTH[x.element_size()])
    return out


@transpose.register_fake
def _transpose_fake(x, perm):
    return x.new_empty([x.shape[p] for p in perm])


@custom_op("dcopy::datacopy_transpose", mutates_args=(), device_types="cuda")
def datacopy_transpose(x: torch.Tensor) -> torch.Tensor:
    _require_cuda(x)
    if x.dtype != torch.int32 or x.dim() != 2:
        raise ValueError("datacopy_transpose takes a 2-D int32 tensor")
    rows, cols = x.shape
    t = dcopy.plan_tiling(rows, cols, 240, 1)
    out = torch.empty(cols, rows, dtype=x.dtype, device=x.device)
    dcopy.datacopy_large(x.contiguous(), out, t)
    return out


@datacopy_transpose.register_fake
def _datacopy_transpose_fake(x):
    return x.new_empty(x.shape[1], x.shape[0])


@custom_op("dcopy::strided_gather", mutates_args=(), device_types="cuda")
def strided_gather(x: torch.Tensor, count: int, block_len: int, src_gap: int) -> torch.Tensor:
    _require_cuda(x)
    x = x.contiguous()
    e = x.element_size()
    out = torch.empty(count * block_len, dtype=x.dtype, device=x.device)
    dcopy.copy_ext(out, x, count, block_len * e, src_gap * e, 0)
    return out


@strided_gather.register_fake
def _strided_gather_fake(x, count, block_len, src_gap):
    return x.new_empty(count * block_len)


@custom_op("dcopy::copy_ext_", mutates_args=("dst",), device_types="cuda")
def copy_ext_(dst: torch.Tensor, src: torch.Tensor, count: int, block_len: int, src_gap: int,
              dst_gap: int) -> None:
    _require_cuda(dst, src)
    if dst.dtype != src.dtype or not dst.is_contiguous():
        raise ValueError("copy_ext_ needs a contiguous dst of src's dtype")
    e = src.element_size()
    dcopy.copy_ext(dst, src.contiguous(), count, block_len * e, src_gap * e, dst_gap * e)


@copy_ext_.register_fake
def _copy_ext_fake(dst, src, count, block_len, src_gap, dst_gap):
    return None


@custom_op("dcopy::box", mutates_args=(), device_types="cuda")
def box(x: torch.Tensor, sizes: List[int], strides: List[int], offset: int = 0) -> torch.Tensor:
    """torch.as_strided(x, sizes, strides, offset).contiguous(), moved by dcopy_copy_nd."""
    _require_cuda(x)
    if len(sizes) != len(strides) or not 1 <= len(sizes) <= 5:
        raise ValueError("box: sizes and strides must have the same rank, 1..5")
    x = x.contiguous()
    last = offset + sum((n - 1) * st for n, st in zip(sizes, strides) if n > 0)
    if offset < 0 or min(strides) < 0 or (all(n > 0 for n in sizes) and last >= x.numel()):
        raise ValueError("box: the box runs outside x")
    out = torch.empty(list(sizes), dtype=x.dtype, device=x.device)
    if out.numel():
        dense = [1] * len(sizes)
        for k in range(len(sizes) - 2, -1, -1):
            dense[k] = dense[k + 1] * sizes[k + 1]
        dcopy.copy_nd(out, x.data_ptr() + offset * x.element_size(), list(sizes), list(strides),
                      dense, x.element_size())
    return out


@box.register_fake
def _box_fake(x, sizes, strides, offset=0):
    return x.new_empty(list(sizes))


@custom_op("dcopy::nd_to_zz", mutates_args=(), device_types="cuda")
def nd_to_zz(x: torch.Tensor, c0: int = 16) -> torch.Tensor:
    _require_cuda(x)
    x = x.contiguous()
    zz, _ = dcopy.zz_shape(list(x.shape), c0)
    out = torch.empty(zz, dtype=x.dtype, device=x.device)
    dcopy.nd_to_zz(out, x, list(x.shape), x.element_size(), c0)
    return out


@nd_to_zz.register_fake
def _nd_to_zz_fake(x, c0=16):
    zz, _ = dcopy.zz_shape(list(x.shape), c0)
    return x.new_empty(zz)


@custom_op("dcopy::zz_to_nd", mutates_args=(), device_types="cuda")
def zz_to_nd(x: torch.Tensor, nd_shape: List[int], c0: int = 16) -> torch.Tensor:
    _require_cuda(x)
    zz, _ = dcopy.zz_shape(list(nd_shape), c0)
    if list(x.shape) != zz:
        raise ValueError(f"ZZ tensor shape {list(x.shape)} is not the ZZ shape {zz} of {nd_shape}")
    x = x.contiguous()
    out = torch.empty(list(nd_shape), dtype=x.dtype, device=x.device)
    dcopy.zz_to_nd(out, x, list(nd_shape), x.element_size(), c0)
    return out


@zz_to_nd.register_fake
def _zz_to_nd_fake(x, nd_shape, c0=16):
    return x.new_empty(list(nd_shape))


def _weight_format(name: str) -> int:
    if name not in ("NCHW", "NHWC", "HWCN", "ND"):
        raise ValueError(f"FRACTAL_Z weights are NCHW, NHWC, HWCN or ND, not {name}")
    return dcopy.FORMAT[name]


@custom_op("dcopy::to_fractal_z", mutates_args=(), device_types="cuda")
def to_fractal_z(w: torch.Tensor, src_format: str, c0: int = 16) -> torch.Tensor:
    _require_cuda(w)
    fmt = _weight_format(src_format)
    w = w.contiguous()
    out = torch.empty(dcopy.fz_shape(fmt, list(w.shape), c0), dtype=w.dtype, device=w.device)
    dcopy.to_fractal_z(out, w, fmt, list(w.shape), w.element_size(), c0)
    return out


@to_fractal_z.register_fake
def _to_fractal_z_fake(w, src_format, c0=16):
    return w.new_empty(dcopy.fz_shape(_weight_format(src_format), list(w.shape), c0))


@custom_op("dcopy::from_fractal_z", mutates_args=(), device_types="cuda")
def from_fractal_z(w: torch.Tensor, dst_format: str, dst_shape: List[int],
                   c0: int = 16) -> torch.Tensor:
    _require_cuda(w)
    fmt = _weight_format(dst_format)
    w = w.contiguous()
    out = torch.empty(list(dst_shape), dtype=w.dtype, device=w.device)
    dcopy.from_fractal_z(out, w, fmt, list(dst_shape), w.element_size(), c0)
    return out


@from_fractal_z.register_fake
def _from_fractal_z_fake(w, dst_format, dst_shape, c0=16):
    return w.new_empty(list(dst_shape))


# ---- operators of language models ------------------------------------------------------


def _dense(t: torch.Tensor) -> torch.Tensor:
    """A gradient as autograd hands it over may be expanded or transposed."""
    return t.contiguous()


@custom_op("dcopy::embedding", mutates_args=(), device_types="cuda")
def embedding(table: torch.Tensor, ids: torch.Tensor, scale: float = 1.0,
              first_id: int = 0) -> torch.Tensor:
    out = table.new_empty(list(ids.shape) + [table.shape[1]])
    dcopy.embedding_lookup(out.view(ids.numel(), table.shape[1]), table, ids.contiguous(), scale,
                           first_id)
    return out


@embedding.register_fake
def _embedding_fake(table, ids, scale=1.0, first_id=0):
    return table.new_empty(list(ids.shape) + [table.shape[1]])


@custom_op("dcopy::embedding_backward", mutates_args=(), device_types="cuda")
def embedding_backward(dout: torch.Tensor, ids: torch.Tensor, vocab: int, scale: float = 1.0,
                       first_id: int = 0) -> torch.Tensor:
    width = dout.shape[-1]
    grad = dout.new_empty(vocab, width)
    dcopy.embedding_grad(grad, _dense(dout).view(ids.numel(), width), ids.contiguous(), scale, first_id)
    return grad


@embedding_backward.register_fake
def _embedding_backward_fake(dout, ids, vocab, scale=1.0, first_id=0):
    return dout.new_empty(vocab, dout.shape[-1])


def _embedding_setup(ctx, inputs, output):
    table, ids, ctx.scale, ctx.first_id = inputs
    ctx.vocab = table.shape[0]
    ctx.save_for_backward(ids)


def _embedding_grad(ctx, dout):
    ids, = ctx.saved_tensors
    return embedding_backward(dout, ids, ctx.vocab, ctx.scale, ctx.first_id), None, None, None


embedding.register_autograd(_embedding_grad, setup_context=_embedding_setup)


@custom_op("dcopy::expert_sort", mutates_args=(), device_types="cuda")
def expert_sort(expert_ids: torch.Tensor, experts: int,
                align: int = 1) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    whole = dict(dtype=torch.int32, device=expert_ids.device)
    dest = torch.empty(expert_ids.shape, **whole)
    source = torch.empty(dcopy.expert_rows(expert_ids.numel(), experts, align), **whole)
    offsets = torch.empty(experts + 1, **whole)
    dcopy.expert_sort(dest, source, offsets, expert_ids.contiguous(), align)
    return dest, source, offsets


def _expert_rows(entries, experts, align):
    """dcopy.expert_rows; where a number is symbolic, its formula, so that it stays so."""
    if all(isinstance(n, int) for n in (entries, experts, align)):
        return dcopy.expert_rows(entries, experts, align)
    return entries + torch.sym_min(experts, entries) * (align - 1)


@expert_sort.register_fake
def _expert_sort_fake(expert_ids, experts, align=1):
    whole = dict(dtype=torch.int32)
    return (expert_ids.new_empty(expert_ids.shape, **whole),
            expert_ids.new_empty(_expert_rows(expert_ids.numel(), experts, align), **whole),
            expert_ids.new_empty(experts + 1, **whole))


@custom_op("dcopy::expert_dispatch", mutates_args=(), device_types="cuda")
def expert_dispatch(x: torch.Tensor, dest: torch.Tensor, source: torch.Tensor) -> torch.Tensor:
    out = x.new_empty(source.numel(), x.shape[1])
    dcopy.expert_dispatch(out, _dense(x), dest, source)
    return out


@expert_dispatch.register_fake
def _expert_dispatch_fake(x, dest, source):
    return x.new_empty(source.numel(), x.shape[1])


@custom_op("dcopy::expert_combine", mutates_args=(), device_types="cuda")
def expert_combine(y: torch.Tensor, dest: torch.Tensor, source: torch.Tensor,
                   weights: Optional[torch.Tensor] = None) -> torch.Tensor:
    out = y.new_empty(dest.shape[0], y.shape[1])
    dcopy.expert_combine(out, _dense(y), dest, None if weights is None else _dense(weights.float()))
    return out


@expert_combine.register_fake
def _expert_combine_fake(y, dest, source, weights=None):
    return y.new_empty(dest.shape[0], y.shape[1])


@custom_op("dcopy::expert_combine_backward", mutates_args=(), device_types="cuda")
def expert_combine_backward(dout: torch.Tensor, y: torch.Tensor, dest: torch.Tensor,
                            source: torch.Tensor,
                            weights: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    dy = y.new_empty(y.shape)
    dweights = weights.new_empty(weights.shape, dtype=torch.float32)  # the kernel's type
    dcopy.expert_combine_grad(dy, dweights, _dense(dout), _dense(y), dest, _dense(weights.float()),
                              source)
    return dy, dweights.to(weights.dtype, copy=weights.dtype != torch.float32)


@expert_combine_backward.register_fake
def _expert_combine_backward_fake(dout, y, dest, source, weights):
    return y.new_empty(y.shape), weights.new_empty(weights.shape)


def _dispatch_setup(ctx, inputs, output):
    _, dest, source = inputs
    ctx.save_for_backward(dest, source)


def _dispatch_grad(ctx, dout):
    dest, source = ctx.saved_tensors
    return expert_combine(dout, dest, source, None), None, None


expert_dispatch.register_autograd(_dispatch_grad, setup_context=_dispatch_setup)


def _combine_setup(ctx, inputs, output):
    y, dest, source, weights = inputs
    ctx.weighted = weights is not None
    ctx.save_for_backward(dest, source, *((y, weights) if ctx.weighted else ()))


def _combine_grad(ctx, dout):
    dest, source, *weighted = ctx.saved_tensors
    if not ctx.weighted:
        return expert_dispatch(dout, dest, source), None, None, None
    dy, dweights = expert_combine_backward(dout, weighted[0], dest, source, weighted[1])
    return dy, None, None, dweights


expert_combine.register_autograd(_combine_grad, setup_context=_combine_setup)
