"""Rows of a shared, learnable table by index, scaled, with the gradients of the table and of the scales -- one launch forward
(vegs_amd/csrc/embedding.hip, C ABI include/vegs_embedding.h).

  lookup(table, ids, scale)     out[i] = scale[i] * table[ids[i]]

What a model shares between its Gaussians, frames or instances is held once and looked up: an SH codebook (table [K, 15, 3],
one id per Gaussian; the result IS the f_rest input of the rasterizer, next to instances.activate's outputs), per-image codes,
pose corrections by frame.  The table's gradient is dense, in the table's type: a float32 table is stepped by
vegs_amd.optim.Adam, counted by grad_norm and exchanged by vegs_amd.dist like any other parameter.  GPU tensors only; there
is no CPU path.
"""
import math
import struct

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _capi

_ID_TYPES = (torch.int32, torch.int64)


def _row_layout(t, lead, width):
    """(t or a contiguous copy, elements between rows): `t` [*lead, ...] as rows of `width` contiguous elements."""
    if t.is_contiguous():
        return t, width
    if lead == 1 and t.stride(0) >= width:
        expect = 1
        for n, st in zip(reversed(t.shape[1:]), reversed(t.stride()[1:])):
            if n != 1 and st != expect:
                return t.contiguous(), width
            expect *= n
        return t, t.stride(0)
    return t.contiguous(), width


_LOOKUP = struct.Struct("3Q4q3if")           # VrLookup
_LARGEST = torch.finfo(torch.float32).max
_ALONE = 1024                                # up to so many entries vr_lookup_scratch_bytes is 0


def _arguments(table, ids, scale, width, dtype):
    """(VrLookup as packed bytes, the tensors behind its pointers: table, ids, scales or None)"""
    stride, rows, at = width, None, 0
    if not table.is_contiguous():
        table, stride = _row_layout(table, 1, width)
    if not ids.is_contiguous():
        ids = ids.contiguous()
    if isinstance(scale, torch.Tensor):
        rows, scale = scale.contiguous(), 1.0
        at = rows.data_ptr()
    kinds = _capi.VR_DTYPES
    return _LOOKUP.pack(table.data_ptr(), ids.data_ptr(), at, ids.numel(), table.shape[0], width, stride, kinds[table.dtype],
                        kinds[dtype], ids.dtype == torch.int64, scale), table, ids, rows


# (What allocates and where follows the host's time, which is what a call of few ids takes: new_empty and empty_like are half of
# torch.empty with its keywords, and torch._C._cuda_getDevice a third of torch.cuda.current_device.)
def _forward(arguments, shape, dtype, table):
    index = table.get_device()
    if torch._C._cuda_getDevice() != index:
        with torch.cuda.device(index):
            return _forward(arguments, shape, dtype, table)
    out = table.new_empty(shape) if dtype is table.dtype else table.new_empty(shape, dtype=dtype)
    if out.numel():
        rc = (_capi._lib or _capi.load()).vr_lookup_forward(arguments, out.data_ptr(), torch._C._cuda_getCurrentRawStream(index))
        if rc:
            _capi.check(rc)
    return out


def _backward(ctx, g):
    index = g.get_device()
    if torch._C._cuda_getDevice() != index:
        with torch.cuda.device(index):
            return _backward(ctx, g)
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(g).tangent is not None:
        raise NotImplementedError("the gradients of lookup have no forward-mode derivative")
    # (hooks on saved tensors -- recomputation, offloading -- give them back at addresses of their own)
    rows, flat, scales = ctx.saved_tensors
    scale, shape, kind, dtype, ids_shape, n, width = ctx.lookup
    want_table, _, want_scale, _, _, _ = ctx.needs_input_grad
    d_table = d_scale = scratch = None
    nbytes = at_table = at_scale = 0
    lib = _capi._lib or _capi.load()
    if want_table:
        if rows is not None and rows.is_contiguous():
            d_table = torch.empty_like(rows)
        else:
            d_table = g.new_empty(shape) if kind is dtype else g.new_empty(shape, dtype=kind)
        at_table = d_table.data_ptr()
        if n > _ALONE:
            nbytes = lib.vr_lookup_scratch_bytes(n, shape[0], width)
    if want_scale:
        d_scale = scales.new_empty(ids_shape)
        at_scale = d_scale.data_ptr()
    if width == 0 or n == 0:
        return (d_table.zero_() if want_table else None), None, (d_scale.zero_() if want_scale else None), None, None, None
    stride = width
    if not g.is_contiguous():
        g, stride = _row_layout(g, len(ids_shape), width)
    if nbytes:
        scratch = g.new_empty(nbytes, dtype=torch.uint8)
    # (the table's values are only read for the gradient of the scales: where that is not wanted, anything of its shape stands for it)
    arguments, *keep = _arguments(d_table if rows is None else rows, flat, scale if scales is None else scales, width, dtype)
    rc = lib.vr_lookup_backward(arguments, g.data_ptr(), stride, at_table, at_scale, scratch.data_ptr() if nbytes else None, nbytes,
                                torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _capi.check(rc)
    return d_table, None, d_scale, None, None, None


_backward_once = once_differentiable(_backward)


class _Lookup(torch.autograd.Function):

    @staticmethod
    def forward(ctx, table, ids, scale, width, dtype, shape):
        arguments, rows, flat, scales = _arguments(table, ids, scale, width, dtype)
        ctx.lookup = None if scales is not None else scale, table.shape, table.dtype, dtype, ids.shape, ids.numel(), width
        ctx.save_for_backward(rows if ctx.needs_input_grad[2] else None, flat, scales)
        return _forward(arguments, shape, dtype, table)

    @staticmethod
    def backward(ctx, g):
        # (grad mode is on where the caller asked for a graph of the gradients, which are not differentiable again)
        return _backward_once(ctx, g) if torch.is_grad_enabled() else _backward(ctx, g)


def lookup(table, ids, scale=None, dtype=None):
    """scale * table[ids]: [*ids.shape, *table.shape[1:]], differentiable with respect to `table` and to a `scale` tensor.

    table: [K, ...] float32, bfloat16 or float16.  ids: int32 or int64 of any shape; an id outside [0, K) -- -1 by
    convention -- means "no row": zeros, and no gradient whatever stands in its place.  scale: a number of float32's range, or a
    float32 tensor shaped like ids.  dtype: of the result, the table's (default) or float32.

    The product is formed in float32 and rounded once.  The table's gradient adds the entries of a row in float32, in an order
    that the sizes and ids fix, and is rounded once to the table's type; it is dense (rows without an entry are zeros) and the same
    bits every time.  Forward-mode differentiation is refused, as by every operator of this package."""
    if not isinstance(table, torch.Tensor) or not table.is_cuda:
        raise ValueError("table must be a GPU tensor (there is no CPU path)")
    shape, kind, device = table.shape, table.dtype, table.device
    if not shape or kind not in _capi.VR_DTYPES or table.layout is not torch.strided:
        raise ValueError(f"table must be a dense float32, bfloat16 or float16 tensor [K, ...] (got {kind} {tuple(shape)})")
    if not isinstance(ids, torch.Tensor) or ids.device != device or ids.dtype not in _ID_TYPES:
        raise ValueError(f"ids must be an int32 or int64 tensor on {device}")
    row = shape[1:]
    width = row.numel()
    if ids.numel() >= 1 << 30 or shape[0] >= (1 << 31) - 1 or width > 1 << 22:
        raise ValueError("at most 2^30 - 1 ids, 2^31 - 2 rows and 2^22 values in a row")
    wanted = table.requires_grad
    if scale is None:
        scale = 1.0
    elif isinstance(scale, torch.Tensor):
        if scale.device != device or scale.dtype != torch.float32 or scale.shape != ids.shape:
            raise ValueError(f"a scale tensor must be float32 {tuple(ids.shape)} on {device}, shaped like ids "
                             f"(got {scale.dtype} {tuple(scale.shape)} on {scale.device})")
        wanted = wanted or scale.requires_grad
    else:
        scale = float(scale)
        if abs(scale) > _LARGEST and scale not in (math.inf, -math.inf):
            raise ValueError(f"a scale must be a float32 number (got {scale})")
    if dtype is None:
        dtype = kind
    elif dtype != kind and dtype != torch.float32:
        raise ValueError(f"the result has the table's type or float32 (got {dtype} for a table of {kind})")
    # (inside a level of forward-mode differentiation an input may carry a tangent: torch refuses those, which the function has no rule for)
    if wanted and torch.is_grad_enabled() or forward_ad._current_level >= 0:
        return _Lookup.apply(table, ids, scale, width, dtype, ids.shape + row)
    arguments, *keep = _arguments(table, ids, scale, width, dtype)
    return _forward(arguments, ids.shape + row, dtype, table)
