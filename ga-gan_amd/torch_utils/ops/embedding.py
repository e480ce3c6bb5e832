"""Rows of a table by index, scaled, plus a bias, with the table's gradient summed over equal indices:

    y[..., :] = table[index[...]] * w_gain + b * b_gain                index [...] int32 / int64, table [V, F], b [F]

The label embedding of a conditional network: what `self.embed(one_hot)` of the reference's mapping network
(DissimilarDomains/training/networks.py:732, 748) computes with a product over all classes - bit for bit in float32 - given
the class numbers themselves; `table` is then the layer's weight transposed (a view: no copy is made, and its gradient comes
in the same layout).  The gradient sums the rows of dy that share an index in the order of the tokens, in float32 and without
atomics, so that the same inputs give the same bits (`sg_embedding`, `sg_embedding_backward`).  The pair of functions is
closed under differentiation: the gradient's own gradient is a lookup again.

Indices outside the table are not checked on the host (that would wait for the device): they read as rows of NaN and take
no gradient."""
import ctypes

import torch

from ... import _lib
from .. import misc
from . import conv2d_gradfix

i32, i64, f32, vp = _lib.i32, _lib.i64, _lib.f32, _lib.vp


class EmbeddingParams(ctypes.Structure):
    _fields_ = [('index', vp), ('table', vp), ('bias', vp), ('dtype', i32), ('index_bytes', i32),
                ('tokens', i64), ('v', i64), ('f', i64), ('stride_v', i64), ('stride_f', i64), ('w_gain', f32), ('b_gain', f32)]


_DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def _params(index, table, bias, gains):
    v, f = table.shape
    return EmbeddingParams(_lib.ptr(index), _lib.ptr(table), _lib.ptr(bias), _lib.DTYPES[table.dtype], index.element_size(),
                           index.numel(), v, f, table.stride(0), table.stride(1), *gains)


def _lookup(index, table, b, gains):
    y = torch.empty([index.numel(), table.shape[1]], dtype=table.dtype, device=table.device)
    if y.numel():
        b = b.contiguous() if b is not None else None
        p = _params(index, table, b, gains)
        fn = _lib.lib().sg_embedding
        _lib.launch_raw(lambda stream: fn(ctypes.byref(p), _lib.ptr(y), stream), table, 'sg_embedding', 'embedding_kernel', 2 * _lib.nbytes(y))
    return y


def _table_gradient(dy, index, shape, by_columns, gains, want_bias):
    v, f = shape
    dtable = torch.empty([f, v], dtype=dy.dtype, device=dy.device).t() if by_columns else torch.empty([v, f], dtype=dy.dtype, device=dy.device)
    dbias = torch.empty([f], dtype=dy.dtype, device=dy.device) if want_bias else None
    if dtable.numel():
        p = _params(index, dtable, None, gains)
        if by_columns:                          # (strides of a one-row or one-column table are not torch's to give)
            p.stride_v, p.stride_f = 1, v
        else:
            p.stride_v, p.stride_f = f, 1
        handle = _lib.lib()
        need = handle.sg_embedding_backward_workspace_bytes(ctypes.byref(p))
        work = torch.empty([need], dtype=torch.uint8, device=dy.device) if need else None
        _lib.launch_raw(lambda stream: handle.sg_embedding_backward(ctypes.byref(p), _lib.ptr(dy), _lib.ptr(dbias), _lib.ptr(work), need, stream),
                        dy, 'sg_embedding_backward', 'embedding_grad_runs_kernel', _lib.nbytes(dy, dtable))
    return dtable, dbias


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, b, index, gains):
        ctx.save_for_backward(index)
        ctx.shape, ctx.gains = tuple(table.shape), gains
        ctx.by_columns = table.stride(1) != 1 and table.stride(0) == 1
        return _lookup(index, table, b, gains)

    @staticmethod
    def backward(ctx, dy):
        index, = ctx.saved_tensors
        if conv2d_gradfix.parameter_gradients_disabled:
            return None, None, None, None
        dtable, dbias = _EmbeddingGrad.apply(dy, index, ctx.shape, ctx.by_columns, ctx.gains, ctx.needs_input_grad[1])
        return (dtable if ctx.needs_input_grad[0] else None), dbias, None, None


class _EmbeddingGrad(torch.autograd.Function):
    @staticmethod
    def forward(ctx, dy, index, shape, by_columns, gains, want_bias):
        ctx.save_for_backward(index)
        ctx.gains = gains
        ctx.set_materialize_grads(False)
        return _table_gradient(dy.contiguous(), index, shape, by_columns, gains, want_bias)

    @staticmethod
    def backward(ctx, ddtable, ddbias):
        index, = ctx.saved_tensors
        if ddtable is None and ddbias is None:
            return (None,) * 6
        w_gain, b_gain = ctx.gains
        if ddtable is None:
            return (ddbias * b_gain).expand(index.numel(), -1), None, None, None, None, None
        return embedding(index, ddtable, ddbias, w_gain=w_gain, b_gain=b_gain), None, None, None, None, None


def embedding(index, table, b=None, w_gain=1.0, b_gain=1.0):
    """index [...] int32 or int64, table [V, F] in any layout, b [F] or None -> [..., F] of the table's dtype (float32, float16 or
    bfloat16); one device."""
    assert isinstance(index, torch.Tensor) and isinstance(table, torch.Tensor)
    misc.require_gpu(table, 'embedding')
    if table.dtype not in _DTYPES:
        raise RuntimeError(f'embedding: unsupported dtype {table.dtype}')
    if index.dtype not in (torch.int32, torch.int64):
        raise RuntimeError(f'embedding: indices must be int32 or int64, not {index.dtype}')
    if table.dim() != 2 or table.shape[0] < 1:
        raise RuntimeError(f'embedding: table {tuple(table.shape)} must be [V, F] with at least one row')
    if index.device != table.device or (b is not None and (b.device != table.device or b.dtype != table.dtype)):
        raise RuntimeError('embedding: index and b must be on the device of the table, b of its dtype')
    if b is not None and tuple(b.shape) != (table.shape[1],):
        raise RuntimeError(f'embedding: b {tuple(b.shape)} must have one entry per column of the table {tuple(table.shape)}')
    flat = index.reshape(-1).contiguous()
    gains = (float(w_gain), float(b_gain))
    if torch.is_grad_enabled() and (table.requires_grad or (b is not None and b.requires_grad)):
        y = _Embedding.apply(table, b, flat, gains)
    else:
        y = _lookup(flat, table, b, gains)
    return y if index.dim() == 1 else y.reshape(*index.shape, table.shape[1])
