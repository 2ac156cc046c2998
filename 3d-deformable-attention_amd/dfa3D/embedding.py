"""Rows looked up in a learned table, scaled and summed over heads, and the gradients of the table, by its entries' places
(csrc/dfa3d_embedding.hip).  The cross-attention layer adds what its sampling left unexplained of the queries that a camera sees in this way
(BEVFormer_DFA3D/projects/mmdet3d_plugin/bevformer/modules/spatial_cross_attention.py:739-740); tokens, rows and columns of a grid, cameras and levels are
looked up in plain tables."""
import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._operands import as_read, check_beside
from .recording import Noted, OperatorFunction, native_for, refuse_capture

__all__ = ["scaled_embedding", "ScaledEmbeddingFunction"]


def _dims(table, index, out_shape):
    """R, N, V, H, E"""
    V, H, E = table if len(table) == 3 else (table[0], 1, table[1])
    rows = 1
    for n in out_shape[:-1]:
        rows *= n
    N = index.numel()
    return rows // N if N else 0, N, V, H, E


class ScaledEmbeddingFunction(OperatorFunction):
    """``apply(table, index, scale or None, plus or None, mul)``: ``scaled_embedding`` below, differentiable in ``table``, ``scale`` and ``plus``."""

    own = True

    @staticmethod
    def forward(ctx, table, index, scale, plus, mul):
        if scale is not None:
            lead = scale.shape[:scale.dim() - index.dim() - (table.dim() - 2)]
        else:
            lead = plus.shape[:plus.dim() - index.dim() - 1] if plus is not None else ()
        want_table, _, want_scale = ctx.needs_input_grad[:3] if ctx.needs_input_grad else (False,) * 3
        ctx.save_for_backward(table if want_scale else None, index, scale if want_table else None)
        ctx.set_materialize_grads(False)
        ctx.of = tuple(table.shape), mul
        out = table.new_empty(*lead, *index.shape, table.shape[-1])
        dims = _dims(table.shape, index, out.shape)
        if out.numel() == 0:
            return out
        if dims[2] * dims[3] == 0:                               # no entries: nothing to add
            return out.zero_() if plus is None else out.copy_(plus)
        table, index = as_read(table), as_read(index)
        scale, plus = (None if t is None else as_read(t) for t in (scale, plus))
        with _lib.on_device(table.device):
            rc = _lib.lib().dfa3d_embedding(_lib.ptr(table), _lib.ptr(index), index.element_size(), _lib.ptr(scale), _lib.ptr(plus), _lib.ptr(out), *dims, mul,
                                            _lib.dtype_code(table), _lib.stream_of(table))
        _lib.check(rc, "dfa3d_embedding")
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        if grad is None:
            return (None,) * 5
        table, index, scale = ctx.saved_tensors
        shape, mul = ctx.of
        want_table, _, want_scale, want_plus = ctx.needs_input_grad[:4]
        grad_table = grad_scale = None
        if want_table or want_scale:
            g, index = as_read(grad), as_read(index)
            dims, dtype, lib = _dims(shape, index, grad.shape), _lib.dtype_code(grad), _lib.lib()
            empty = grad.numel() == 0 or dims[2] * dims[3] == 0
            if want_scale:
                lead = grad.shape[:-1] if len(shape) == 2 else (*grad.shape[:-1], shape[1])
                grad_scale = torch.empty(lead, dtype=torch.float32 if dtype == _lib.DFA3D_BF16 else grad.dtype, device=grad.device)
                table = as_read(table)
            if want_table:
                grad_table = torch.empty(shape, dtype=grad.dtype, device=grad.device)
                scale = None if scale is None else as_read(scale)
            with _lib.on_device(grad.device):
                stream = _lib.stream_of(grad)
                if empty:
                    for t in (grad_table, grad_scale):
                        if t is not None:
                            t.zero_()
                elif want_table:                                 # and the scales' with it
                    nbytes = lib.dfa3d_embedding_grad_table_workspace_bytes(*dims, dtype)
                    workspace = torch.empty(nbytes, dtype=torch.uint8, device=grad.device)
                    rc = lib.dfa3d_embedding_grad_table(_lib.ptr(table), _lib.ptr(index), index.element_size(), _lib.ptr(scale), _lib.ptr(g), _lib.ptr(grad_table),
                                                        _lib.ptr(grad_scale), _lib.ptr(workspace), nbytes, *dims, mul, dtype, stream)
                    _lib.check(rc, "dfa3d_embedding_grad_table")
                else:
                    rc = lib.dfa3d_embedding_grad_scale(_lib.ptr(table), _lib.ptr(index), index.element_size(), _lib.ptr(g), _lib.ptr(grad_scale), *dims, mul, dtype,
                                                        stream)
                    _lib.check(rc, "dfa3d_embedding_grad_scale")
        return grad_table, None, grad_scale, grad if want_plus else None, None


def backward_of(saved, numbers, wanted, grads):
    """The backward for a native node."""
    mul, V, H, dims = numbers
    E = grads[0].shape[-1]
    ctx = Noted(saved, (wanted[0], False, *wanted[1:]), of=((V, H, E) if dims == 3 else (V, E), mul))
    got = ScaledEmbeddingFunction.backward(ctx, *grads)
    return got[0], got[2], got[3]


def scaled_embedding(table, index, scale=None, plus=None, mul=1.0):
    """``plus[..., n, :] + mul * sum over h of scale[..., n, h] * table[index[n], h, :]``, n the places of ``index`` (any shape, int32 or int64).

    ``table``: (V, H, E), or (V, E) for one row per entry; float32, float64 or bfloat16 on the GPU.  ``scale``: (..., *index.shape, H), without the
    last dimension for a table (V, E); of the table's type, float32 for bfloat16; ones if None.  ``plus``: (..., *index.shape, E) of the table's type;
    zeros if None.  The leading dimensions, batch elements that share the places, are the same in both; there are none without either.
    ``mul``: a number.  Returns (..., *index.shape, E) of the table's type; sums are formed in float32 (float64).

    A place whose index is negative or not below V (the padding of a list) takes what ``plus`` holds there, and no gradient goes through it.
    Gradients of the table are formed in an order that the sizes decide, without atomics: the same every time.  They are refused where more than 2^20 batch
    elements have more than 2^30 places in all."""
    mul = float(mul)
    if (here := native_for(table)) is not None and (got := here[0].embedding(here[1], here[2], table, index, scale, plus, mul)) is not None:
        return got
    if not table.is_cuda:
        raise RuntimeError("table must be a CUDA tensor")
    _lib.dtype_code(table)
    if table.dim() not in (2, 3):
        raise RuntimeError(f"table must be (V, H, E) or (V, E), got {tuple(table.shape)}")
    if index.dtype not in (torch.int32, torch.int64):
        raise RuntimeError(f"index has dtype {index.dtype}, expected torch.int32 or torch.int64")
    check_beside(table, index, "index", index.shape, index.dtype)
    heads = tuple(table.shape[1:-1])
    lead = None
    for t, name, tail, dtype in ((scale, "scale", heads, torch.float32 if table.dtype == torch.bfloat16 else table.dtype),
                                 (plus, "plus", (table.shape[-1],), table.dtype)):
        if t is None:
            continue
        tail = (*index.shape, *tail)
        if lead is None:
            lead = tuple(t.shape[:max(t.dim() - len(tail), 0)])
        check_beside(table, t, name, (*lead, *tail), dtype)
    refuse_capture(table, scale, plus)
    return ScaledEmbeddingFunction.apply(table, index, scale, plus, mul)
