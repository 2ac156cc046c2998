"""Dropout whose mask is a function of a seed, a site and an element's place, and is stored nowhere: the backward draws it again
(csrc/dfa3d_dropout.hip).  What it is added to, the residual of a layer, is added in the same pass."""
import torch

from . import _lib
from ._operands import as_read, check_beside
from .recording import Noted, OperatorFunction, native_for, refuse_capture

__all__ = ["dropout", "DropoutFunction"]


def _drop(x, residual, p, seed, site):
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if x.numel() == 0:
        return y
    there = isinstance(seed, torch.Tensor)
    with _lib.on_device(x.device):
        rc = _lib.lib().dfa3d_dropout(_lib.ptr(x), _lib.ptr(residual), _lib.ptr(y), _lib.ptr(seed) if there else None,
                                      0 if there else seed & (2 ** 64 - 1), site, p, x.numel(), _lib.dtype_code(x), _lib.stream_of(x))
    _lib.check(rc, "dfa3d_dropout")
    return y


class DropoutFunction(OperatorFunction):
    """``apply(x, residual or None, p, seed, site)``: ``dropout`` below, differentiable in ``x`` and ``residual`` any number of times."""

    own = True

    @staticmethod
    def forward(ctx, x, residual, p, seed, site):
        there = isinstance(seed, torch.Tensor)
        ctx.save_for_backward(seed if there else None)
        ctx.set_materialize_grads(False)
        ctx.drawn = p, None if there else seed, site
        return _drop(as_read(x), None if residual is None else as_read(residual), p, seed, site)

    @staticmethod
    def backward(ctx, grad):
        if grad is None:
            return (None,) * 5
        p, seed, site = ctx.drawn
        seed = ctx.saved_tensors[0] if seed is None else seed
        want_x, want_residual = ctx.needs_input_grad[:2]
        return DropoutFunction.apply(grad, None, p, seed, site) if want_x else None, grad if want_residual else None, None, None, None


def backward_of(saved, numbers, wanted, grads):
    """The backward for a native node."""
    p, seed, site, _ = numbers
    ctx = Noted(saved, wanted[:2], drawn=(p, None if saved[0] is not None else seed, site))
    return (*DropoutFunction.backward(ctx, *grads)[:2], None)


def dropout(x, p, seed, site=0, residual=None):
    """``x`` with each element kept with probability ``1 - p`` and divided by that, else zero (whatever it was), plus ``residual`` (shape and
    type of ``x``) if given.  float32, float64 or bfloat16 on the GPU; any strides, a contiguous result.

    ``seed``: an int of 64 bits, or an int64 tensor of one element on the device of ``x``, which is read when the kernel runs: a captured graph
    draws anew on a replay where the tensor holds something else by then.  The backward reads it again, so it may be changed only after the
    backward (autograd says so if it was changed before).  ``site``: a non-negative int of 63 bits.  The same seed, site and number of an element
    in ``x`` (row-major) give the same decision: give every layer a site of its own and every step a seed of its own."""
    p = float(p)
    if (here := native_for(x)) is not None and (got := here[0].dropout(here[1], here[2], x, residual, p, seed, site)) is not None:
        return got
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability has to be between 0 and 1, but got {p}")
    if not x.is_cuda:
        raise RuntimeError("x must be a CUDA tensor")
    _lib.dtype_code(x)
    if residual is not None:
        check_beside(x, residual, "residual", x.shape, x.dtype)
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1 or seed.device != x.device:
            raise RuntimeError(f"seed must be an int or an int64 tensor of one element on {x.device}, got {seed.dtype} of shape {tuple(seed.shape)} "
                               f"on {seed.device}")
    else:
        seed = int(seed)
        if not -2 ** 63 <= seed < 2 ** 64:
            raise ValueError(f"seed has more than 64 bits: {seed}")
    site = int(site)
    if not 0 <= site < 2 ** 63:
        raise ValueError(f"site must be a non-negative int of 63 bits, got {site}")
    refuse_capture(x, residual)
    return DropoutFunction.apply(x, residual, p, seed, site)
