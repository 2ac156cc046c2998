"""Group norm with an activation on feature maps as the attention operators take them: channels last, the levels behind one another
(csrc/dfa3d_norm.hip)."""
import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._operands import as_read, check_beside
from .recording import Noted, OperatorFunction, native_for, refuse_capture

__all__ = ["level_group_norm", "LevelGroupNormFunction"]


def _keys(x):
    """B, S, C of (B, ..., C)"""
    keys = 1
    for n in x.shape[1:-1]:
        keys *= n
    return x.shape[0], keys, x.shape[-1]


class LevelGroupNormFunction(OperatorFunction):
    """``apply(x, weight or None, bias or None, level_start_index or None, num_groups, eps, act)``: ``level_group_norm`` below on operands that have been
    checked, weight and bias of the type that sums have; differentiable in ``x``, ``weight`` and ``bias``."""

    own = True

    @staticmethod
    def forward(ctx, x, weight, bias, level_start, groups, eps, act):
        x = as_read(x)
        weight, bias, level_start = (None if t is None else as_read(t) for t in (weight, bias, level_start))
        ctx.set_materialize_grads(False)
        ctx.of = groups, act
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        if y.numel() == 0:
            ctx.save_for_backward(x, weight, bias, level_start, None)
            return y
        dtype, dims = _lib.dtype_code(x), (*_keys(x), groups, 1 if level_start is None else level_start.numel())
        stats = torch.empty(dims[0], dims[4], groups, 2, dtype=torch.float64 if x.dtype == torch.float64 else torch.float32, device=x.device)
        lib = _lib.lib()
        nbytes = lib.dfa3d_group_norm_workspace_bytes(*dims, 0, dtype)
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
        with _lib.on_device(x.device):
            rc = lib.dfa3d_group_norm(_lib.ptr(x), _lib.ptr(weight), _lib.ptr(bias), _lib.ptr(level_start), _lib.ptr(y), _lib.ptr(stats), _lib.ptr(workspace), nbytes,
                                      *dims, eps, act, dtype, _lib.stream_of(x))
        _lib.check(rc, "dfa3d_group_norm")
        ctx.save_for_backward(x, weight, bias, level_start, stats)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        if grad is None:
            return (None,) * 7
        x, weight, bias, level_start, stats = ctx.saved_tensors
        groups, act = ctx.of
        wanted = ctx.needs_input_grad[:3]
        grad = as_read(grad)
        got = [torch.empty(t.shape, dtype=t.dtype, device=t.device) if want else None for t, want in zip((x, weight, bias), wanted)]
        if stats is None:
            return (*(None if t is None else t.zero_() for t in got), None, None, None, None)
        dtype, dims = _lib.dtype_code(x), (*_keys(x), groups, stats.shape[1])
        lib = _lib.lib()
        nbytes = lib.dfa3d_group_norm_workspace_bytes(*dims, 1, dtype)
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
        with _lib.on_device(x.device):
            rc = lib.dfa3d_group_norm_grad(_lib.ptr(x), _lib.ptr(weight), _lib.ptr(bias), _lib.ptr(level_start), _lib.ptr(stats), _lib.ptr(grad),
                                           *(_lib.ptr(t) for t in got), _lib.ptr(workspace), nbytes, *dims, act, dtype, _lib.stream_of(x))
        _lib.check(rc, "dfa3d_group_norm_grad")
        return (*got, None, None, None, None)


def backward_of(saved, numbers, wanted, grads):
    """The backward for a native node."""
    return LevelGroupNormFunction.backward(Noted(saved, wanted, of=tuple(numbers[1:3])), *grads)[:3]


def level_group_norm(x, num_groups, weight=None, bias=None, level_start_index=None, eps=1e-5, act=None):
    """``act((x - mean) / sqrt(variance + eps) * weight + bias)`` with a mean and a variance (about the mean, divided by the count) for each batch element, level and
    group of ``C / num_groups`` neighbouring channels.

    ``x`` (B, ..., C), channels last: float32, float64 or bfloat16 on the GPU.  ``level_start_index`` (L,) int64 for ``x`` (B, S, C), up to 16 levels: the first
    key of each, on the device, as the attention operators take it; a level ends where the next one begins, the last one at S, whatever order the table has
    them in, and keys before the first level come out as zeros (and have no gradient).  None: one level.  ``weight`` and ``bias`` (C,): ones and zeros if
    None; of any floating type, used in float32 (float64 for float64).  ``act``: None, "relu" or "silu".  Sums are formed in float32 (float64) and results
    rounded once."""
    here = native_for(x)
    if here is not None and (code := _lib.ACTIVATIONS.get(act)) is not None:
        kind = torch.float64 if x.dtype == torch.float64 else torch.float32
        w, b = (t.to(kind) if isinstance(t, torch.Tensor) and t.dtype != kind and t.is_floating_point() else t for t in (weight, bias))
        got = here[0].group_norm(here[1], here[2], x, w, b, level_start_index, num_groups, eps, code)
        if got is not None:
            return got
    if not x.is_cuda:
        raise RuntimeError("x must be a CUDA tensor")
    _lib.dtype_code(x)
    if x.dim() < 2:
        raise RuntimeError(f"x must be (B, ..., C), got {tuple(x.shape)}")
    C = x.shape[-1]
    num_groups = int(num_groups)
    if num_groups <= 0 or C % num_groups:
        raise ValueError(f"num_channels ({C}) must be divisible by num_groups ({num_groups})")
    if act not in _lib.ACTIVATIONS:
        raise ValueError(f"act must be None, 'relu' or 'silu', got {act!r}")
    eps = float(eps)
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    kind = torch.float64 if x.dtype == torch.float64 else torch.float32
    params = []
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is not None:
            if not t.is_floating_point():
                raise RuntimeError(f"{name} has dtype {t.dtype}, expected a floating type")
            check_beside(x, t, name, (C,), t.dtype)
            t = t.to(kind)
        params.append(t)
    if level_start_index is not None:
        if x.dim() != 3:
            raise RuntimeError(f"x must be (B, S, C) beside level_start_index, got {tuple(x.shape)}")
        check_beside(x, level_start_index, "level_start_index", level_start_index.shape, torch.int64)
        if level_start_index.dim() != 1 or not 0 < len(level_start_index) <= _lib.MAX_LEVELS:
            raise RuntimeError(f"level_start_index must hold 1 to {_lib.MAX_LEVELS} levels, got {tuple(level_start_index.shape)}")
    refuse_capture(x, *params)
    return LevelGroupNormFunction.apply(x, *params, level_start_index, num_groups, eps, _lib.ACTIVATIONS[act])
