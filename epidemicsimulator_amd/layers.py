"""Layer operators on torch tensors that live on the GPU: dropout from a counter-based generator (its mask is computed
again where it is needed and never stored), layer normalisation, and both in one pass, with their gradients.

They are what a Q-network is regularised with that replays its buffer many times (linear -> dropout -> layer norm ->
ReLU); the learners of `Agents` run the same kernels inside their networks (`Agents.regularise`).  All arithmetic is in
libepi.so (epi_dropout, epi_layer_norm_forward, epi_layer_norm_backward of include/epi.h); a tensor that is not on a GPU
is refused.  Work is enqueued on torch's current stream of the tensor's device, and every array, the workspaces among
them, is one of torch's, so calls can be captured into a graph.  Leading dimensions are rows, the last one the columns;
tensors whose rows are evenly spaced are read where they are, others are copied first.
"""
import ctypes as C
from typing import Optional, Tuple, Union

import torch

from . import _capi
from ._capi import check, lib

__all__ = ["dropout", "layer_norm", "layer_norm_forward", "layer_norm_backward"]

_DTYPES = {torch.float64: 0, torch.float32: 1, torch.bfloat16: 2, torch.float16: 3}

Offset = Union[int, torch.Tensor]


def _refuse(text, *args):
    raise _capi.EpiError(_capi.EPI_ERR_BAD_ARGUMENT, text % args)


def _check(name, t, like=None):
    if not isinstance(t, torch.Tensor):
        _refuse("%s is a %s, not a tensor", name, type(t).__name__)
    if not t.is_cuda:
        _refuse("%s is on %s: the operators run on the GPU only", name, t.device)
    if like is None:
        if t.dtype not in _DTYPES:
            _refuse("%s holds %s: float64, float32, bfloat16 and float16 are implemented", name, t.dtype)
        if t.dim() < 1 or t.shape[-1] < 1:
            _refuse("%s has the shape %s: at least one column is needed", name, tuple(t.shape))
    else:
        if t.dtype != like.dtype:
            _refuse("%s holds %s, x holds %s", name, t.dtype, like.dtype)
        if t.device != like.device:
            _refuse("%s is on %s, x on %s", name, t.device, like.device)


def _rows(t):
    """(tensor to read, distance of its rows): the tensor itself where its rows are evenly spaced, else a copy."""
    cols = t.shape[-1]
    if t.is_contiguous():
        return t, cols
    if cols == 1 or t.stride(-1) == 1:
        if t.dim() == 1:
            return t, cols
        if t.dim() == 2:
            return t, t.stride(0)
        try:
            return t, t.view(-1, cols).stride(0)
        except RuntimeError:
            pass
    return t.contiguous(), cols


def _vector(name, w, x):
    if w is None:
        return None
    _check(name, w, x)
    if w.shape != x.shape[-1:]:
        _refuse("%s has the shape %s for %d columns", name, tuple(w.shape), x.shape[-1])
    return w if w.is_contiguous() else w.contiguous()


def _desc(x, eps, p, seed, offset):
    d = _capi.LayerDesc()
    d.cols = x.shape[-1]
    d.rows = x.numel() // d.cols
    d.eps = eps
    d.dropout = p
    d.seed = seed
    if isinstance(offset, torch.Tensor):
        if not offset.is_cuda or offset.device != x.device or offset.dtype != torch.int64 or offset.numel() != 1:
            _refuse("offset is a number, or a tensor of one int64 on %s", x.device)
        d.offset_dev = offset.data_ptr()
    else:
        d.offset = offset
    d.dtype = _DTYPES[x.dtype]
    d.device = x.device.index
    return d


def _stream(x):
    return torch._C._cuda_getCurrentRawStream(x.device.index)


def _ptr(t):
    return None if t is None else t.data_ptr()


# ------------------------------------------------------------------------------------------------
# dropout
# ------------------------------------------------------------------------------------------------
def _dropout(x, p, seed, offset):
    x, stride = _rows(x)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    d = _desc(x, 0.0, p, seed, offset)
    d.x_stride, d.y_stride = stride, d.cols
    check(lib().epi_dropout(C.byref(d), x.data_ptr(), y.data_ptr(), _stream(x)))
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, offset):
        ctx.args = (p, seed)
        if isinstance(offset, torch.Tensor):
            ctx.save_for_backward(offset)
        else:
            ctx.offset = offset
        return _dropout(x, p, seed, offset)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        offset = ctx.saved_tensors[0] if ctx.saved_tensors else ctx.offset
        return _dropout(dy, *ctx.args, offset), None, None, None


def dropout(x: torch.Tensor, p: float, seed: int, offset: Offset = 0) -> torch.Tensor:
    """Each element dropped with probability p (rounded to a multiple of 2^-16), the others multiplied so that the mean
    stays; differentiable.  The mask is a function of (seed, offset, row, column) alone: calls that are to draw
    independently -- layers, steps -- take different offsets or seeds.  `offset` may be a tensor of one int64 on x's
    device, read when the kernels run: a captured graph then drops other elements on every replay if the program
    changes it between replays (not between a forward pass and its backward pass)."""
    _check("x", x)
    if torch.is_grad_enabled() and x.requires_grad:
        return _Dropout.apply(x, p, seed, offset)
    return _dropout(x, p, seed, offset)


# ------------------------------------------------------------------------------------------------
# layer norm
# ------------------------------------------------------------------------------------------------
def _norm_forward(x, weight, bias, eps, p, seed, offset, stats):
    x, stride = _rows(x)
    weight, bias = _vector("weight", weight, x), _vector("bias", bias, x)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    d = _desc(x, eps, p, seed, offset)
    d.x_stride, d.y_stride = stride, d.cols
    mean = rstd = None
    if stats:
        both = torch.empty((2, d.rows), dtype=torch.float64 if d.dtype == 0 else torch.float32, device=x.device)
        mean, rstd = both[0], both[1]
    check(lib().epi_layer_norm_forward(C.byref(d), x.data_ptr(), _ptr(weight), _ptr(bias), y.data_ptr(), _ptr(mean),
                                       _ptr(rstd), _stream(x)))
    return y, mean, rstd


def _norm_backward(dy, x, weight, mean, rstd, p, seed, offset, want):
    x, stride = _rows(x)
    dy, dy_stride = _rows(dy)
    weight = _vector("weight", weight, x)
    d = _desc(x, 0.0, p, seed, offset)
    d.x_stride, d.dy_stride, d.y_stride = stride, dy_stride, d.cols
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if want[0] else None
    dweight = torch.empty(x.shape[-1:], dtype=x.dtype, device=x.device) if want[1] else None
    dbias = torch.empty(x.shape[-1:], dtype=x.dtype, device=x.device) if want[2] else None
    need = C.c_size_t(0)
    check(lib().epi_layer_norm_backward_workspace(C.byref(d), C.byref(need)))
    work = torch.empty(need.value, dtype=torch.uint8, device=x.device) if need.value else None
    check(lib().epi_layer_norm_backward(C.byref(d), x.data_ptr(), dy.data_ptr(), _ptr(weight), mean.data_ptr(),
                                        rstd.data_ptr(), _ptr(dx), _ptr(dweight), _ptr(dbias), _ptr(work), need,
                                        _stream(x)))
    return dx, dweight, dbias


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, p, seed, offset):
        y, mean, rstd = _norm_forward(x, weight, bias, eps, p, seed, offset, True)
        ctx.args = (p, seed)
        on_device = isinstance(offset, torch.Tensor)
        ctx.offset = None if on_device else offset
        ctx.save_for_backward(x, weight, mean, rstd, offset if on_device else None)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd, offset = ctx.saved_tensors
        grads = _norm_backward(dy, x, weight, mean, rstd, *ctx.args, ctx.offset if offset is None else offset,
                               ctx.needs_input_grad[:3])
        return grads + (None, None, None, None)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, dropout: float = 0.0, seed: int = 0, offset: Offset = 0) -> torch.Tensor:
    """(h - mean h) / sqrt(mean (h - mean h)^2 + eps) * weight + bias over the last dimension, with h = x, or
    h = dropout(x, dropout, seed, offset) in the same pass; differentiable in x, weight and bias.  weight and bias hold
    x's type; sums are taken in float32 (float64 for float64) and y is rounded once."""
    _check("x", x)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return _LayerNorm.apply(x, weight, bias, eps, dropout, seed, offset)
    return _norm_forward(x, weight, bias, eps, dropout, seed, offset, False)[0]


def layer_norm_forward(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                       eps: float = 1e-5, dropout: float = 0.0, seed: int = 0,
                       offset: Offset = 0) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """layer_norm without autograd: (y, mean, 1 / standard deviation), the latter two one number a row."""
    _check("x", x)
    with torch.no_grad():
        return _norm_forward(x, weight, bias, eps, dropout, seed, offset, True)


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: Optional[torch.Tensor], mean: torch.Tensor,
                        rstd: torch.Tensor, dropout: float = 0.0, seed: int = 0,
                        offset: Offset = 0) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, dweight, dbias) from dy and what layer_norm_forward took and gave; without autograd, so it can be captured
    into a graph whatever else holds on to the leaves."""
    _check("x", x)
    _check("dy", dy, x)
    if dy.shape != x.shape:
        _refuse("dy has the shape %s, x %s", tuple(dy.shape), tuple(x.shape))
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    for name, t in (("mean", mean), ("rstd", rstd)):
        if not isinstance(t, torch.Tensor) or t.dtype != wide or t.device != x.device or not t.is_contiguous() \
                or t.numel() != x.numel() // x.shape[-1]:
            _refuse("%s is not the forward pass's: %d numbers of %s on %s", name, x.numel() // x.shape[-1], wide, x.device)
    with torch.no_grad():
        return _norm_backward(dy, x, weight, mean, rstd, dropout, seed, offset, (True, True, True))
