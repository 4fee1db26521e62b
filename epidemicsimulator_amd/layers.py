"""Layer operators on torch tensors that live on the GPU: dropout from a counter-based generator (its mask is computed
again where it is needed and never stored), layer normalisation, and both in one pass, with their gradients.

They are what a Q-network is regularised with that replays its buffer many times (linear -> dropout -> layer norm ->
ReLU); the learners of `Agents` run the same kernels inside their networks (`Agents.regularise`).  All arithmetic is in
libepi.so (epi_dropout, epi_layer_norm_forward, epi_layer_norm_backward of include/epi.h); a tensor that is not on a GPU
is refused.  Work is enqueued on torch's current stream of the tensor's device, and every array, the workspaces among
them, is one of torch's, so calls can be captured into a graph (a number as dropout offset is captured with it: every
replay then drops the same units; a tensor's value is read by every replay).  Leading dimensions are rows, the last one the columns;
tensors whose rows are evenly spaced are read where they are, others are copied first.
"""
import ctypes as C
from typing import Optional, Tuple, Union

import torch

from . import _capi
from . import _layers


def _hip_runtimes():
    """The HIP runtimes this process has loaded.  torch brings one of its own: libepi.so uses it where torch came first,
    and loads the system's where it came first itself; devices, streams and memory of two are strangers to each other."""
    with open("/proc/self/maps") as maps:
        return sorted({line.split(None, 5)[5].strip() for line in maps if "libamdhip64.so" in line})


_capi.lib()
if len(_hip_runtimes()) > 1:
    raise ImportError("two HIP runtimes are loaded (%s): import torch, or epidemicsimulator_amd.layers, before the first "
                      "call into libepi.so" % ", ".join(_hip_runtimes()))

__all__ = ["dropout", "layer_norm", "layer_norm_forward", "layer_norm_backward"]

_layers.bind({name: C.cast(getattr(_capi.lib(), name), C.c_void_p).value for name in (
    "epi_dropout", "epi_layer_norm_forward", "epi_layer_norm_backward_workspace", "epi_layer_norm_backward", "epi_last_error")})

Offset = Union[int, torch.Tensor]


def dropout(x: torch.Tensor, p: float, seed: int, offset: Offset = 0) -> torch.Tensor:
    """Each element dropped with probability p (rounded to a multiple of 2^-16), the others multiplied so that the mean
    stays; differentiable.  The mask is a function of (seed, offset, row, column) alone: calls that are to draw
    independently -- layers, steps -- take different offsets or seeds.  `offset` may be a tensor of one int64 on x's
    device, read when the kernels run: a captured graph then drops other elements on every replay if the program
    changes it between replays (not between a forward pass and its backward pass)."""
    return _layers.dropout(x, p, seed, offset)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, dropout: float = 0.0, seed: int = 0, offset: Offset = 0) -> torch.Tensor:
    """(h - mean h) / sqrt(mean (h - mean h)^2 + eps) * weight + bias over the last dimension, with h = x, or
    h = dropout(x, dropout, seed, offset) in the same pass; differentiable in x, weight and bias.  weight and bias hold
    x's type; sums are taken in float32 (float64 for float64) and y is rounded once.  Captured into a graph with its
    backward pass while an eager graph of the same leaves is alive, the call is refused."""
    return _layers.layer_norm(x, weight, bias, eps, dropout, seed, offset)


def layer_norm_forward(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                       eps: float = 1e-5, dropout: float = 0.0, seed: int = 0,
                       offset: Offset = 0) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """layer_norm without autograd: (y, mean, 1 / standard deviation), the latter two one number a row."""
    return _layers.layer_norm_forward(x, weight, bias, eps, dropout, seed, offset)


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: Optional[torch.Tensor], mean: torch.Tensor,
                        rstd: torch.Tensor, dropout: float = 0.0, seed: int = 0,
                        offset: Offset = 0) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, dweight, dbias) from dy and what layer_norm_forward took and gave; without autograd, so it can be captured
    into a graph whatever else holds on to the leaves."""
    return _layers.layer_norm_backward(dy, x, weight, mean, rstd, dropout, seed, offset)
