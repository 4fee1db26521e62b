"""Layer operators on torch tensors that live on the GPU: dropout from a counter-based generator (its mask is computed
again where it is needed and never stored), layer normalisation, and both in one pass, with their gradients.

They are what a Q-network is regularised with that replays its buffer many times (linear -> dropout -> layer norm ->
ReLU); the learners of `Agents` run the same kernels inside their networks (`Agents.regularise`).  All arithmetic is in
libepi.so (epi_dropout, epi_layer_norm_forward, epi_layer_norm_backward of include/epi.h); a tensor that is not on a GPU
is refused.  Work is enqueued on torch's current stream of the tensor's device, and every array, the workspaces among
them, is one of torch's, so calls can be captured into a graph (a number as dropout offset is captured with it: every
replay then drops the same units; a tensor's value is read by every replay).  Leading dimensions are rows, the last
one the columns; tensors whose rows are evenly spaced over all leading dimensions are read where they are, others (a
dimension expanded inside of one that moves, columns apart) are copied first.  Derivatives are taken backwards only, and
once: tensors with a tangent, and second derivatives, are refused.
"""
import ctypes as C

import torch  # noqa: F401  (before libepi.so: the two share torch's HIP runtime)

from . import _capi
from . import _layers
from ._layers import dropout, layer_norm, layer_norm_backward, layer_norm_forward

__all__ = ["dropout", "layer_norm", "layer_norm_forward", "layer_norm_backward"]


def _hip_runtimes():
    """The HIP runtimes this process has loaded.  torch brings one of its own: libepi.so uses it where torch came first,
    and loads the system's where it came first itself; devices, streams and memory of two are strangers to each other."""
    with open("/proc/self/maps") as maps:
        return sorted({line.split(None, 5)[5].strip() for line in maps if "libamdhip64.so" in line})


_capi.lib()
if len(_hip_runtimes()) > 1:
    raise ImportError("two HIP runtimes are loaded (%s): import torch, or epidemicsimulator_amd.layers, before the first "
                      "call into libepi.so" % ", ".join(_hip_runtimes()))

_layers.bind({name: C.cast(getattr(_capi.lib(), name), C.c_void_p).value for name in (
    "epi_dropout", "epi_layer_norm_forward", "epi_layer_norm_backward_workspace", "epi_layer_norm_backward", "epi_last_error")})
