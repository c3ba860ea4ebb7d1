"""The operators of an encoder's layers on the HIP kernels (csrc/gnnx_norm.hpp, C ABI: include/gnnx.h): what the reference's encoders do between two graph
convolutions (models.py:230-267 ReLU and normalisation, :58-61 the next layer's dropout) and its gradients.

    layer_norm(x, weight, bias, eps, relu)                       y;      differentiable in x, weight, bias
    dropout(x, p, seed, step)                                    y;      differentiable in x
    layer_norm_dropout(x, weight, bias, p, seed, step, ...)      h, d;   h = layer_norm(x), d = dropout(h), one pass forward and one backward
    layer_norm_forward / layer_norm_backward, layer_norm_dropout_forward / layer_norm_dropout_backward
                                                                 the same passes without autograd, for loops that keep their own (mean, rstd)

x is fp32, bf16 or fp16 with any leading dimensions; the last dimension is a row.  weight and bias have one element per column, in fp32 or in x's type; either
may be None.  Arithmetic, statistics and the sums of the parameters' gradients are fp32; results are rounded once.  Rows that are evenly spaced (a slice of the
columns of a wider tensor) are read in place, anything else is copied first.  Outputs are contiguous.

dropout's mask is a function of (seed, step, row, column) - Philox-4x32-10, see include/gnnx.h - and is never stored: the backward pass computes it again, and the
same call gives the same result on every run, stream and shape of launch.  `seed` is an int in [0, 2^63) with `step` in [0, 2^32) counting the uses of that seed, or
an int64 tensor (seed, step) on x's device that the kernel reads when it runs (`step` is then added to the tensor's): a training step captured into a graph
advances that tensor in the graph and draws a new mask at every replay.  row_offset: where x's first row lies in the tensor of which x is a shard.  A dropped
element is 0 whatever it was.

The calls run on the current stream of x's device and can be captured into graphs.  There is no CPU fallback: tensors elsewhere are refused, as are tensors without memory
of their own (sparse, batched, fake, functional) and tensors that carry forward-mode derivatives.  Gradients cannot be differentiated again.  Argument checks, outputs
and the autograd nodes are csrc/gnnx_torch.cpp (a call is a few microseconds of host time); the kernels and the C ABI below it are libgnnx_hip.so."""
import importlib.machinery
import importlib.util
import os

from .engine import GnnxError, library_path

# which build of the library serves the calls: None = libgnnx_hip.so.  The CPU-only tests put the emulator build (a ctypes.CDLL) here, host memory standing in for
# the device's.
_ENGINE = {"lib": None}

_module = None
_serving = False       # the value of _ENGINE["lib"] that _module was last pointed at (False: none yet)


def _load():
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "csrc", "gnnx_torch.so")
    for p in (path, library_path()):
        if not os.path.exists(p):
            raise RuntimeError("%s not found: the HIP extension is not built (run `python __graft_entry__.py`). The operators have no CPU fallback." % p)
    loader = importlib.machinery.ExtensionFileLoader("gnnx_torch", path)
    module = importlib.util.module_from_spec(importlib.util.spec_from_file_location("gnnx_torch", path, loader=loader))
    loader.exec_module(module)
    return module


def _native():
    global _module, _serving
    lib = _ENGINE["lib"]
    if lib is not _serving:
        import torch  # noqa: F401  (the extension links against it)
        if _module is None:
            _module = _load()
        _module.use_library(library_path() if lib is None else lib._name, lib is not None, GnnxError)
        _serving = lib
    return _module


def layer_norm(x, weight=None, bias=None, eps=1e-5, relu=False):
    """y = (v - mean v) / sqrt(var v + eps) * weight + bias over the last dimension, v = relu(x) or x (models.py:222-228 standardises an encoder's rows this way,
    without parameters)."""
    return _native().layer_norm(x, weight, bias, eps, relu)


def dropout(x, p, seed, step=0, row_offset=0):
    """x / (1 - p) where the element stays, 0 where it is dropped (models.py:58-61 with a mask that (seed, step) determine)."""
    return _native().dropout(x, p, seed, step, row_offset)


def layer_norm_dropout(x, weight=None, bias=None, p=0.5, seed=0, step=0, eps=1e-5, relu=False, row_offset=0):
    """(h, d): h = layer_norm(x, weight, bias, eps, relu), d = dropout(h, p, seed, step, row_offset) of the unrounded h."""
    return _native().layer_norm_dropout(x, weight, bias, p, seed, step, eps, relu, row_offset)


def layer_norm_forward(x, weight=None, bias=None, eps=1e-5, relu=False):
    """(y, mean, rstd): layer_norm without autograd, and the rows' statistics (fp32) that layer_norm_backward takes."""
    return _native().layer_norm_forward(x, weight, bias, eps, relu)


def layer_norm_backward(dy, x, mean, rstd, weight=None, relu=False):
    """(dx, dweight, dbias) of layer_norm_forward's y; the last two are None without a weight."""
    return _native().layer_norm_backward(dy, x, mean, rstd, weight, relu)


def layer_norm_dropout_forward(x, weight=None, bias=None, p=0.5, seed=0, step=0, eps=1e-5, relu=False, row_offset=0):
    """(h, d, mean, rstd): layer_norm_dropout without autograd."""
    return _native().layer_norm_dropout_forward(x, weight, bias, p, seed, step, eps, relu, row_offset)


def layer_norm_dropout_backward(dh, dd, x, mean, rstd, weight=None, p=0.5, seed=0, step=0, relu=False, row_offset=0):
    """(dx, dweight, dbias) from the gradients of both outputs of layer_norm_dropout_forward (either may be None); the last two are None without a weight."""
    return _native().layer_norm_dropout_backward(dh, dd, x, mean, rstd, weight, p, seed, step, relu, row_offset)
