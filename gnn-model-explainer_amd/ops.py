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

The calls run on the current stream of x's device and can be captured into graphs.  There is no CPU fallback: tensors elsewhere are refused."""
import ctypes

import torch

from .engine import _check, _Drop, _Norm, get_library

# which build of the library serves the calls: None = libgnnx_hip.so.  The CPU-only tests put the emulator build here, host memory standing in for the device's.
_ENGINE = {"lib": None}

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _library(x):
    lib = _ENGINE["lib"]
    if lib is not None:
        return lib
    if not x.is_cuda:
        raise RuntimeError("the operators run on MI355X only (no CPU fallback): got a tensor on %s" % x.device)
    return get_library()


def _call(x, fn, lib, *args):
    """fn(*args, stream) with x's device current, on its current stream."""
    if not x.is_cuda:
        _check(lib, fn(*args, None))
    elif x.get_device() == torch.cuda.current_device():
        _check(lib, fn(*args, torch.cuda.current_stream().cuda_stream))
    else:
        with torch.cuda.device(x.device):
            _check(lib, fn(*args, torch.cuda.current_stream().cuda_stream))


def _rows(x):
    """x as a matrix over its last dimension -> (tensor, rows, cols, row stride in elements); a copy where its rows are not evenly spaced."""
    cols = x.shape[-1]
    rows = x.numel() // cols if cols else 0
    if x.is_contiguous():
        return x, rows, cols, cols
    if cols == 1 or x.stride(-1) == 1:
        size, step = 1, 0                 # rows so far, from the innermost leading dimension outwards, and their spacing
        for n, st in zip(reversed(x.shape[:-1]), reversed(x.stride()[:-1])):
            if n == 1:
                continue
            if size == 1:
                step = st
            elif st != step * size:
                break
            size *= n
        else:
            return x, rows, cols, step if size > 1 else cols
    return x.contiguous(), rows, cols, cols


def _check_input(name, x):
    if not isinstance(x, torch.Tensor) or x.dtype not in _TYPES:
        raise TypeError("%s must be a float32, bfloat16 or float16 tensor, got %s" % (name, getattr(x, "dtype", type(x).__name__)))
    if x.dim() < 1:
        raise ValueError("%s needs at least one dimension" % name)


def _check_norm(x, weight, bias):
    _check_input("x", x)
    if x.shape[-1] < 1:
        raise ValueError("layer norm over rows of no elements")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if not isinstance(p, torch.Tensor) or p.dtype != x.dtype and p.dtype != torch.float32:
            raise TypeError("%s must be float32 or of x's type %s, got %s" % (name, x.dtype, getattr(p, "dtype", type(p).__name__)))
        if p.shape != (x.shape[-1],):
            raise ValueError("%s must have shape (%d,), got %s" % (name, x.shape[-1], tuple(p.shape)))
        if p.device != x.device:
            raise ValueError("%s is on %s, x on %s" % (name, p.device, x.device))
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError("weight and bias must have one type, got %s and %s" % (weight.dtype, bias.dtype))


def _check_like(name, t, x, shape=None, dtype=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a tensor, got %s" % (name, type(t).__name__))
    if t.shape != (x.shape if shape is None else shape) or t.dtype != (dtype or x.dtype) or t.device != x.device:
        raise ValueError("%s must be %s %s on %s, got %s %s on %s" % (name, tuple(x.shape if shape is None else shape), dtype or x.dtype, x.device,
                                                                      tuple(t.shape), t.dtype, t.device))


def _drop(x, p, seed, step, row_offset):
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError("p must be in [0, 1], got %r" % p)
    if not 0 <= step < 1 << 32:
        raise ValueError("step must be in [0, 2^32), got %r" % step)
    if not 0 <= row_offset < 1 << 62:
        raise ValueError("row_offset must be in [0, 2^62), got %r" % row_offset)
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.shape != (2,) or not seed.is_contiguous() or seed.device != x.device:
            raise ValueError("a seed tensor must be two contiguous int64 (seed, step) on x's device %s, got %s %s on %s" %
                             (x.device, tuple(seed.shape), seed.dtype, seed.device))
        return _Drop(p, 0, seed.data_ptr(), row_offset, step)
    if not 0 <= seed < 1 << 63:
        raise ValueError("seed must be in [0, 2^63), got %r" % seed)
    return _Drop(p, seed, None, row_offset, step)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _param(p):
    return p if p is None or p.is_contiguous() else p.contiguous()


_SHORT = 4096      # rows of no more columns never need scratch of their own


def _workspace(lib, x, rows, cols, backward):
    nb = lib.gnnx_layer_norm_workspace_bytes(_TYPES[x.dtype], rows, cols, backward)
    return torch.empty(nb, dtype=torch.uint8, device=x.device), nb


def _norm_forward(x, weight, bias, eps, relu, drop, stats):
    """-> (y, d or None, mean or None, rstd or None); drop: None or the tuple (p, seed, step, row_offset)"""
    _check_norm(x, weight, bias)
    eps = float(eps)
    if not eps >= 0.0:
        raise ValueError("eps must not be negative, got %r" % eps)
    lib = _library(x)
    d = None if drop is None else _drop(x, *drop)
    xm, rows, cols, stride = _rows(x)
    weight, bias = _param(weight), _param(bias)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    out = None if d is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    mean = rstd = None
    if stats:
        mean = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
        rstd = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    par = weight if weight is not None else bias
    a = _Norm(_TYPES[x.dtype], int(par is not None and par.dtype == torch.float32), rows, cols, stride, 0, 0, xm.data_ptr(), _ptr(weight), _ptr(bias), None, None,
              y.data_ptr(), _ptr(out), None, None, None, _ptr(mean), _ptr(rstd), eps, int(bool(relu)))
    ws, nb = _workspace(lib, x, rows, cols, 0) if cols > _SHORT else (None, 0)
    _call(x, lib.gnnx_layer_norm_forward, lib, a, d, _ptr(ws), nb)
    return y, out, mean, rstd


def _norm_backward(dy, dd, x, mean, rstd, weight, relu, drop, need, param_dtype):
    """-> (dx, dw, db), None where `need` says so"""
    _check_norm(x, weight, None)
    for name, g in (("dy", dy), ("dd", dd)):
        if g is not None:
            _check_like(name, g, x)
    for name, t in (("mean", mean), ("rstd", rstd)):
        _check_like(name, t, x, x.shape[:-1], torch.float32)
    lib = _library(x)
    d = None if dd is None else _drop(x, *drop)
    xm, rows, cols, stride = _rows(x)
    dym, _, _, dys = (None, 0, 0, 0) if dy is None else _rows(dy)
    ddm, _, _, dds = (None, 0, 0, 0) if dd is None else _rows(dd)
    weight, mean, rstd = _param(weight), _param(mean), _param(rstd)
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    dw = torch.empty(cols, dtype=param_dtype, device=x.device) if need[1] else None
    db = torch.empty(cols, dtype=param_dtype, device=x.device) if need[2] else None
    ws, nb = _workspace(lib, x, rows, cols, 1) if need[1] or need[2] or cols > _SHORT else (None, 0)
    a = _Norm(_TYPES[x.dtype], int(param_dtype == torch.float32), rows, cols, stride, dys, dds, xm.data_ptr(), _ptr(weight), None, _ptr(dym), _ptr(ddm),
              None, None, _ptr(dx), _ptr(dw), _ptr(db), mean.data_ptr(), rstd.data_ptr(), 0.0, int(bool(relu)))
    _call(x, lib.gnnx_layer_norm_backward, lib, a, d, _ptr(ws), nb)
    return dx if need[0] else None, dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, relu, drop):
        y, d, mean, rstd = _norm_forward(x, weight, bias, eps, relu, drop, True)
        seed = drop[1] if drop is not None and isinstance(drop[1], torch.Tensor) else None
        ctx.save_for_backward(x, weight, mean, rstd, seed)       # a seed tensor advanced before the backward pass is an error, like any saved tensor
        ctx.relu, ctx.drop = relu, drop if seed is None else (drop[0], None) + drop[2:]
        ctx.param_dtype = weight.dtype if weight is not None else bias.dtype if bias is not None else x.dtype
        ctx.set_materialize_grads(False)
        return y if d is None else (y, d)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dd=None):
        if dy is None and dd is None:
            return None, None, None, None, None, None
        x, weight, mean, rstd, seed = ctx.saved_tensors
        drop = ctx.drop if seed is None else (ctx.drop[0], seed) + ctx.drop[2:]
        return _norm_backward(dy, dd, x, mean, rstd, weight, ctx.relu, drop, ctx.needs_input_grad[:3], ctx.param_dtype) + (None, None, None)


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, step, row_offset):
        ctx.save_for_backward(seed if isinstance(seed, torch.Tensor) else None)
        ctx.p, ctx.seed, ctx.step, ctx.row_offset = p, None if isinstance(seed, torch.Tensor) else seed, step, row_offset
        return _dropout(x, p, seed, step, row_offset)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        seed, = ctx.saved_tensors
        return _dropout(dy, ctx.p, ctx.seed if seed is None else seed, ctx.step, ctx.row_offset), None, None, None, None


def _dropout(x, p, seed, step, row_offset):
    _check_input("x", x)
    lib = _library(x)
    d = _drop(x, p, seed, step, row_offset)
    xm, rows, cols, stride = _rows(x)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    _call(x, lib.gnnx_dropout, lib, _TYPES[x.dtype], rows, cols, xm.data_ptr(), stride, y.data_ptr(), d)
    return y


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(getattr(t, "requires_grad", False) for t in tensors)


def layer_norm(x, weight=None, bias=None, eps=1e-5, relu=False):
    """y = (v - mean v) / sqrt(var v + eps) * weight + bias over the last dimension, v = relu(x) or x (models.py:222-228 standardises an encoder's rows this way,
    without parameters)."""
    if _wants_grad(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, eps, relu, None)
    return _norm_forward(x, weight, bias, eps, relu, None, False)[0]


def dropout(x, p, seed, step=0, row_offset=0):
    """x / (1 - p) where the element stays, 0 where it is dropped (models.py:58-61 with a mask that (seed, step) determine)."""
    if _wants_grad(x):
        return _Dropout.apply(x, p, seed, step, row_offset)
    return _dropout(x, p, seed, step, row_offset)


def layer_norm_dropout(x, weight=None, bias=None, p=0.5, seed=0, step=0, eps=1e-5, relu=False, row_offset=0):
    """(h, d): h = layer_norm(x, weight, bias, eps, relu), d = dropout(h, p, seed, step, row_offset) of the unrounded h."""
    if _wants_grad(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, eps, relu, (p, seed, step, row_offset))
    return _norm_forward(x, weight, bias, eps, relu, (p, seed, step, row_offset), False)[:2]


def layer_norm_forward(x, weight=None, bias=None, eps=1e-5, relu=False):
    """(y, mean, rstd): layer_norm without autograd, and the rows' statistics (fp32) that layer_norm_backward takes."""
    y, _, mean, rstd = _norm_forward(x, weight, bias, eps, relu, None, True)
    return y, mean, rstd


def layer_norm_backward(dy, x, mean, rstd, weight=None, relu=False):
    """(dx, dweight, dbias) of layer_norm_forward's y; the last two are None without a weight."""
    return _norm_backward(dy, None, x, mean, rstd, weight, relu, None, (True, weight is not None, weight is not None), None if weight is None else weight.dtype)


def layer_norm_dropout_forward(x, weight=None, bias=None, p=0.5, seed=0, step=0, eps=1e-5, relu=False, row_offset=0):
    """(h, d, mean, rstd): layer_norm_dropout without autograd."""
    return _norm_forward(x, weight, bias, eps, relu, (p, seed, step, row_offset), True)


def layer_norm_dropout_backward(dh, dd, x, mean, rstd, weight=None, p=0.5, seed=0, step=0, relu=False, row_offset=0):
    """(dx, dweight, dbias) from the gradients of both outputs of layer_norm_dropout_forward (either may be None); the last two are None without a weight."""
    if dh is None and dd is None:
        raise ValueError("dh and dd are both None")
    return _norm_backward(dh, dd, x, mean, rstd, weight, relu, (p, seed, step, row_offset), (True, weight is not None, weight is not None),
                          None if weight is None else weight.dtype)
