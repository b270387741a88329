"""The attribute network over the C ABI: a small network whose outputs are Gaussian attributes (or changes of them)
and the operators it is built from. No counterpart in the reference.

  LayerOps          linear layers with bias, activation and residual, layer norm, and their gradients: one call each
                    on the caller's tensors
  AttributeNetwork  features -> linear -> [layer norm -> linear, activation -> linear + residual] x blocks ->
                    layer norm -> linear -> attributes, forward and backward over every Gaussian

Matrices are 2-D tensors of one dtype (float32, float16 or bfloat16) whose rows' elements lie next to each other;
rows may lie further apart (a column range of a wider tensor). Vectors are packed float32.
"""
from __future__ import annotations

import ctypes as C
import math

from . import _lib

ACTIVATIONS = {"none": _lib.TGS_ACTIVATION_NONE, "relu": _lib.TGS_ACTIVATION_RELU,
               "silu": _lib.TGS_ACTIVATION_SILU, "gelu": _lib.TGS_ACTIVATION_GELU}

_DTYPES = None


def _dtypes():
    global _DTYPES
    if _DTYPES is None:
        import torch
        _DTYPES = {torch.float32: _lib.TGS_DTYPE_FLOAT32, torch.float16: _lib.TGS_DTYPE_FLOAT16,
                   torch.bfloat16: _lib.TGS_DTYPE_BFLOAT16}
    return _DTYPES


def matrix(t, name: str) -> _lib.tgs_matrix:
    """The C ABI's view of a 2-D tensor; raises for tensors that it cannot address."""
    shape = t.shape
    if len(shape) != 2:
        raise RuntimeError(f"{name}: a matrix has two dimensions, not {len(shape)}")
    rows, cols = shape
    step, unit = t.stride()
    if unit != 1 and cols > 1:
        raise RuntimeError(f"{name}: the elements of a row must lie next to each other")
    dtype = (_DTYPES or _dtypes()).get(t.dtype)
    if dtype is None:
        raise RuntimeError(f"{name}: only float32, float16 and bfloat16 are supported")
    if not t.is_cuda:
        raise RuntimeError(f"{name}: not on the device")
    # the stride of a single row says nothing
    return _lib.tgs_matrix(t.data_ptr(), rows, cols, step if rows > 1 else cols, dtype)


def _vector(t, n: int, name: str):
    """The address of a packed float32 vector of n elements on the device, or None."""
    if t is None:
        return None
    if t.dim() != 1 or t.shape[0] != n or t.dtype is not _float32() or (n > 1 and t.stride(0) != 1) or not t.is_cuda:
        raise RuntimeError(f"{name}: a packed float32 vector of {n} elements on the device is needed")
    return t.data_ptr()


_FLOAT32 = None


def _float32():
    global _FLOAT32
    if _FLOAT32 is None:
        import torch
        _FLOAT32 = torch.float32
    return _FLOAT32


class LayerOps:
    """The layer operators on one handle, which owns their workspace: its calls run on one stream, or the caller
    orders them. `stream` is a torch.cuda.Stream, or None for the current one; outputs that are not given are
    allocated on it. Inputs made on another stream are the caller's to order, as for any kernel."""

    def __init__(self):
        h = C.c_void_p()
        self._lib = _lib.load()
        _lib.check(self._lib.tgs_network_create(C.byref(h)), "LayerOps")
        self._h = h
        self._current = None

    def __del__(self):
        h = getattr(self, "_h", None)
        if h is not None and h.value:
            try:
                self._lib.tgs_network_destroy(h)
            except Exception:
                pass
            self._h = None

    @staticmethod
    def _empty(stream, like, shape, dtype=None):
        if stream is None:
            return like.new_empty(shape, dtype=dtype)
        import torch
        with torch.cuda.stream(stream):
            return like.new_empty(shape, dtype=dtype)

    def _stream(self, stream, like):
        if stream is not None:
            return stream.cuda_stream
        if self._current is None:
            import torch
            # the stream's address without the Stream object around it: 0.1 us a call against 2.8
            raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
            self._current = raw or (lambda device: torch.cuda.current_stream(device).cuda_stream)
        return self._current(like.device.index)

    def linear(self, x, weight, bias=None, activation: str = "none", residual=None, keep_preact: bool = False,
               out=None, preact=None, stream=None):
        """act(x weight^T + bias) + residual; with keep_preact (or preact given) also the values before the
        activation, which linear_backward takes. out may be residual itself."""
        rows, outs = x.shape[0], weight.shape[0]
        if out is None:
            out = self._empty(stream, x, (rows, outs))
        if preact is None and keep_preact:
            preact = self._empty(stream, x, (rows, outs))
        act = ACTIVATIONS.get(activation)
        if act is None:
            raise RuntimeError(f"linear: unknown activation: {activation}")
        rc = self._lib.tgs_linear_forward(
            self._h, matrix(x, "x"), matrix(weight, "weight"), _vector(bias, outs, "bias"), act,
            None if residual is None else matrix(residual, "residual"),
            None if preact is None else matrix(preact, "preact"), matrix(out, "out"), self._stream(stream, x))
        if rc:
            _lib.check(rc, "linear")
        return out if preact is None else (out, preact)

    def linear_backward(self, grad_y, x, weight, preact=None, activation: str = "none", need_x: bool = True,
                        need_weight: bool = True, need_bias: bool = True, grad_x=None, grad_weight=None,
                        grad_bias=None, stream=None):
        """(grad_x, grad_weight, grad_bias) of linear for grad_y; None where not needed. The residual's gradient is
        grad_y itself. Gradients are assigned, not accumulated."""
        if need_x and grad_x is None:
            grad_x = self._empty(stream, x, x.shape)
        if need_weight and grad_weight is None:
            grad_weight = self._empty(stream, weight, weight.shape)
        if need_bias and grad_bias is None:
            grad_bias = self._empty(stream, x, (weight.shape[0],), _float32())
        act = ACTIVATIONS.get(activation)
        if act is None:
            raise RuntimeError(f"linear_backward: unknown activation: {activation}")
        if act and preact is None:
            raise RuntimeError("linear_backward: an activation's gradient needs preact")
        rc = self._lib.tgs_linear_backward(
            self._h, matrix(grad_y, "grad_y"), matrix(x, "x"), matrix(weight, "weight"),
            matrix(preact, "preact") if act else None, act, None if grad_x is None else matrix(grad_x, "grad_x"),
            None if grad_weight is None else matrix(grad_weight, "grad_weight"),
            _vector(grad_bias, weight.shape[0], "grad_bias"), self._stream(stream, x))
        if rc:
            _lib.check(rc, "linear_backward")
        return grad_x, grad_weight, grad_bias

    def layer_norm(self, x, gamma=None, beta=None, eps: float = 1e-5, out=None, mean=None, rstd=None, stream=None):
        """((x - mean) rstd gamma + beta, mean, rstd) over each row. out may be x itself."""
        rows, n = x.shape
        if out is None:
            out = self._empty(stream, x, (rows, n))
        if mean is None:
            mean = self._empty(stream, x, (rows,), _float32())
        if rstd is None:
            rstd = self._empty(stream, x, (rows,), _float32())
        rc = self._lib.tgs_layer_norm_forward(
            self._h, matrix(x, "x"), _vector(gamma, n, "gamma"), _vector(beta, n, "beta"), eps, matrix(out, "out"),
            _vector(mean, rows, "mean"), _vector(rstd, rows, "rstd"), self._stream(stream, x))
        if rc:
            _lib.check(rc, "layer_norm")
        return out, mean, rstd

    def layer_norm_backward(self, grad_y, x, gamma, mean, rstd, residual_grad=None, grad_x=None, grad_gamma=None,
                            grad_beta=None, stream=None):
        """(grad_x, grad_gamma, grad_beta) of layer_norm for grad_y; grad_x includes residual_grad, the gradient that
        reaches x past the norm. grad_x may be grad_y or residual_grad itself."""
        rows, n = x.shape
        if grad_x is None:
            grad_x = self._empty(stream, x, (rows, n))
        if grad_gamma is None:
            grad_gamma = self._empty(stream, x, (n,), _float32())
        if grad_beta is None:
            grad_beta = self._empty(stream, x, (n,), _float32())
        rc = self._lib.tgs_layer_norm_backward(
            self._h, matrix(grad_y, "grad_y"), matrix(x, "x"), _vector(gamma, n, "gamma"),
            _vector(mean, rows, "mean"), _vector(rstd, rows, "rstd"),
            None if residual_grad is None else matrix(residual_grad, "residual_grad"), matrix(grad_x, "grad_x"),
            _vector(grad_gamma, n, "grad_gamma"), _vector(grad_beta, n, "grad_beta"), self._stream(stream, x))
        if rc:
            _lib.check(rc, "layer_norm_backward")
        return grad_x, grad_gamma, grad_beta
