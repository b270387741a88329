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


class AttributeNetwork:
    """A network over the Gaussians: features [n, inputs] -> attributes [n, outputs].

    h = features w_in^T + b_in; blocks times h = h + act(norm(h) w_1^T + b_1) w_2^T + b_2; attributes =
    norm(h) w_out^T + b_out. norm is a layer norm with its own gamma and beta. The last matrix starts at zero, so an
    untrained network changes nothing.

    weights are the float32 matrices that an optimiser updates: net.optimizer(), which is create_optimizer("muon",
    net.weights, net.grads, copies=net.copies). For a half dtype the products read net.copies, which Muon writes in its
    step: an optimiser that is not given them changes nothing that forward reads. vectors and vector_grads hold all
    biases, gammas and betas, and their gradients, as one float32 vector each, for an optimiser of vectors. backward
    assigns every gradient."""

    def __init__(self, inputs: int, outputs: int, width: int = 256, hidden: int | None = None, blocks: int = 2,
                 activation: str = "gelu", dtype=None, seed: int = 0, eps: float = 1e-5, device: str = "cuda"):
        import torch
        if activation not in ACTIVATIONS:
            raise RuntimeError(f"AttributeNetwork: unknown activation: {activation}")
        hidden = width if hidden is None else hidden
        if min(inputs, outputs, width, hidden) < 1 or blocks < 0:
            raise RuntimeError("AttributeNetwork: sizes must be positive")
        self.dtype = torch.float32 if dtype is None else dtype
        if self.dtype not in _dtypes():
            raise RuntimeError("AttributeNetwork: only float32, float16 and bfloat16 are supported")
        self.inputs, self.outputs, self.activation, self.eps = inputs, outputs, activation, float(eps)
        shapes = [(width, inputs)] + [(hidden, width), (width, hidden)] * blocks + [(outputs, width)]
        g = torch.Generator().manual_seed(seed)
        self.weights = [(torch.randn(o, i, generator=g) / math.sqrt(i)).to(device) for o, i in shapes]
        self.weights[-1].zero_()
        half = self.dtype != torch.float32
        self.copies = [w.to(self.dtype) for w in self.weights] if half else None
        self.grads = [torch.zeros(s, dtype=self.dtype, device=device) for s in shapes]
        # the vectors: a bias for every matrix, then gamma and beta of the blocks' norms and the last one
        sizes = [o for o, _ in shapes] + [width, width] * (blocks + 1)
        self.vectors = torch.zeros(sum(sizes), device=device)
        self.vector_grads = torch.zeros_like(self.vectors)
        views, grads = self.vectors.split(sizes), self.vector_grads.split(sizes)
        m = len(shapes)
        self.biases, self.bias_grads = views[:m], grads[:m]
        self.norms = list(zip(views[m::2], views[m + 1::2]))
        self.norm_grads = list(zip(grads[m::2], grads[m + 1::2]))
        for gamma, _ in self.norms:
            gamma.fill_(1.0)
        self.blocks = blocks
        self.ops = LayerOps()
        self._kept = None

    def optimizer(self):
        """Muon on the matrices, which also writes the half-precision copies."""
        from .optim import Muon
        return Muon(self.weights, self.grads, copies=self.copies)

    def matrices(self):
        """The matrices that the products read."""
        return self.weights if self.copies is None else self.copies

    def forward(self, features, keep: bool = True, stream=None):
        """The attributes, in the network's dtype. keep: hold what backward needs (until the next forward)."""
        ops, w = self.ops, self.matrices()
        self._kept = None
        h = ops.linear(features, w[0], self.biases[0], stream=stream)
        kept = [features]
        for k in range(self.blocks):
            n, mean, rstd = ops.layer_norm(h, *self.norms[k], eps=self.eps, stream=stream)
            up, down = 1 + 2 * k, 2 + 2 * k
            a = ops.linear(n, w[up], self.biases[up], activation=self.activation, keep_preact=keep, stream=stream)
            a, z = a if keep else (a, None)
            if keep:
                kept.append((h, n, mean, rstd, a, z))
            # without a backward the block's input is not needed again: its sum takes its place
            h = ops.linear(a, w[down], self.biases[down], residual=h, out=None if keep else h, stream=stream)
        n, mean, rstd = ops.layer_norm(h, *self.norms[-1], eps=self.eps, stream=stream)
        if keep:
            kept.append((h, n, mean, rstd))
            self._kept = kept
        return ops.linear(n, w[-1], self.biases[-1], stream=stream)

    def backward(self, grad_attributes, need_features: bool = False, stream=None):
        """Fills grads and vector_grads for dL/dattributes (in the network's dtype) of the last forward; returns
        dL/dfeatures where needed."""
        if self._kept is None:
            raise RuntimeError("AttributeNetwork::backward: no forward that kept its values")
        ops, w, kept = self.ops, self.matrices(), self._kept
        act = self.activation
        h, n, mean, rstd = kept[-1]
        g, _, _ = ops.linear_backward(grad_attributes, n, w[-1], grad_weight=self.grads[-1],
                                      grad_bias=self.bias_grads[-1], stream=stream)
        gg, gb = self.norm_grads[-1]
        g, _, _ = ops.layer_norm_backward(g, h, self.norms[-1][0], mean, rstd, grad_x=g, grad_gamma=gg, grad_beta=gb,
                                          stream=stream)
        for k in reversed(range(self.blocks)):
            h, n, mean, rstd, a, z = kept[1 + k]
            up, down = 1 + 2 * k, 2 + 2 * k
            ga, _, _ = ops.linear_backward(g, a, w[down], grad_weight=self.grads[down],
                                           grad_bias=self.bias_grads[down], stream=stream)
            gn, _, _ = ops.linear_backward(ga, n, w[up], preact=z, activation=act, grad_weight=self.grads[up],
                                           grad_bias=self.bias_grads[up], stream=stream)
            gg, gb = self.norm_grads[k]
            # the residual path's gradient joins the norm's
            g, _, _ = ops.layer_norm_backward(gn, h, self.norms[k][0], mean, rstd, residual_grad=g, grad_x=g,
                                              grad_gamma=gg, grad_beta=gb, stream=stream)
        gx, _, _ = ops.linear_backward(g, kept[0], w[0], need_x=need_features, grad_weight=self.grads[0],
                                       grad_bias=self.bias_grads[0], stream=stream)
        return gx


def encode_positions(means, octaves: int = 10, dtype=None):
    """Positions [n, 3] with the sines and cosines of their multiples by 2^0 .. 2^(octaves - 1): [n, 3 + 6 octaves],
    the usual input of a network over positions."""
    import torch
    scaled = means[:, None, :] * (2.0 ** torch.arange(octaves, device=means.device))[None, :, None]
    scaled = scaled.reshape(means.shape[0], 3 * octaves)
    out = torch.cat([means, torch.sin(scaled), torch.cos(scaled)], dim=1)
    return out if dtype is None else out.to(dtype)
