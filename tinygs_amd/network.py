"""The attribute network over the C ABI: a small network whose outputs are Gaussian attributes (or changes of them)
and the operators it is built from. No counterpart in the reference.

  LayerOps          linear layers with bias, activation and residual, layer norm, attention to an encoder's states,
                    norms of its heads with turned pairs, and their gradients: one call each on the caller's tensors
  AttributeNetwork  features -> linear -> [attention to states + residual -> layer norm -> linear, activation ->
                    linear + residual] x blocks -> layer norm -> linear -> attributes, forward and backward over every
                    Gaussian; the attention is there where the network has a context

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

    def attention(self, q, k, v, heads: int, kv_heads: int | None = None, batch: int = 1, mask=None,
                  scale: float | None = None, keep_lse: bool = False, out=None, lse=None, stream=None):
        """softmax(scale q k^T) v for each head over the states that exist; with keep_lse (or lse given) also the
        logarithms of the weights' sums [rows, heads], which attention_backward takes.

        q [batch x queries, heads d]; k and v [batch x states, kv_heads d], d up to 128; heads share those of the
        states in equal groups. mask [batch, states] (bool or uint8): False where a state does not exist; it may hold
        anything then. Rows without a state are 0, their lse -inf. scale: 1 / sqrt(d) unless given."""
        rows = q.shape[0]
        if out is None:
            out = self._empty(stream, q, q.shape)
        if lse is None and keep_lse:
            # heads of rows: neighbouring rows' are written together
            lse = self._empty(stream, q, (heads, rows), _float32()).t()
        tensors = (matrix(q, "q"), matrix(k, "k"), matrix(v, "v"))
        a = self._attention(q, k, heads, kv_heads, batch, mask, scale)
        _on_one_device("q k v mask out lse", q, k, v, mask, out, lse)
        rc = self._lib.tgs_attention_forward(self._h, *tensors, a, matrix(out, "out"), *_lse(lse, rows, heads),
                                             self._stream(stream, q))
        if rc:
            _lib.check(rc, "attention")
        return out if lse is None else (out, lse)

    def attention_backward(self, grad_out, q, k, v, out, lse, heads: int, kv_heads: int | None = None, batch: int = 1,
                           mask=None, scale: float | None = None, need_q: bool = True, need_k: bool = True,
                           need_v: bool = True, grad_q=None, grad_k=None, grad_v=None, stream=None):
        """(grad_q, grad_k, grad_v) of attention for grad_out, from its out and lse; None where not needed. Gradients
        are assigned, zeros for states that do not exist."""
        if need_q and grad_q is None:
            grad_q = self._empty(stream, q, q.shape)
        if need_k and grad_k is None:
            grad_k = self._empty(stream, k, k.shape)
        if need_v and grad_v is None:
            grad_v = self._empty(stream, v, v.shape)
        tensors = (matrix(grad_out, "grad_out"), matrix(q, "q"), matrix(k, "k"), matrix(v, "v"), matrix(out, "out"))
        a = self._attention(q, k, heads, kv_heads, batch, mask, scale)
        _on_one_device("grad_out q k v out lse mask grad_q grad_k grad_v", grad_out, q, k, v, out, lse, mask, grad_q,
                       grad_k, grad_v)
        rc = self._lib.tgs_attention_backward(
            self._h, *tensors, *_lse(lse, q.shape[0], heads), a, None if grad_q is None else matrix(grad_q, "grad_q"),
            None if grad_k is None else matrix(grad_k, "grad_k"), None if grad_v is None else matrix(grad_v, "grad_v"),
            self._stream(stream, q))
        if rc:
            _lib.check(rc, "attention_backward")
        return grad_q, grad_k, grad_v

    @staticmethod
    def _attention(q, k, heads, kv_heads, batch, mask, scale):
        kv_heads = heads if kv_heads is None else kv_heads
        if scale is None:
            scale = math.sqrt(heads / max(q.shape[1], 1)) if heads > 0 else 0.0
        at, step = None, 0
        if mask is not None:
            if mask.dim() != 2 or mask.shape[0] != batch or mask.shape[0] * mask.shape[1] != k.shape[0]:
                raise RuntimeError(f"mask: [batch, states] is needed, not {list(mask.shape)}")
            if mask.element_size() != 1 or mask.is_floating_point() or (mask.shape[1] > 1 and mask.stride(1) != 1):
                raise RuntimeError("mask: packed rows of bool or uint8 are needed")
            at, step = mask.data_ptr(), mask.stride(0)
        return _lib.tgs_attention(batch, heads, kv_heads, scale, at, step)

    def head_norm(self, x, heads: int, gamma=None, positions=None, frequencies=None, eps: float = 1e-6, out=None,
                  stream=None):
        """x / sqrt(mean(x^2) + eps) gamma over each head of d = columns / heads (up to 256) columns; with positions
        [rows, axes] and frequencies [pairs, axes] (float32, up to 4 axes, up to d / 2 pairs) the pairs (2 i, 2 i + 1)
        of every head are then turned by the angle positions . frequencies[i]. gamma [d] is shared by the heads.
        out may be x itself."""
        if out is None:
            out = self._empty(stream, x, x.shape)
        at = matrix(x, "x")
        turn = _turn(positions, frequencies)
        _on_one_device("x gamma positions frequencies out", x, gamma, positions, frequencies, out)
        rc = self._lib.tgs_head_norm_forward(self._h, at, heads, _vector(gamma, x.shape[1] // max(heads, 1), "gamma"),
                                             turn, eps, matrix(out, "out"), self._stream(stream, x))
        if rc:
            _lib.check(rc, "head_norm")
        return out

    def head_norm_backward(self, grad_y, x, heads: int, gamma=None, positions=None, frequencies=None,
                           eps: float = 1e-6, need_x: bool = True, grad_x=None, grad_gamma=None, stream=None):
        """(grad_x, grad_gamma) of head_norm for grad_y; grad_gamma is None where there is no gamma. Positions and
        frequencies get no gradient. grad_x may be grad_y itself."""
        if need_x and grad_x is None:
            grad_x = self._empty(stream, x, x.shape)
        d = x.shape[1] // max(heads, 1)
        if gamma is not None and grad_gamma is None:
            grad_gamma = self._empty(stream, x, (d,), _float32())
        at = (matrix(grad_y, "grad_y"), matrix(x, "x"))
        turn = _turn(positions, frequencies)
        _on_one_device("grad_y x gamma positions frequencies grad_x grad_gamma", grad_y, x, gamma, positions,
                       frequencies, grad_x, grad_gamma)
        rc = self._lib.tgs_head_norm_backward(self._h, *at, heads, _vector(gamma, d, "gamma"), turn, eps,
                                              None if grad_x is None else matrix(grad_x, "grad_x"),
                                              _vector(grad_gamma, d, "grad_gamma"), self._stream(stream, x))
        if rc:
            _lib.check(rc, "head_norm_backward")
        return grad_x, grad_gamma


_CURRENT = None


def _current_device() -> int:
    global _CURRENT
    if _CURRENT is None:
        import torch
        torch.cuda.current_device()   # initialises
        # without the checks around it, which take longer than the question
        _CURRENT = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
    return _CURRENT()


def _on_one_device(names: str, *tensors):
    """All on the current device, whose streams and workspaces a handle uses."""
    current = _current_device()
    for i, t in enumerate(tensors):
        if t is not None and t.get_device() != current:
            raise RuntimeError(f"{names.split()[i]}: not on the current device")


def _lse(t, rows: int, heads: int):
    """Address and steps of a float32 [rows, heads] tensor, in rows of heads or heads of rows."""
    if t is None:
        return None, 1, 1
    if t.shape != (rows, heads) or t.dtype is not _float32() or not t.is_cuda:
        raise RuntimeError(f"lse: float32 [{rows}, {heads}] on the device is needed")
    # the step of a single row or head says nothing
    return t.data_ptr(), t.stride(0) if rows > 1 else 1, t.stride(1) if heads > 1 else 1


def _turn(positions, frequencies):
    if positions is None and frequencies is None:
        return None
    if positions is None or frequencies is None:
        raise RuntimeError("head_norm: positions and frequencies come together")
    return _lib.tgs_turn(matrix(positions, "positions"), matrix(frequencies, "frequencies"))


class AttributeNetwork:
    """A network over the Gaussians: features [n, inputs] -> attributes [n, outputs].

    h = features w_in^T + b_in; blocks times h = h + act(norm(h) w_1^T + b_1) w_2^T + b_2; attributes =
    norm(h) w_out^T + b_out. norm is a layer norm with its own gamma and beta. The last matrix starts at zero, so an
    untrained network changes nothing.

    With context (the columns of an encoder's states) each block first attends to the states: h = h +
    attention(q, k, v) w_o^T + b_o with q of norm(h), k and v of the states, each a linear layer, and a head norm on q
    and k. heads divide width (heads of at most 128), kv_heads divide heads. With axes (1 to 4) forward takes positions of
    the rows and of the states, and the head norms turn queries and keys by them: scores then depend on where a state
    lies from a row. extent is the positions' usual size: the slowest pairs turn once over it, the fastest 64 times.

    weights are the float32 matrices that an optimiser updates: net.optimizer(), which is create_optimizer("muon",
    net.weights, net.grads, copies=net.copies). For a half dtype the products read net.copies, which Muon writes in its
    step: an optimiser that is not given them changes nothing that forward reads. vectors and vector_grads hold all
    biases, gammas and betas, and their gradients, as one float32 vector each, for an optimiser of vectors. backward
    assigns every gradient; clip bounds their norm together."""

    def __init__(self, inputs: int, outputs: int, width: int = 256, hidden: int | None = None, blocks: int = 2,
                 activation: str = "gelu", dtype=None, seed: int = 0, eps: float = 1e-5, device: str = "cuda",
                 context: int | None = None, heads: int = 4, kv_heads: int | None = None, axes: int = 0,
                 extent: float = 1.0):
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
        sizes = [o for o, _ in shapes] + [width, width] * (blocks + 1)
        m, self.last = len(shapes), len(shapes) - 1
        self.context, self.heads, self.kv_heads, self.axes = context, heads, heads if kv_heads is None else kv_heads, axes
        if context is not None:
            head = self._check_context(width, extent)
            # after the others': the matrices of q, k, v and the output; their biases, the norm, the head norms' gammas
            kv = self.kv_heads * head
            attending = [(width, width), (kv, context), (kv, context), (width, width)] * blocks
            sizes = sizes + [o for o, _ in attending] + [width, width, head, head] * blocks
            shapes = shapes + attending
        g = torch.Generator().manual_seed(seed)
        self.weights = [(torch.randn(o, i, generator=g) / math.sqrt(i)).to(device) for o, i in shapes]
        self.weights[self.last].zero_()
        half = self.dtype != torch.float32
        self.copies = [w.to(self.dtype) for w in self.weights] if half else None
        self.grads = [torch.zeros(s, dtype=self.dtype, device=device) for s in shapes]
        # the vectors: a bias for every matrix, then gamma and beta of the blocks' norms and the last one
        self.vectors = torch.zeros(sum(sizes), device=device)
        self.vector_grads = torch.zeros_like(self.vectors)
        views, grads = self.vectors.split(sizes), self.vector_grads.split(sizes)
        n = m + 2 * (blocks + 1)
        self.biases, self.bias_grads = views[:m], grads[:m]
        self.norms = list(zip(views[m:n:2], views[m + 1:n:2]))
        self.norm_grads = list(zip(grads[m:n:2], grads[m + 1:n:2]))
        ones = [gamma for gamma, _ in self.norms]
        if context is not None:
            self.biases, self.bias_grads = (t[:m] + t[n:n + 4 * blocks] for t in (views, grads))
            # of each block: gamma, beta, and the gammas of q and k
            self.attention_norms = [views[n + 4 * (blocks + k):n + 4 * (blocks + k + 1)] for k in range(blocks)]
            self.attention_norm_grads = [grads[n + 4 * (blocks + k):n + 4 * (blocks + k + 1)] for k in range(blocks)]
            ones += [v[i] for v in self.attention_norms for i in (0, 2, 3)]
            if axes:   # pairs from one turn over the extent to 64, in directions all around
                pairs = head // 2
                size = 2.0 * math.pi / extent * torch.logspace(0.0, 6.0, pairs, base=2.0)
                direction = torch.randn(pairs, axes, generator=g)
                self.frequencies = (size[:, None] * direction / direction.norm(dim=1, keepdim=True)).to(device)
        for gamma in ones:
            gamma.fill_(1.0)
        self.blocks = blocks
        self.ops = LayerOps()
        self._kept = None
        self._clip = None

    def _check_context(self, width: int, extent: float) -> int:
        if self.context < 1 or self.heads < 1 or self.kv_heads < 1 or width % self.heads or self.heads % self.kv_heads:
            raise RuntimeError("AttributeNetwork: heads must divide the width, and kv_heads the heads")
        head = width // self.heads
        if head > 128 or not 0 <= self.axes <= 4 or (self.axes and head < 2) or not extent > 0.0:
            raise RuntimeError("AttributeNetwork: heads of at most 128 columns, 0 to 4 axes and a positive extent are "
                               "supported")
        return head

    def optimizer(self):
        """Muon on the matrices, which also writes the half-precision copies."""
        from .optim import Muon
        return Muon(self.weights, self.grads, copies=self.copies)

    def clip(self, max_norm: float, scale: float = 1.0, stream=None):
        """Bounds the norm of all gradients together, those of the vectors included, in place; returns the norm on the
        device (GradientClip). scale multiplies the gradients first: 1 / the factor of a scaled loss."""
        if self._clip is None:
            from .optim import GradientClip
            self._clip = GradientClip(self.grads + [self.vector_grads])
        return self._clip.clip(max_norm, scale=scale, stream=stream)

    def matrices(self):
        """The matrices that the products read."""
        return self.weights if self.copies is None else self.copies

    def _turn(self, positions):
        if not self.axes:
            return {}
        if positions is None:
            raise RuntimeError("AttributeNetwork: positions of the rows and of the states are needed")
        return {"positions": positions, "frequencies": self.frequencies}

    def _attend(self, k, h, context, turns, mask, batch, keep, stream):
        """h + the block's attention to the states, and what its backward needs."""
        ops, w = self.ops, self.matrices()
        wq = self.last + 1 + 4 * k
        gamma, beta, gamma_q, gamma_k = self.attention_norms[k]
        n, mean, rstd = ops.layer_norm(h, gamma, beta, eps=self.eps, stream=stream)
        q = ops.linear(n, w[wq], self.biases[wq], stream=stream)
        key = ops.linear(context, w[wq + 1], self.biases[wq + 1], stream=stream)
        v = ops.linear(context, w[wq + 2], self.biases[wq + 2], stream=stream)
        qn = ops.head_norm(q, self.heads, gamma_q, out=None if keep else q, stream=stream, **turns[0])
        kn = ops.head_norm(key, self.kv_heads, gamma_k, out=None if keep else key, stream=stream, **turns[1])
        a = ops.attention(qn, kn, v, self.heads, kv_heads=self.kv_heads, batch=batch, mask=mask, keep_lse=keep,
                          stream=stream)
        a, lse = a if keep else (a, None)
        to = ops.linear(a, w[wq + 3], self.biases[wq + 3], residual=h, out=None if keep else h, stream=stream)
        return to, (h, n, mean, rstd, q, key, v, qn, kn, a, lse)

    def _attend_backward(self, k, g, kept, context, turns, mask, batch, need_context, stream):
        """The gradient of the block's input for its output's g, and that of the states by this block."""
        ops, w = self.ops, self.matrices()
        wq = self.last + 1 + 4 * k
        h, n, mean, rstd, q, key, v, qn, kn, a, lse = kept
        gamma, _, gamma_q, gamma_k = self.attention_norms[k]
        grad_gamma, grad_beta, grad_gamma_q, grad_gamma_k = self.attention_norm_grads[k]

        def linear(i, gy, x, need=True):
            return ops.linear_backward(gy, x, w[wq + i], need_x=need, grad_weight=self.grads[wq + i],
                                       grad_bias=self.bias_grads[wq + i], stream=stream)[0]

        ga = linear(3, g, a)
        gq, gk, gv = ops.attention_backward(ga, qn, kn, v, a, lse, self.heads, kv_heads=self.kv_heads, batch=batch,
                                            mask=mask, stream=stream)
        ops.head_norm_backward(gq, q, self.heads, gamma_q, grad_x=gq, grad_gamma=grad_gamma_q, stream=stream, **turns[0])
        ops.head_norm_backward(gk, key, self.kv_heads, gamma_k, grad_x=gk, grad_gamma=grad_gamma_k, stream=stream,
                               **turns[1])
        gn = linear(0, gq, n)
        parts = [linear(1, gk, context, need_context), linear(2, gv, context, need_context)]
        g, _, _ = ops.layer_norm_backward(gn, h, gamma, mean, rstd, residual_grad=g, grad_x=g, grad_gamma=grad_gamma,
                                          grad_beta=grad_beta, stream=stream)
        return g, parts

    def forward(self, features, keep: bool = True, stream=None, context=None, mask=None, batch: int = 1, positions=None,
                context_positions=None):
        """The attributes, in the network's dtype. keep: hold what backward needs (until the next forward).

        A network with context takes the states [batch x states, context] in its dtype (features are batch x rows then),
        mask [batch, states] where some do not exist, and with axes the float32 positions [rows, axes] and
        context_positions [states, axes] of both."""
        ops, w, last = self.ops, self.matrices(), self.last
        self._kept = None
        turns = None
        if (context is None) != (self.context is None):
            raise RuntimeError("AttributeNetwork::forward: states are for a network with context")
        if context is not None:
            turns = self._turn(positions), self._turn(context_positions)
        h = ops.linear(features, w[0], self.biases[0], stream=stream)
        kept = [features]
        attended = []
        for k in range(self.blocks):
            if context is not None:
                h, of = self._attend(k, h, context, turns, mask, batch, keep, stream)
                if keep:
                    attended.append(of)
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
            self._kept = kept, attended, (context, turns, mask, batch)
        return ops.linear(n, w[last], self.biases[last], stream=stream)

    def backward(self, grad_attributes, need_features: bool = False, stream=None, need_context: bool = False):
        """Fills grads and vector_grads for dL/dattributes (in the network's dtype) of the last forward; returns
        dL/dfeatures where needed, and with need_context a pair of it and dL/dcontext (float32)."""
        if self._kept is None:
            raise RuntimeError("AttributeNetwork::backward: no forward that kept its values")
        ops, w, last = self.ops, self.matrices(), self.last
        kept, attended, (context, turns, mask, batch) = self._kept
        if need_context and context is None:
            raise RuntimeError("AttributeNetwork::backward: a network without context")
        act = self.activation
        h, n, mean, rstd = kept[-1]
        g, _, _ = ops.linear_backward(grad_attributes, n, w[last], grad_weight=self.grads[last],
                                      grad_bias=self.bias_grads[last], stream=stream)
        gg, gb = self.norm_grads[-1]
        g, _, _ = ops.layer_norm_backward(g, h, self.norms[-1][0], mean, rstd, grad_x=g, grad_gamma=gg, grad_beta=gb,
                                          stream=stream)
        parts = []
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
            if context is not None:
                g, of = self._attend_backward(k, g, attended[k], context, turns, mask, batch, need_context, stream)
                parts += of
        gx, _, _ = ops.linear_backward(g, kept[0], w[0], need_x=need_features, grad_weight=self.grads[0],
                                       grad_bias=self.bias_grads[0], stream=stream)
        if not need_context:
            return gx
        return gx, self._sum(parts, context, stream)

    @staticmethod
    def _sum(parts, like, stream):
        """Of the blocks' gradients, in float32."""
        import contextlib

        import torch
        with torch.cuda.stream(stream) if stream is not None else contextlib.nullcontext():
            total = torch.zeros(like.shape, dtype=torch.float32, device=like.device)
            for t in parts:
                total += t
        return total


def encode_positions(means, octaves: int = 10, dtype=None):
    """Positions [n, 3] with the sines and cosines of their multiples by 2^0 .. 2^(octaves - 1): [n, 3 + 6 octaves],
    the usual input of a network over positions."""
    import torch
    scaled = means[:, None, :] * (2.0 ** torch.arange(octaves, device=means.device))[None, :, None]
    scaled = scaled.reshape(means.shape[0], 3 * octaves)
    out = torch.cat([means, torch.sin(scaled), torch.cos(scaled)], dim=1)
    return out if dtype is None else out.to(dtype)
