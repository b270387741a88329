"""SimpleAdam, Muon for an attribute network's matrices, and the clipping of gradients, over the C ABI.

Mirrors tinygs's OptimizerBase / SimpleAdam / create_optimizer
(tinygs/include/tinygs/optim/optim.hpp:39-106,
tinygs/include/tinygs/optim/simple_adam.hpp:30-87, tinygs/src/optim/optim.cu:86-105).
"""
from __future__ import annotations

import contextlib
import ctypes as C

from . import _lib
from .core import GPUGaussian3d, stream_ptr

GROUPS = ("means", "opacities", "rotations", "scales", "sh0", "sh_rest")


class OptimizerBase:
    def __init__(self, gaussians: GPUGaussian3d, gaussians_grad: GPUGaussian3d):
        self.m_gaussians = gaussians
        self.m_gaussians_grad = gaussians_grad

    def get_gaussians(self):
        return self.m_gaussians

    def get_gaussians_grad(self):
        return self.m_gaussians_grad


class SimpleAdam(OptimizerBase):
    def __init__(self, gaussians: GPUGaussian3d, gaussians_grad: GPUGaussian3d):
        super().__init__(gaussians, gaussians_grad)
        if gaussians.size() != gaussians_grad.size():
            raise RuntimeError("SimpleAdam::step: gaussians and gaussians_grad must have same size")
        self._cp = gaussians.to_c()
        self._cg = gaussians_grad.to_c()
        h = C.c_void_p()
        _lib.check(_lib.load().tgs_adam_create(C.byref(self._cp), C.byref(self._cg), C.byref(h)), "create_optimizer")
        self._h = h

    def __del__(self):
        h = getattr(self, "_h", None)
        if h is not None and h.value:
            try:
                _lib.load().tgs_adam_destroy(h)
            except Exception:
                pass
            self._h = None

    def _rebind(self):
        self._cp = self.m_gaussians.to_c()
        self._cg = self.m_gaussians_grad.to_c()
        _lib.check(_lib.load().tgs_adam_set_gaussians(self._h, C.byref(self._cp), C.byref(self._cg)), "set_gaussians")

    def step(self, scale: float, stream=None, row_mask: int | None = None, device_step: bool = False,
             rows: str | None = None, same_step: bool = False):
        """OptimizerBase::step. row_mask: device address of a per-Gaussian
        byte mask (a sparse backward's); unmarked gradient rows are taken as
        zero without being read. device_step=True keeps the step count and
        bias corrections on the device (TGS_ADAM_DEVICE_STEP), so the step
        can be captured into a graph and replayed. rows="unmarked" / "marked"
        updates only the rows whose mask byte is 0 / nonzero
        (TGS_ADAM_ROWS_UNMARKED / _MARKED), same_step=True repeats the last
        call's step count (TGS_ADAM_SAME_STEP): one step in two parts."""
        self._rebind()
        L = _lib.load()
        flags = _lib.TGS_ADAM_DEVICE_STEP if device_step else 0
        if rows is not None:
            flags |= {"unmarked": _lib.TGS_ADAM_ROWS_UNMARKED, "marked": _lib.TGS_ADAM_ROWS_MARKED}[rows]
        if same_step:
            flags |= _lib.TGS_ADAM_SAME_STEP
        if flags:
            _lib.check(L.tgs_adam_step_ex(self._h, float(scale), C.c_void_p(row_mask) if row_mask else None,
                                          flags, stream_ptr(stream)), "SimpleAdam::step")
        elif row_mask is None:
            _lib.check(L.tgs_adam_step(self._h, float(scale), stream_ptr(stream)), "SimpleAdam::step")
        else:
            _lib.check(L.tgs_adam_step_masked(self._h, float(scale), C.c_void_p(row_mask), stream_ptr(stream)),
                       "SimpleAdam::step")

    def device_steps(self, stream=None) -> int:
        """The step count of the device-step mode (waits for the stream)."""
        v = C.c_int64()
        _lib.check(_lib.load().tgs_adam_device_steps(self._h, C.byref(v), stream_ptr(stream)), "device_steps")
        return v.value

    def reset(self, stream=None):
        _lib.check(_lib.load().tgs_adam_reset(self._h, stream_ptr(stream)), "SimpleAdam::reset")

    def remove(self, kept_flag, num_kept: int, stream=None):
        """SimpleAdam::remove (simple_adam.cu:841-906). The reference builds
        its row mapping from the optimiser's Gaussians, which StrategyBase has
        already shrunk to num_kept rows: the kept rows among the first
        num_kept flags, in order, then row 0 for the remaining moment rows.
        That mapping is reproduced here."""
        torch = __import__("torch")
        rows = torch.zeros(max(num_kept, 1), dtype=torch.int32, device=kept_flag.device)
        cnt = C.c_int64()
        L = _lib.load()
        _lib.check(L.tgs_flags_compact(C.c_void_p(kept_flag.data_ptr()), int(num_kept), C.c_void_p(rows.data_ptr()),
                                       C.byref(cnt), stream_ptr(stream)), "SimpleAdam::remove")
        _lib.check(L.tgs_adam_gather(self._h, C.c_void_p(rows.data_ptr()), int(num_kept), stream_ptr(stream)),
                   "SimpleAdam::remove")

    def duplicate(self, num_duplicate: int, stream=None):
        """SimpleAdam::duplicate (simple_adam.cu:908-924): zero moment rows
        for the appended Gaussians."""
        if num_duplicate <= 0:
            return
        _lib.check(_lib.load().tgs_adam_append(self._h, int(num_duplicate), stream_ptr(stream)),
                   "SimpleAdam::duplicate")

    def reset_indices(self, indices, num_reset: int | None = None, stream=None):
        """SimpleAdam::reset(int* indices, int num_reset) (simple_adam.cu:
        944-979): zero both moments of the given rows (device int32 tensor)."""
        n = int(indices.numel() if num_reset is None else num_reset)
        _lib.check(_lib.load().tgs_adam_reset_rows(self._h, C.c_void_p(indices.data_ptr()), n, stream_ptr(stream)),
                   "SimpleAdam::reset")

    def reorder(self, indices, stream=None):
        """SimpleAdam::reorder(uint* indices) (simple_adam.cu:1037-1097):
        new row i = old row indices[i] (device int32/uint32 tensor, one per row)."""
        _lib.check(_lib.load().tgs_adam_reorder(self._h, C.c_void_p(indices.data_ptr()), stream_ptr(stream)),
                   "SimpleAdam::reorder")

    def reset_opacity(self, stream=None):
        """SimpleAdam::reset_opacity (simple_adam.cu:981-985)."""
        _lib.check(_lib.load().tgs_adam_reset_opacity(self._h, stream_ptr(stream)), "SimpleAdam::reset_opacity")

    def set_lr(self, lr: float):
        _lib.check(_lib.load().tgs_adam_set_lr(self._h, float(lr)), "set_lr")

    def get_lr(self) -> float:
        return float(_lib.load().tgs_adam_get_lr(self._h))

    def global_steps(self) -> int:
        return int(_lib.load().tgs_adam_global_steps(self._h))

    def get_params(self) -> dict:
        p = _lib.tgs_adam_params()
        _lib.check(_lib.load().tgs_adam_get_params(self._h, C.byref(p)), "get_params")
        return {f: getattr(p, f) for f, _ in p._fields_}

    def set_params(self, config: dict):
        p = _lib.tgs_adam_params()
        _lib.check(_lib.load().tgs_adam_get_params(self._h, C.byref(p)), "get_params")
        alias = {"eps": "epsilon"}
        for k, v in config.items():
            k = alias.get(k, k)
            if k == "decay_reduction":
                p.decay_mean = 1 if v == "mean" else 0
            elif hasattr(p, k):
                setattr(p, k, v)
            else:
                raise RuntimeError(f"SimpleAdam: unknown parameter {k}")
        _lib.check(_lib.load().tgs_adam_set_params(self._h, C.byref(p)), "set_params")

    def moments(self, group: str):
        import torch
        k = GROUPS.index(group)
        a, b = C.c_void_p(), C.c_void_p()
        _lib.check(_lib.load().tgs_adam_moments(self._h, k, C.byref(a), C.byref(b)), "moments")
        mult = (3, 1, 4, 3, 3, 45)[k]
        n = mult * self.m_gaussians.size()
        dev = self.m_gaussians.means().device
        m1 = torch.empty(n, dtype=torch.float32, device=dev)
        m2 = torch.empty(n, dtype=torch.float32, device=dev)
        _lib.copy_device(a.value, 4 * n, m1)
        _lib.copy_device(b.value, 4 * n, m2)
        return m1, m2


class Muon:
    """Muon on a network's matrices: momentum, the update orthogonalised by Newton-Schulz products, decoupled weight
    decay. weights and momenta (zeros when not given) are float32 and updated in place; grads are of one dtype;
    copies, when given, receive the updated weights rounded to their dtype (the network's half-precision matrices).
    The tensors are kept: a step reads what they hold then. Steps run on one stream, or the caller orders them."""

    def __init__(self, weights, grads, momenta=None, copies=None):
        self._lib = _lib.load()
        self._h = None
        count = len(weights)
        if momenta is None:
            torch = __import__("torch")
            momenta = [torch.zeros(w.shape, dtype=torch.float32, device=w.device) for w in weights]
        if len(grads) != count or len(momenta) != count or (copies is not None and len(copies) != count):
            raise RuntimeError("Muon: weights, grads, momenta and copies must have the same count")
        self.m_weights, self.m_grads, self.m_momenta = list(weights), list(grads), list(momenta)
        self.m_copies = None if copies is None else list(copies)
        h = C.c_void_p()
        _lib.check(self._lib.tgs_muon_create(*self._arrays(), count, C.byref(h)), "create_optimizer")
        self._h = h

    def _arrays(self):
        from .network import matrix

        def array(tensors, name):
            if tensors is None:
                return None
            return (_lib.tgs_matrix * len(tensors))(*[matrix(t, f"{name}[{i}]") for i, t in enumerate(tensors)])

        return (array(self.m_weights, "weights"), array(self.m_grads, "grads"), array(self.m_momenta, "momenta"),
                array(self.m_copies, "copies"))

    def __del__(self):
        h = getattr(self, "_h", None)
        if h is not None and h.value:
            try:
                self._lib.tgs_muon_destroy(h)
            except Exception:
                pass
            self._h = None

    def get_weights(self):
        return self.m_weights

    def get_grads(self):
        return self.m_grads

    def momenta(self):
        return self.m_momenta

    def set_grads(self, grads):
        """Other gradient tensors of the same shapes and dtype."""
        if len(grads) != len(self.m_weights):
            raise RuntimeError("Muon: weights and grads must have the same count")
        kept, self.m_grads = self.m_grads, list(grads)
        try:
            _lib.check(self._lib.tgs_muon_set_matrices(self._h, *self._arrays(), len(grads)), "Muon::set_grads")
        except Exception:
            self.m_grads = kept
            raise

    def step(self, scale: float, stream=None):
        """One step on gradients multiplied by scale."""
        _lib.check(self._lib.tgs_muon_step(self._h, float(scale), stream_ptr(stream)), "Muon::step")

    def reset(self, stream=None):
        _lib.check(self._lib.tgs_muon_reset(self._h, stream_ptr(stream)), "Muon::reset")

    def set_lr(self, lr: float):
        _lib.check(self._lib.tgs_muon_set_lr(self._h, float(lr)), "set_lr")

    def get_lr(self) -> float:
        return float(self._lib.tgs_muon_get_lr(self._h))

    def get_params(self) -> dict:
        p = _lib.tgs_muon_params()
        _lib.check(self._lib.tgs_muon_get_params(self._h, C.byref(p)), "get_params")
        return {f: getattr(p, f) for f, _ in p._fields_}

    def set_params(self, config: dict):
        p = _lib.tgs_muon_params()
        _lib.check(self._lib.tgs_muon_get_params(self._h, C.byref(p)), "get_params")
        alias = {"eps": "epsilon"}
        for k, v in config.items():
            k = alias.get(k, k)
            if not hasattr(p, k):
                raise RuntimeError(f"Muon: unknown parameter {k}")
            setattr(p, k, int(v) if k in ("nesterov", "iterations") else float(v))
        _lib.check(self._lib.tgs_muon_set_params(self._h, C.byref(p)), "set_params")


class GradientClip:
    """The norm of many gradients together, and clipping: norm = scale sqrt(sum of squares),
    g <- g scale min(1, max_norm / (norm + epsilon)). grads are tensors of any shapes and of float32, float16 or
    bfloat16 each, packed or 2-D with rows further apart; with clipped (tensors of the same shapes) these receive the
    result in their own dtypes and grads stay as they are. The tensors are kept: a run reads what they hold then. Runs
    are on one stream, or the caller orders them. The first run, and the first after set_grads, place a table on the
    device and wait for it: capture only later ones, and do not call set_grads while the graph is in use."""

    def __init__(self, grads, clipped=None):
        self._lib = _lib.load()
        self._h = None
        self._norm = None
        self._bind(grads, clipped)
        h = C.c_void_p()
        _lib.check(self._lib.tgs_gradient_clip_create(*self._arrays(), C.byref(h)), "GradientClip")
        self._h = h

    def _bind(self, grads, clipped):
        self.m_grads = list(grads)
        self.m_clipped = None if clipped is None else list(clipped)
        if not self.m_grads or (clipped is not None and len(self.m_clipped) != len(self.m_grads)):
            raise RuntimeError("GradientClip: grads, and as many clipped tensors, are needed")
        for name, tensors in (("grads", self.m_grads), ("clipped", self.m_clipped or ())):
            for i, t in enumerate(tensors):
                if t.get_device() != self.m_grads[0].get_device():
                    raise RuntimeError(f"GradientClip: {name}[{i}] is on another device")
                if name == "clipped" and t.shape != self.m_grads[i].shape:
                    raise RuntimeError(f"GradientClip: clipped[{i}] is not of its gradient's shape")

    def _arrays(self):
        from .network import matrix
        outs = self.m_clipped or [None] * len(self.m_grads)
        views, out_views = [], []
        for i, (g, c) in enumerate(zip(self.m_grads, outs)):
            # a packed tensor is a column of its elements, whatever its shape
            if g.is_contiguous() and (c is None or c.is_contiguous()):
                g, c = g.reshape(-1, 1), None if c is None else c.reshape(-1, 1)
            views.append(matrix(g, f"grads[{i}]"))
            if c is not None:
                out_views.append(matrix(c, f"clipped[{i}]"))
        n = len(views)
        return ((_lib.tgs_matrix * n)(*views), (_lib.tgs_matrix * n)(*out_views) if out_views else None, n)

    def __del__(self):
        h = getattr(self, "_h", None)
        if h is not None and h.value:
            try:
                self._lib.tgs_gradient_clip_destroy(h)
            except Exception:
                pass
            self._h = None

    def set_grads(self, grads, clipped=None):
        """Other tensors, of any number and shapes."""
        kept = self.m_grads, self.m_clipped
        try:
            self._bind(grads, clipped)
            if self.m_grads[0].get_device() != kept[0][0].get_device():
                raise RuntimeError("GradientClip::set_grads: on another device")
            _lib.check(self._lib.tgs_gradient_clip_set_matrices(self._h, *self._arrays()), "GradientClip::set_grads")
        except Exception:
            self.m_grads, self.m_clipped = kept
            raise

    def clip(self, max_norm: float, scale: float = 1.0, epsilon: float = 1e-6, stream=None):
        """One run. Returns the norm (scale included, before clipping), a float32 scalar on the device that the next
        run overwrites. max_norm infinite: the norm alone, and scale where it is not 1."""
        from .network import _current_device
        device = self.m_grads[0].get_device()
        if device != _current_device():
            raise RuntimeError("GradientClip: the gradients are not on the current device")
        if self._norm is None:
            import torch
            with torch.cuda.stream(stream) if stream is not None else contextlib.nullcontext():
                self._norm = torch.empty((), dtype=torch.float32, device=self.m_grads[0].device)
            # the stream's address without the Stream object around it: 0.1 us a call against 2.8
            self._current = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
                lambda index: torch.cuda.current_stream(index).cuda_stream)
        rc = self._lib.tgs_gradient_clip_run(self._h, max_norm, scale, epsilon, self._norm.data_ptr(),
                                             self._current(device) if stream is None else stream.cuda_stream)
        if rc:
            _lib.check(rc, "GradientClip::clip")
        return self._norm


def create_optimizer(optimizer_type: str, gaussians, gaussians_grad, copies=None):
    """"simple_adam" on Gaussians and their gradients, or "muon" on lists of matrices and of theirs; copies, for "muon",
    receive the updated matrices rounded to their dtype, which is what a half-precision network reads."""
    t = optimizer_type.lower()
    if t == "simple_adam":
        if copies is not None:
            raise RuntimeError("create_optimizer: simple_adam writes no copies")
        return SimpleAdam(gaussians, gaussians_grad)
    if t == "muon":
        return Muon(gaussians, gaussians_grad, copies=copies)
    raise RuntimeError(f"Unknown optimizer type: {optimizer_type}")
