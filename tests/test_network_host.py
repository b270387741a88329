"""What the attribute network's entry points refuse: checked on the host, before anything is launched."""
import ctypes as C

import pytest
import torch

from tinygs_amd import _lib

BASE = 1 << 20   # an address that nothing reads: every call here is refused
F32, F16, BF16 = _lib.TGS_DTYPE_FLOAT32, _lib.TGS_DTYPE_FLOAT16, _lib.TGS_DTYPE_BFLOAT16


def mat(slot, rows, cols, stride=None, dtype=F32, off=0):
    return _lib.tgs_matrix(BASE * (slot + 1) + off, rows, cols, cols if stride is None else stride, dtype)


@pytest.fixture(scope="module")
def net():
    lib = _lib.load()
    h = C.c_void_p()
    assert lib.tgs_network_create(C.byref(h)) == 0
    yield h
    assert lib.tgs_network_destroy(h) == 0


def refused(rc, words):
    assert rc in (_lib.TGS_ERR_INVALID, _lib.TGS_ERR_UNSUPPORTED), rc
    assert words in _lib.load().tgs_last_error().decode()


def forward(net, **kw):
    a = dict(x=mat(0, 4, 8), w=mat(1, 6, 8), bias=None, act=0, residual=None, preact=None, y=mat(2, 4, 6))
    a.update(kw)
    return _lib.load().tgs_linear_forward(net, a["x"], a["w"], a["bias"], a["act"], a["residual"], a["preact"], a["y"],
                                          None)


def backward(net, **kw):
    a = dict(gy=mat(3, 4, 6), x=mat(0, 4, 8), w=mat(1, 6, 8), z=mat(2, 4, 6), act=3, gx=mat(4, 4, 8), gw=mat(5, 6, 8),
             gb=BASE * 9)
    a.update(kw)
    return _lib.load().tgs_linear_backward(net, a["gy"], a["x"], a["w"], a["z"], a["act"], a["gx"], a["gw"], a["gb"],
                                           None)


def norm(net, **kw):
    a = dict(x=mat(0, 4, 8), gamma=None, beta=None, eps=1e-5, y=mat(2, 4, 8), mean=None, rstd=None)
    a.update(kw)
    return _lib.load().tgs_layer_norm_forward(net, a["x"], a["gamma"], a["beta"], a["eps"], a["y"], a["mean"],
                                              a["rstd"], None)


def norm_backward(net, **kw):
    a = dict(gy=mat(3, 4, 8), x=mat(0, 4, 8), gamma=None, mean=BASE * 8, rstd=BASE * 9, res=None, gx=mat(4, 4, 8),
             gg=BASE * 10, gb=BASE * 11)
    a.update(kw)
    return _lib.load().tgs_layer_norm_backward(net, a["gy"], a["x"], a["gamma"], a["mean"], a["rstd"], a["res"],
                                               a["gx"], a["gg"], a["gb"], None)


def test_linear_refusals(net):
    refused(forward(None), "network is NULL")
    refused(forward(net, x=None), "x is NULL")
    refused(forward(net, x=mat(0, 4, 8, dtype=2)), "dtype 2")
    refused(forward(net, x=mat(0, -1, 8)), "rows")
    refused(forward(net, x=mat(0, 1 << 31, 8)), "rows")
    refused(forward(net, x=mat(0, 4, 0)), "columns")
    refused(forward(net, x=mat(0, 4, 8, 7)), "stride")
    refused(forward(net, x=mat(0, 4, 8, 1 << 21)), "stride")
    refused(forward(net, x=_lib.tgs_matrix(None, 4, 8, 8, F32)), "data is NULL")
    refused(forward(net, x=mat(0, 4, 8, off=2)), "aligned")
    refused(forward(net, x=mat(0, 4, 8, dtype=F16, off=1), w=mat(1, 6, 8, dtype=F16), y=mat(2, 4, 6, dtype=F16)),
            "aligned")
    refused(forward(net, w=mat(1, 6, 9)), "w is 6 x 9")
    refused(forward(net, w=mat(1, 0, 8)), "no rows")
    refused(forward(net, w=mat(1, 6, 8, dtype=BF16)), "w: dtype 3")
    refused(forward(net, y=mat(2, 4, 5)), "y is 4 x 5")
    refused(forward(net, y=None), "y is NULL")
    refused(forward(net, residual=mat(3, 3, 6)), "residual is 3 x 6")
    refused(forward(net, preact=mat(3, 4, 6, dtype=F16)), "preact: dtype")
    refused(forward(net, act=4), "activation 4")
    refused(forward(net, act=-1), "activation -1")
    refused(forward(net, bias=BASE * 7 + 2), "bias")


def test_linear_overlaps(net):
    refused(forward(net, y=mat(0, 4, 6)), "y overlaps x")
    refused(forward(net, y=mat(1, 4, 6, off=100)), "y overlaps w")
    refused(forward(net, preact=mat(2, 4, 6)), "preact overlaps y")
    refused(forward(net, residual=mat(2, 4, 6, off=4)), "y overlaps residual")
    refused(forward(net, residual=mat(3, 4, 6), preact=mat(3, 4, 6)), "preact overlaps residual")
    refused(forward(net, bias=BASE * 3 + 8), "y overlaps bias")
    # columns of one buffer side by side share nothing: refused for their shapes only
    refused(forward(net, x=mat(0, 4, 8, 16), y=mat(0, 4, 7, 16, off=32)), "y is 4 x 7")
    refused(forward(net, x=mat(0, 4, 8, 16), y=mat(0, 4, 6, 16, off=28)), "y overlaps x")
    refused(forward(net, x=mat(0, 4, 8, 13, off=40), y=mat(0, 4, 6, 13)), "y overlaps x")


def test_linear_backward_refusals(net):
    refused(backward(None), "network is NULL")
    refused(backward(net, gy=mat(3, 4, 7)), "grad_y is 4 x 7")
    refused(backward(net, z=None), "preact is NULL")
    refused(backward(net, z=mat(2, 5, 6)), "preact is 5 x 6")
    refused(backward(net, gx=mat(4, 4, 9)), "grad_x is 4 x 9")
    refused(backward(net, gw=mat(5, 6, 8, dtype=F16)), "grad_w: dtype")
    refused(backward(net, gb=BASE * 9 + 1), "grad_bias")
    refused(backward(net, act=9), "activation 9")
    refused(backward(net, gx=mat(3, 4, 8)), "grad_x overlaps grad_y")
    refused(backward(net, gx=mat(0, 4, 8)), "grad_x overlaps x")
    refused(backward(net, gw=mat(1, 6, 8)), "grad_w overlaps w")
    refused(backward(net, gw=mat(2, 6, 8)), "grad_w overlaps preact")
    refused(backward(net, gw=mat(4, 6, 8)), "grad_w overlaps grad_x")
    refused(backward(net, gb=BASE * 6), "grad_bias overlaps grad_w")


def test_layer_norm_refusals(net):
    refused(norm(None), "network is NULL")
    refused(norm(net, y=mat(2, 4, 9)), "y is 4 x 9")
    refused(norm(net, eps=-1.0), "epsilon")
    refused(norm(net, eps=float("nan")), "epsilon")
    refused(norm(net, gamma=BASE * 5 + 1), "gamma")
    refused(norm(net, y=mat(0, 4, 8, off=4)), "y overlaps x")
    refused(norm(net, mean=BASE), "mean overlaps x")
    refused(norm(net, mean=BASE * 7, rstd=BASE * 7 + 8), "mean overlaps rstd")
    refused(norm(net, rstd=BASE * 7, gamma=BASE * 7), "rstd overlaps gamma")
    refused(norm_backward(None), "network is NULL")
    refused(norm_backward(net, mean=None), "mean or rstd")
    refused(norm_backward(net, gx=None, res=mat(6, 4, 8)), "residual_grad without grad_x")
    refused(norm_backward(net, res=mat(6, 4, 7)), "residual_grad is 4 x 7")
    refused(norm_backward(net, gx=mat(0, 4, 8)), "grad_x overlaps x")
    refused(norm_backward(net, gx=mat(3, 4, 8, off=4)), "grad_x overlaps grad_y")
    refused(norm_backward(net, gg=BASE * 11), "grad_gamma overlaps grad_beta")
    refused(norm_backward(net, gg=BASE * 8), "grad_gamma overlaps mean")


def muon(weights, grads, momenta, copies=None, count=None):
    def arr(v):
        return None if v is None else (_lib.tgs_matrix * len(v))(*v)
    h = C.c_void_p()
    rc = _lib.load().tgs_muon_create(arr(weights), arr(grads), arr(momenta), arr(copies),
                                     len(weights) if count is None else count, C.byref(h))
    return rc, h


def test_muon_refusals():
    lib = _lib.load()
    w, g, m = [mat(0, 4, 8), mat(1, 3, 3)], [mat(2, 4, 8), mat(3, 3, 3)], [mat(4, 4, 8), mat(5, 3, 3)]
    refused(lib.tgs_muon_create(None, None, None, None, 1, C.byref(C.c_void_p())), "NULL")
    refused(muon(w, g, m, count=0)[0], "0 matrices")
    refused(muon([mat(0, 4, 8, dtype=F16)], g, m, count=1)[0], "weights[0]: dtype 1, not float32")
    refused(muon([mat(0, 0, 8)], g, m, count=1)[0], "0 rows")
    refused(muon(w, [g[0], mat(3, 3, 4)], m)[0], "grads[1] is 3 x 4")
    refused(muon(w, [g[0], mat(3, 3, 3, dtype=F16)], m)[0], "grads[1]: dtype")
    refused(muon(w, g, [m[0], mat(5, 3, 3, dtype=F16)])[0], "momenta[1]: dtype")
    refused(muon(w, g, m, [mat(6, 4, 8, dtype=F16), mat(7, 3, 3, dtype=BF16)])[0], "copies[1]: dtype")
    refused(muon([w[0], mat(0, 3, 3, off=16)], g, m)[0], "weights[0] overlaps weights[1]")
    refused(muon(w, g, [m[0], mat(3, 3, 3)])[0], "momenta[1] overlaps grads[1]")
    refused(muon(w, g, m, [mat(0, 4, 8), mat(7, 3, 3)])[0], "weights[0] overlaps copies[0]")
    rc, h = muon(w, g, m)
    assert rc == 0
    p = _lib.tgs_muon_params()
    assert lib.tgs_muon_get_params(h, C.byref(p)) == 0 and p.iterations == 5 and p.nesterov == 1
    for field, bad in (("iterations", 33), ("iterations", -1), ("momentum", 1.0), ("epsilon", 0.0),
                       ("lr", float("inf"))):
        q = _lib.tgs_muon_params.from_buffer_copy(p)
        setattr(q, field, bad)
        assert lib.tgs_muon_set_params(h, C.byref(q)) == _lib.TGS_ERR_INVALID
    arr = (_lib.tgs_matrix * 2)
    refused(lib.tgs_muon_set_matrices(h, arr(*w), arr(*g), arr(*m), None, 1), "1 matrices, not 2")
    half = arr(mat(2, 4, 8, dtype=F16), mat(3, 3, 3, dtype=F16))
    refused(lib.tgs_muon_set_matrices(h, arr(*w), half, arr(*m), None, 2), "dtype is not that of the creation")
    other = [mat(0, 8, 4), w[1]], [mat(2, 8, 4), g[1]], [mat(4, 8, 4), m[1]]
    refused(lib.tgs_muon_set_matrices(h, arr(*other[0]), arr(*other[1]), arr(*other[2]), None, 2), "shape at creation")
    assert lib.tgs_muon_set_lr(None, 1.0) == _lib.TGS_ERR_INVALID and lib.tgs_muon_step(None, 1.0, None) == 1
    assert lib.tgs_muon_destroy(h) == 0


def test_python_refusals():
    from tinygs_amd import network, optim
    with pytest.raises(RuntimeError, match="two dimensions"):
        network.matrix(torch.zeros(3), "x")
    with pytest.raises(RuntimeError, match="next to each other"):
        network.matrix(torch.zeros(3, 4).t(), "x")
    with pytest.raises(RuntimeError, match="float32, float16 and bfloat16"):
        network.matrix(torch.zeros(3, 4, dtype=torch.float64), "x")
    with pytest.raises(RuntimeError, match="not on the device"):
        network.matrix(torch.zeros(3, 4), "x")
    ops = network.LayerOps()
    x, w = torch.zeros(3, 4), torch.zeros(5, 4)
    with pytest.raises(RuntimeError, match="unknown activation"):
        ops.linear(x, w, activation="tanh", out=x)
    with pytest.raises(RuntimeError, match="needs preact"):
        ops.linear_backward(x, x, w, activation="relu")
    with pytest.raises(RuntimeError, match="packed float32 vector"):
        network._vector(torch.zeros(4), 5, "bias")
    with pytest.raises(RuntimeError, match="same count"):
        optim.Muon([x], [x, x])
