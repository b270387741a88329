"""What the entry points of attention, head norms and clipping refuse: checked on the host, before anything is launched."""
import ctypes as C
import math

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


def shape(batch=2, heads=4, kv_heads=2, scale=0.5, mask=None, mask_stride=0):
    return _lib.tgs_attention(batch, heads, kv_heads, scale, mask, mask_stride)


def forward(net, **kw):
    a = dict(q=mat(0, 6, 32), k=mat(1, 10, 16), v=mat(2, 10, 16), a=shape(), out=mat(3, 6, 32), lse=BASE * 9, steps=(4, 1))
    a.update(kw)
    return _lib.load().tgs_attention_forward(net, a["q"], a["k"], a["v"], a["a"], a["out"], a["lse"],
                                             *a["steps"], None)


def backward(net, **kw):
    a = dict(go=mat(4, 6, 32), q=mat(0, 6, 32), k=mat(1, 10, 16), v=mat(2, 10, 16), out=mat(3, 6, 32), lse=BASE * 9,
             steps=(1, 6), a=shape(), gq=mat(5, 6, 32), gk=mat(6, 10, 16), gv=mat(7, 10, 16))
    a.update(kw)
    return _lib.load().tgs_attention_backward(net, a["go"], a["q"], a["k"], a["v"], a["out"], a["lse"], *a["steps"],
                                              a["a"], a["gq"], a["gk"], a["gv"], None)


def turn(rows=4, axes=3, pairs=4, d1=F32, d2=F32, faxes=None, off=0):
    return _lib.tgs_turn(mat(6, rows, axes, dtype=d1, off=off), mat(7, pairs, axes if faxes is None else faxes, dtype=d2))


def norm(net, **kw):
    a = dict(x=mat(0, 4, 16), heads=2, gamma=BASE * 11, turn=turn(), eps=1e-6, y=mat(2, 4, 16))
    a.update(kw)
    return _lib.load().tgs_head_norm_forward(net, a["x"], a["heads"], a["gamma"], a["turn"], a["eps"], a["y"], None)


def norm_backward(net, **kw):
    a = dict(gy=mat(3, 4, 16), x=mat(0, 4, 16), heads=2, gamma=BASE * 11, turn=turn(), eps=1e-6, gx=mat(4, 4, 16),
             gg=BASE * 12)
    a.update(kw)
    return _lib.load().tgs_head_norm_backward(net, a["gy"], a["x"], a["heads"], a["gamma"], a["turn"], a["eps"], a["gx"],
                                              a["gg"], None)


def test_attention_shapes(net):
    refused(forward(None), "network is NULL")
    refused(forward(net, q=None), "q is NULL")
    refused(forward(net, k=None), "k is NULL")
    refused(forward(net, v=None), "v is NULL")
    refused(forward(net, out=None), "out is NULL")
    refused(forward(net, a=None), "attention is NULL")
    refused(forward(net, a=shape(heads=0)), "0 heads")
    refused(forward(net, a=shape(heads=5, kv_heads=1)), "5 heads")
    refused(forward(net, a=shape(heads=4097, kv_heads=1)), "4097 heads")
    refused(forward(net, a=shape(kv_heads=3)), "do not share")
    refused(forward(net, a=shape(kv_heads=0)), "do not share")
    refused(forward(net, a=shape(heads=-4, kv_heads=-2)), "heads")
    refused(forward(net, a=shape(batch=0)), "batch of 0")
    refused(forward(net, a=shape(batch=4)), "batch of 4")
    refused(forward(net, a=shape(batch=3)), "batch of 3")
    refused(forward(net, a=shape(scale=-1.0)), "scale")
    refused(forward(net, a=shape(scale=math.nan)), "scale")
    refused(forward(net, a=shape(scale=math.inf)), "scale")
    refused(forward(net, a=shape(mask=BASE * 20, mask_stride=-1)), "mask's stride")
    refused(forward(net, q=mat(0, 6, 516), out=mat(3, 6, 516)), "heads of 129")
    refused(forward(net, k=mat(1, 10, 24)), "k is 10 x 24")
    refused(forward(net, v=mat(2, 8, 16)), "v is 8 x 16")
    refused(forward(net, v=mat(2, 10, 16, dtype=F16)), "v: dtype")
    refused(forward(net, k=mat(1, 10, 16, dtype=BF16)), "k: dtype")
    refused(forward(net, q=mat(0, 6, 32, dtype=2)), "dtype 2")
    refused(forward(net, out=mat(3, 5, 32)), "out is 5 x 32")
    refused(forward(net, lse=BASE * 9 + 2), "lse")
    refused(forward(net, q=mat(0, 6, 32, 31)), "stride")
    for steps in ((0, 1), (1, 0), (-1, 6), (3, 1), (1, 5), (2, 3)):
        refused(forward(net, steps=steps), "lse's steps")


def test_attention_overlaps(net):
    refused(forward(net, out=mat(0, 6, 32)), "out overlaps q")
    refused(forward(net, out=mat(1, 6, 32, off=64)), "out overlaps k")
    refused(forward(net, out=mat(2, 6, 32, off=64)), "out overlaps v")
    refused(forward(net, lse=BASE * 4 + 8), "lse overlaps out")
    refused(forward(net, lse=BASE + 8), "lse overlaps q")
    refused(forward(net, a=shape(mask=BASE * 4 + 3, mask_stride=5)), "out overlaps the mask")
    refused(forward(net, a=shape(mask=BASE * 9 - 9, mask_stride=5)), "lse overlaps the mask")
    refused(backward(net, gq=mat(4, 6, 32)), "grad_q overlaps grad_out")
    refused(backward(net, gq=mat(0, 6, 32)), "grad_q overlaps q")
    refused(backward(net, gk=mat(1, 10, 16)), "grad_k overlaps k")
    refused(backward(net, gv=mat(6, 10, 16)), "grad_v overlaps grad_k")
    refused(backward(net, gv=mat(5, 10, 16, off=4)), "grad_v overlaps grad_q")
    refused(backward(net, gk=mat(3, 10, 16)), "grad_k overlaps out")
    refused(backward(net, gq=mat(8, 6, 32)), "grad_q overlaps lse")
    refused(backward(net, a=shape(mask=BASE * 8, mask_stride=5)), "grad_v overlaps the mask")


def test_attention_backward_shapes(net):
    refused(backward(None), "network is NULL")
    refused(backward(net, go=mat(4, 6, 31)), "grad_out is 6 x 31")
    refused(backward(net, go=None), "grad_out is NULL")
    refused(backward(net, out=mat(3, 7, 32)), "out is 7 x 32")
    refused(backward(net, lse=None), "lse is NULL")
    refused(backward(net, gq=mat(5, 5, 32)), "grad_q is 5 x 32")
    refused(backward(net, gk=mat(6, 10, 32)), "grad_k is 10 x 32")
    refused(backward(net, gv=mat(7, 10, 16, dtype=F16)), "grad_v: dtype")


def test_head_norm(net):
    refused(norm(None), "network is NULL")
    refused(norm(net, heads=0), "0 heads")
    refused(norm(net, heads=3), "3 heads")
    refused(norm(net, x=mat(0, 4, 514), y=mat(2, 4, 514)), "heads of 257")
    refused(norm(net, eps=-1.0), "epsilon")
    refused(norm(net, eps=math.nan), "epsilon")
    refused(norm(net, gamma=BASE * 11 + 1), "gamma")
    refused(norm(net, turn=turn(rows=3)), "positions is 3 x 3")
    refused(norm(net, turn=turn(axes=5)), "5 axes")
    refused(norm(net, turn=turn(faxes=2)), "frequencies is 4 x 2")
    refused(norm(net, turn=turn(pairs=5)), "5 pairs")
    refused(norm(net, turn=turn(pairs=0)), "0 pairs")
    refused(norm(net, turn=turn(d1=F16)), "positions: dtype")
    refused(norm(net, turn=turn(d2=F16)), "frequencies: dtype")
    refused(norm(net, y=mat(2, 4, 15)), "y is 4 x 15")
    refused(norm(net, y=mat(0, 4, 16, off=4)), "y overlaps x")
    refused(norm(net, y=mat(6, 4, 16)), "y overlaps positions")
    refused(norm(net, y=mat(7, 4, 16)), "y overlaps frequencies")
    refused(norm(net, y=mat(10, 4, 16)), "y overlaps gamma")
    refused(norm_backward(net, gy=mat(3, 4, 17)), "grad_y is 4 x 17")
    refused(norm_backward(net, gx=mat(0, 4, 16)), "grad_x overlaps x")
    refused(norm_backward(net, gx=mat(3, 4, 16, off=4)), "grad_x overlaps grad_y")
    refused(norm_backward(net, gg=BASE * 4), "grad_gamma overlaps grad_y")
    refused(norm_backward(net, gg=BASE * 5), "grad_gamma overlaps grad_x")
    refused(norm_backward(net, gg=BASE * 11), "grad_gamma overlaps gamma")
    refused(norm_backward(net, gg=BASE * 7), "grad_gamma overlaps positions")
    refused(norm_backward(net, gg=BASE * 12 + 2), "grad_gamma")


def clip(grads, clipped=None, count=None):
    h = C.c_void_p()
    n = len(grads) if count is None else count
    rc = _lib.load().tgs_gradient_clip_create((_lib.tgs_matrix * len(grads))(*grads),
                                              None if clipped is None else (_lib.tgs_matrix * len(clipped))(*clipped), n,
                                              C.byref(h))
    return rc, h


def test_clip():
    lib = _lib.load()
    a, b = mat(0, 4, 8), mat(1, 16, 1, dtype=F16)
    refused(lib.tgs_gradient_clip_create(None, None, 1, C.byref(C.c_void_p())), "grads is NULL")
    refused(lib.tgs_gradient_clip_create((_lib.tgs_matrix * 1)(a), None, 1, None), "out is NULL")
    refused(clip([a], count=0)[0], "0 matrices")
    refused(clip([a], count=4097)[0], "4097 matrices")
    refused(clip([a, mat(1, 4, 8, dtype=2)])[0], "grads[1]: dtype 2")
    refused(clip([a, b, a])[0], "grads[2] overlaps grads[0]")
    refused(clip([a, b], [mat(2, 4, 8), mat(3, 16, 2)])[0], "clipped[1] is 16 x 2")
    refused(clip([a, b], [mat(2, 4, 8), mat(2, 16, 1, off=8)])[0], "clipped[1] overlaps clipped[0]")
    refused(clip([a, b], [mat(2, 4, 8), mat(0, 16, 1)])[0], "clipped[1] overlaps grads[0]")
    refused(clip([a, b], [a, mat(3, 16, 1)])[0], "clipped[0] overlaps grads[0]")
    # 2^31 rows of 2^20: more work than a launch can count
    refused(clip([mat(0, (1 << 31) - 1, 1 << 20, dtype=F16)])[0], "too many elements")
    rc, h = clip([a, b])
    assert rc == 0
    run = lib.tgs_gradient_clip_run
    refused(run(None, 1.0, 1.0, 0.0, None, None), "gradient clip is NULL")
    refused(run(h, -1.0, 1.0, 0.0, None, None), "max_norm")
    refused(run(h, math.nan, 1.0, 0.0, None, None), "max_norm")
    for scale in (0.0, -1.0, math.inf, math.nan):
        refused(run(h, 1.0, scale, 0.0, None, None), "scale")
    for eps in (-1.0, math.inf, math.nan):
        refused(run(h, 1.0, 1.0, eps, None, None), "epsilon")
    refused(run(h, 1.0, 1.0, 0.0, BASE * 30 + 2, None), "norm")
    refused(run(h, 1.0, 1.0, 0.0, BASE + 4, None), "norm overlaps")
    refused(lib.tgs_gradient_clip_set_matrices(h, (_lib.tgs_matrix * 2)(a, a), None, 2), "grads[1] overlaps")
    refused(lib.tgs_gradient_clip_set_matrices(None, (_lib.tgs_matrix * 1)(a), None, 1), "gradient clip is NULL")
    assert lib.tgs_gradient_clip_destroy(h) == 0
    assert lib.tgs_gradient_clip_destroy(None) == 0


def test_python_refusals():
    from tinygs_amd.network import LayerOps
    from tinygs_amd.optim import GradientClip
    ops = LayerOps()
    x = torch.zeros(4, 8)
    for call in (lambda: ops.attention(x, x, x, 2), lambda: ops.head_norm(x, 2), lambda: GradientClip([x])):
        with pytest.raises(RuntimeError, match="not on the device"):
            call()
    with pytest.raises(RuntimeError, match="come together"):
        from tinygs_amd.network import _turn
        _turn(x, None)
    for mask, words in ((torch.ones(4, dtype=torch.bool), "mask"), (torch.ones(2, 4, dtype=torch.bool), "mask"),
                        (torch.ones(1, 4), "bool or uint8"), (torch.ones(1, 8, dtype=torch.bool)[:, ::2], "packed")):
        with pytest.raises(RuntimeError, match=words):
            LayerOps._attention(x, x, 2, None, 1, mask, None)
    with pytest.raises(RuntimeError, match="are needed"):
        GradientClip([])
    with pytest.raises(RuntimeError, match="are needed"):
        GradientClip([x], clipped=[])
    with pytest.raises(RuntimeError, match="shape"):
        GradientClip([x], clipped=[x.t()])
