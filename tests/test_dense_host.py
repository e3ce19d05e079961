"""Refusals and host logic of the dense projection and of activations in 8 bits (no GPU)."""
import ctypes

import pytest
import torch

from granulelayer_amd import (CoverTopK16Layer, DenseProjection, SparsePoolingLayer, dense_projection,
                              pack_activation)
from granulelayer_amd import _native as N

BF, F32 = torch.bfloat16, torch.float32


def test_refused_arguments():
    x, w = torch.zeros(4, 8), torch.zeros(6, 8)
    for bad in (dict(activation="tanh"), dict(activation_checkpoint="fp8"), dict(bias=torch.zeros(8)),
                dict(residual=torch.zeros(4, 8)), dict(residual=torch.zeros(1, 6)), dict(residual=torch.zeros(6))):
        with pytest.raises(ValueError):
            dense_projection(x, w, **bad)
    for bad in ((x, w[:, :7]), (x, w[0]), (x, w[:0]), (torch.zeros(4, 7), w), (torch.tensor(1.0), w)):
        with pytest.raises(ValueError):
            dense_projection(*bad)
    for bad in (dict(x=x.half(), weight=w.half()), dict(x=x.bfloat16(), weight=w), dict(x=x, weight=w, bias=torch.zeros(6).bfloat16()),
                dict(x=x, weight=w, residual=torch.zeros(4, 6).half()), dict(x=x.double(), weight=w.double())):
        with pytest.raises(TypeError):
            dense_projection(**bad)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        dense_projection(x, w)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        dense_projection(x, w.requires_grad_(True))
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        pack_activation(x)
    for bad in (torch.tensor(1.0), torch.zeros(3, 0)):
        with pytest.raises(ValueError):
            pack_activation(bad)


def test_module():
    lay = DenseProjection(64, 48, "relu", dtype=F32, seed=3, bias_std=0.1)
    again = DenseProjection(64, 48, "relu", dtype=F32, seed=3, bias_std=0.1)
    assert torch.equal(lay.weight, again.weight) and torch.equal(lay.bias, again.bias)
    assert sorted(lay.state_dict()) == ["bias", "weight"] and lay.weight.shape == (48, 64)
    assert abs(float(lay.weight.detach().std()) * 8 - 1) < 0.1  # 3072 values: the deviation is good to 1.3%
    assert DenseProjection(64, 48, bias=False).bias is None
    lay.enable_main_grad()
    assert lay.weight.main_grad.dtype == F32 and lay.bias.main_grad.shape == (48,)
    assert "activation_checkpoint=exact" in repr(lay)
    for bad in (dict(activation="swish"), dict(activation_checkpoint="int4")):
        with pytest.raises(ValueError):
            DenseProjection(8, 8, **bad)
    with pytest.raises(ValueError):
        DenseProjection(0, 8)
    with pytest.raises(NotImplementedError):
        DenseProjection(8, 8, dtype=torch.float16)


def test_library_refuses_before_the_device():
    L = N.library().lib
    out = ctypes.c_size_t()

    def pack(**kw):
        base = dict(x=4096, sx=40, rows=4, cols=40, x_dtype=0, q=4096, e=4096)
        return L.gl_pack8(ctypes.byref(N.GlPack8Args(**dict(base, **kw))), None)

    for bad in (dict(rows=-1), dict(cols=0), dict(cols=N.DENSE_MAX_FEATURES + 1), dict(x=0), dict(q=0), dict(e=0), dict(sx=39),
                dict(x=4098), dict(q=4100)):
        assert pack(**bad) == -1, bad
    for bad in (dict(x_dtype=2), dict(rows=1 << 26)):
        assert pack(**bad) == -2, bad
    assert pack(rows=0, x=0, q=0, e=0) == 0
    assert L.gl_pack8(None, None) == -1 and L.gl_unpack8(None, None) == -1

    def fwd(query=True, **kw):
        base = dict(X=4096, sx=64, W=8192, sw=64, Y=16384, sy=48, M=100, N=48, K=64, dtype=1, y_dtype=1)
        a = N.GlDenseArgs(**dict(base, **kw))
        return L.gl_dense_fwd_workspace(ctypes.byref(a), ctypes.byref(out)) if query else L.gl_dense_fwd(ctypes.byref(a), None)

    assert fwd() == 0
    for bad in (dict(X=0), dict(W=0), dict(Y=0), dict(sx=63), dict(sw=63), dict(sy=47), dict(M=-1), dict(N=0), dict(K=0),
                dict(act=3), dict(keep=4), dict(keep=2), dict(keep=3, z=4096), dict(X=4097), dict(bias=4097),
                dict(res=4096, sr=47, res_dtype=1), dict(res=4098, sr=48, res_dtype=0), dict(keep=1, z=4100)):
        assert fwd(**bad) == -1 and fwd(False, **bad) == -1, bad
    for bad in (dict(dtype=2), dict(y_dtype=7), dict(res=4096, sr=48, res_dtype=9), dict(N=N.DENSE_MAX_FEATURES + 1),
                dict(M=1 << 26)):
        assert fwd(**bad) == -2, bad
    # more workgroups than a launch has
    big = dict(M=(1 << 26) - 1, N=1 << 20, K=1 << 20, sx=1 << 20, sw=1 << 20, sy=1 << 20)
    assert fwd(**big) == -2 and fwd(False, **big) == -2
    # odd rows are copied through workspace, which has to be there, aligned and large enough
    assert fwd(sx=65) == 0 and out.value >= 100 * 64 * 2
    assert fwd(False, sx=65) == -3 and fwd(False, sx=65, ws_bytes=1 << 20) == -1
    assert fwd(False, sx=65, ws=4096 + 16, ws_bytes=1 << 20) == -1
    assert fwd(False, sx=65, ws=4096, ws_bytes=100) == -3
    assert fwd(False, M=0, X=0, W=0, Y=0) == 0

    def bwd(query=True, **kw):
        base = dict(dY=4096, sdy=48, X=4096, sx=64, W=8192, sw=64, M=100, N=48, K=64, dtype=1, dy_dtype=1, dX=4096, dW=4096,
                    db=4096, g_dtype=1)
        a = N.GlDenseBwdArgs(**dict(base, **kw))
        return L.gl_dense_bwd_workspace(ctypes.byref(a), ctypes.byref(out)) if query else L.gl_dense_bwd(ctypes.byref(a), None)

    assert bwd() == 0 and bwd(act=1, keep=1, z=4096) == 0 and bwd(act=2, keep=3, z=4096, z_exp=4096) == 0
    for bad in (dict(dY=0), dict(sdy=47), dict(act=1), dict(act=2, keep=1, z=4096), dict(act=0, keep=2, z=4096),
                dict(act=2, keep=2), dict(act=2, keep=3, z=4096), dict(W=0), dict(X=0), dict(X=0, xq=4096), dict(sx=3),
                dict(accumulate=1), dict(dX=4097), dict(X=0, xq=4100, xe=4096)):
        assert bwd(**bad) == -1 and bwd(False, **bad) == -1, bad
    for bad in (dict(dtype=3), dict(dy_dtype=3), dict(g_dtype=3), dict(K=N.DENSE_MAX_FEATURES + 1)):
        assert bwd(**bad) == -2, bad
    big = dict(M=(1 << 26) - 1, N=1 << 20, K=1 << 20, sx=1 << 20, sw=1 << 20, sdy=1 << 20)
    assert bwd(**big) == -2 and bwd(False, **big) == -2
    assert bwd(False, ws=4096, ws_bytes=8) == -3
    assert bwd(False, M=0, dY=0) == 0


@pytest.mark.parametrize("form", ["sparse", "cover"])
def test_sparse_layers_take_the_option(form):
    def make(**kw):
        if form == "sparse":
            return SparsePoolingLayer(64, 2048, 8, shared_neurons=None, pooling="mean", dtype=F32, **kw)
        return CoverTopK16Layer(64, 2048, 8, 256, **kw)

    assert make().activation_checkpoint == "exact"
    assert make(activation_checkpoint="int8").activation_checkpoint == "int8"
    with pytest.raises(ValueError, match="activation_checkpoint"):
        make(activation_checkpoint="int2")


def test_row_limit_is_what_launches_hold():
    """64 threads a row in workgroups of 4 rows: from 2^26 - 3 rows on that is 2^32 threads, more than a launch has.  Such
    calls are refused before they reach the device, with a query and without."""
    L = N.library().lib
    out = ctypes.c_size_t()
    for M, code in (((1 << 26) - 4, 0), ((1 << 26) - 3, -2), ((1 << 26) - 1, -2)):
        f = N.GlDenseArgs(X=4096, sx=9, W=8192, sw=9, Y=16384, sy=8, M=M, N=8, K=9, dtype=1, y_dtype=1)
        assert L.gl_dense_fwd_workspace(ctypes.byref(f), ctypes.byref(out)) == code
        b = N.GlDenseBwdArgs(dY=4096, sdy=8, X=4096, sx=9, W=8192, sw=9, M=M, N=8, K=9, dtype=1, dy_dtype=1, dX=4096, dW=4096,
                             db=4096, g_dtype=1)
        assert L.gl_dense_bwd_workspace(ctypes.byref(b), ctypes.byref(out)) == code
        if code:
            p = N.GlPack8Args(x=4096, sx=512, rows=M, cols=512, x_dtype=1, q=4096, e=4096)
            assert L.gl_dense_fwd(ctypes.byref(f), None) == code and L.gl_dense_bwd(ctypes.byref(b), None) == code
            assert L.gl_pack8(ctypes.byref(p), None) == code and L.gl_unpack8(ctypes.byref(p), None) == code


@pytest.mark.parametrize("answers,calls", [([0], 1), ([-3, 0], 2), ([-1], 1), ([2], 1), ([719, 0], 1), ([-3, 2], 2)])
def test_only_a_missing_workspace_is_asked_for(monkeypatch, answers, calls):
    """The forward is issued a second time where the first one wants a workspace, and for no other error: kernels may have
    been enqueued before it."""
    from types import SimpleNamespace

    from granulelayer_amd import backend as B

    seen = []

    def fwd(a, stream):
        seen.append(a._obj.ws_bytes)
        return answers[len(seen) - 1]

    def query(a, out):
        out._obj.value = 512
        return 0

    lib = N.Library.__new__(N.Library)
    lib.lib = SimpleNamespace(gl_dense_fwd=fwd, gl_dense_fwd_workspace=query, gl_error_string=lambda code: b"it failed")
    monkeypatch.setattr(B, "_on", lambda dev: B._NO_SWITCH)
    monkeypatch.setattr(B, "_stream", lambda dev: 0)
    be = B.HipBackend(lib)
    args = (torch.zeros(3, 8), torch.zeros(5, 8), None, None, "identity", "none")
    if answers[-1] == 0 and calls == len(answers):
        assert be.dense_forward(*args)[0].shape == (3, 5)
    else:
        with pytest.raises(N.NativeError, match=f"gl_dense_fwd failed .code {answers[calls - 1]}: it failed"):
            be.dense_forward(*args)
    assert seen == [0, 512][:calls]


class _Products:
    """The dense products of an identity projection in plain torch."""

    def dense_forward(self, x, w, b, res, activation, keep):
        return x @ w.t() + (0 if b is None else b), None, None

    def dense_backward(self, dy, activation, keep, z, z_exp, x, xq, xe, w, dx, dw, db, accumulate):
        for out, grad, add in ((dx, lambda: dy @ w, False), (dw, lambda: dy.t() @ x, accumulate),
                               (db, lambda: dy.sum(0), accumulate)):
            if out is not None:
                out.copy_(grad() + out if add else grad())


@pytest.fixture
def plain_products(monkeypatch):
    from granulelayer_amd import dense

    monkeypatch.setattr(dense, "backend_for", lambda dev: _Products())


@pytest.mark.parametrize("main_grad", [False, True])
@pytest.mark.parametrize("x_grad", [False, True])
def test_the_bias_may_change_before_the_backward(plain_products, x_grad, main_grad):
    """No gradient is computed from it, so F.linear allows it too; a changed weight is refused."""
    x = torch.randn(5, 3, requires_grad=x_grad)
    w, b = torch.randn(4, 3, requires_grad=True), torch.randn(4, requires_grad=True)
    dy = torch.randn(5, 4)
    y = dense_projection(x, w, b)
    if main_grad:
        w.main_grad, b.main_grad = torch.ones(4, 3), torch.ones(4)
    with torch.no_grad():
        b.add_(1)
    y.backward(dy)
    got = (w.main_grad - 1, b.main_grad - 1) if main_grad else (w.grad, b.grad)
    torch.testing.assert_close(got[0], dy.t() @ x.detach())
    torch.testing.assert_close(got[1], dy.sum(0))
    assert not main_grad or (w.grad is None and b.grad is None)
    if x_grad:
        assert torch.equal(x.grad, dy @ w.detach())
    y = dense_projection(x, w, b)
    with torch.no_grad():
        w.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward(dy)


def test_a_computed_bias_is_not_held(plain_products):
    import weakref

    x, w, b = torch.randn(5, 3), torch.randn(4, 3), torch.randn(4, requires_grad=True)
    b2 = b * 2
    y = dense_projection(x, w, b2)
    gone = weakref.ref(b2)
    del b2
    assert gone() is None
    dy = torch.randn(5, 4)
    y.backward(dy)
    torch.testing.assert_close(b.grad, 2 * dy.sum(0))


def test_under_activation_checkpointing(plain_products):
    from torch.utils.checkpoint import checkpoint

    x, w, b = (torch.randn(*s, requires_grad=True) for s in ((5, 3), (4, 3), (4,)))

    def call(x):
        return dense_projection(x, w * 2, b * 2)

    want = torch.autograd.grad(call(x).sum(), (x, w, b))
    got = torch.autograd.grad(checkpoint(call, x, use_reentrant=False).sum(), (x, w, b))
    for g, t in zip(got, want):
        assert torch.equal(g, t)
