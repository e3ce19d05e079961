"""Layer norm, CPU side: what the function, the module and the C entry points refuse before any device use."""
import ctypes

import pytest
import torch

from granulelayer_amd import LayerNorm, layer_norm
from granulelayer_amd import _native as N


def test_arguments_are_checked():
    x, w = torch.zeros(4, 8), torch.ones(8)
    for bad in (dict(weight=torch.ones(7)), dict(bias=torch.ones(1, 8)), dict(eps=-1.0), dict(eps=float("nan"))):
        with pytest.raises(ValueError):
            layer_norm(x, **bad)
    for bad in (dict(weight=w.double()), dict(weight=w, bias=w.bfloat16()), dict(out_dtype=torch.float16)):
        with pytest.raises(TypeError):
            layer_norm(x, **bad)
    with pytest.raises(TypeError):
        layer_norm(x.double())
    for shape in ((), (3, 0)):
        with pytest.raises(ValueError):
            layer_norm(torch.zeros(shape))
    with pytest.raises(ValueError):
        layer_norm(x, torch.ones(8, device="meta"))
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        layer_norm(x, w)


def test_module():
    m = LayerNorm(6, dtype=torch.bfloat16)
    assert m.weight.dtype == torch.bfloat16 and m.bias.shape == (6,) and bool((m.weight == 1).all()) and not m.bias.any()
    assert LayerNorm(6, bias=False).bias is None
    m.enable_main_grad()
    assert m.weight.main_grad.dtype == torch.float32
    for bad in (dict(dim=0), dict(dim=4, eps=-1)):
        with pytest.raises(ValueError):
            LayerNorm(**bad)
    for bad in (dict(dtype=torch.float16), dict(out_dtype=torch.float64)):
        with pytest.raises(NotImplementedError):
            LayerNorm(4, **bad)


def test_the_c_entry_points_refuse():
    lib = N.library()
    out = ctypes.c_size_t()

    def fwd(**kw):
        a = N.GlNormArgs(**{**dict(X=16, Y=16, sx=8, sy=8, M=4, D=8, eps=1e-5), **kw})
        return lib.lib.gl_norm_fwd(ctypes.byref(a), None)

    assert lib.lib.gl_norm_fwd(None, None) == -1 and fwd(M=0) == 0
    for bad in (dict(M=-1), dict(D=0), dict(X=0), dict(Y=0), dict(sx=7), dict(sy=7), dict(X=18), dict(Y=17, y_dtype=1),
                dict(weight=18), dict(bias=17, w_dtype=1), dict(stats=18), dict(eps=-1.0), dict(eps=float("nan"))):
        assert fwd(**bad) == -1, bad
    for bad in (dict(D=(1 << 20) + 1), dict(M=(1 << 40) + 1), dict(x_dtype=2), dict(y_dtype=2), dict(w_dtype=-1)):
        assert fwd(**bad) == -2, bad

    base = dict(X=16, dY=16, stats=16, sx=8, sdy=8, dX=16, dweight=16, dbias=16, M=4, D=8)

    def bwd(name="gl_norm_bwd", **kw):
        a = N.GlNormBwdArgs(**{**base, **kw})
        return lib.lib.gl_norm_bwd(ctypes.byref(a), None) if name == "gl_norm_bwd" else getattr(lib.lib, name)(
            ctypes.byref(a), ctypes.byref(out))

    assert bwd() == -3 and bwd(ws=16, ws_bytes=1 << 30) == -1  # too little, then off 256 bytes
    assert bwd(M=0) == 0 and bwd(dX=0, dweight=0, dbias=0) == 0
    for bad in (dict(M=-1), dict(D=0), dict(X=0), dict(dY=0), dict(stats=0), dict(sx=7), dict(sdy=7), dict(X=18), dict(dX=18),
                dict(dweight=18), dict(dbias=18), dict(accumulate=1, g_dtype=1)):
        assert bwd(**bad) == -1 and bwd("gl_norm_bwd_workspace", **bad) == -1, bad
    for bad in (dict(D=(1 << 20) + 1), dict(x_dtype=2), dict(dy_dtype=2), dict(w_dtype=2), dict(g_dtype=2)):
        assert bwd(**bad) == -2, bad
    assert bwd("gl_norm_bwd_workspace") == 0 and out.value == 256  # one workgroup's 16 sums
    assert bwd("gl_norm_bwd_workspace", dweight=0, dbias=0) == 0 and out.value == 0
    assert bwd("gl_norm_bwd_workspace", M=10 ** 6, D=4096, sx=4096, sdy=4096) == 0 and out.value == 256 * 2 * 4096 * 4
    assert bwd("gl_norm_bwd_workspace", M=1000, D=1 << 20, sx=1 << 20, sdy=1 << 20) == 0
    assert out.value == 64 * 2 * (1 << 20) * 4 + 8192
