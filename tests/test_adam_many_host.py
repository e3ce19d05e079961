"""FusedAdamW over many tensors, CPU side: what it and the C entry points refuse before any device use."""
import ctypes

import pytest
import torch

from granulelayer_amd import FusedAdamW
from granulelayer_amd import _native as N


def test_moments_kinds():
    p = torch.nn.Parameter(torch.zeros(4))
    for kind in ("fp32", "bf16", "int8"):
        assert FusedAdamW([p], moments=kind).moments == kind
    with pytest.raises(ValueError):
        FusedAdamW([p], moments="int4")


def test_new_state_of_8bit_moments():
    p = torch.nn.Parameter(torch.zeros(3, 100, dtype=torch.bfloat16))
    st = FusedAdamW([p], moments="int8", master_weights=True)._new_state(p)
    assert st["m"].dtype == torch.int8 and st["v"].dtype == torch.uint8 and st["m"].shape == p.shape
    assert st["m_scale"].shape == st["v_scale"].shape == (2,) and st["master"].dtype == torch.float32


def test_a_refused_tensor_leaves_every_state_as_it_was():
    good, bad = torch.nn.Parameter(torch.zeros(8)), torch.nn.Parameter(torch.zeros(8, dtype=torch.float16))
    for p in (good, bad):
        p.grad = torch.ones_like(p)
    opt = FusedAdamW([good, bad])
    with pytest.raises(NotImplementedError):
        opt.step()
    assert not opt.state and good.grad is not None


@pytest.mark.parametrize("grad,error", [(torch.zeros(7), ValueError), (torch.zeros(8, dtype=torch.bfloat16), TypeError),
                                        (torch.zeros(16)[::2], ValueError)])
def test_main_grads_that_do_not_fit(grad, error):
    p = torch.nn.Parameter(torch.zeros(8))
    p.main_grad = grad
    with pytest.raises(error):
        FusedAdamW([p]).step()


def test_states_that_do_not_fit():
    p = torch.nn.Parameter(torch.zeros(300))
    opt = FusedAdamW([p], moments="int8")
    good = opt._new_state(p)
    assert opt._check_state(p, good) == torch.int8
    for key, value in (("m", torch.zeros(299, dtype=torch.int8)), ("m_scale", torch.zeros(1)),
                       ("v_scale", torch.zeros(3)), ("v", torch.zeros(600, dtype=torch.uint8)[::2])):
        with pytest.raises(ValueError):
            opt._check_state(p, dict(good, **{key: value}))
    for key, value in (("m", torch.zeros(300)), ("v", torch.zeros(300, dtype=torch.int8)),
                       ("m_scale", torch.zeros(2, dtype=torch.float64)), ("master", torch.zeros(300))):
        with pytest.raises(TypeError):
            opt._check_state(p, dict(good, **{key: value}))


def test_the_c_entry_points_refuse():
    lib = N.library()

    def call(name="gl_adam", tensors=None, **kw):
        t = tensors if tensors is not None else [dict(p=16, g=16, m=16, v=16, m_scale=16, v_scale=16, n=5)]
        arr = (N.GlAdamTensor * max(1, len(t)))(*[N.GlAdamTensor(**x) for x in t])
        a = N.GlAdamArgs(tensors=ctypes.addressof(arr), **{"count": len(t), **kw})
        return getattr(lib.lib, name)(ctypes.byref(a), None)

    ok = dict(p=16, g=16, m=16, v=16, m_scale=16, v_scale=16, n=5)
    i8 = N.GL_MOMENTS_INT8
    assert lib.lib.gl_adam(None, None) == -1 and lib.lib.gl_adam_values(None, None) == -1
    empty = N.GlAdamArgs(moments_dtype=N.GL_MOMENTS_INT8)
    assert lib.lib.gl_adam_values(ctypes.byref(empty), None) == -1  # of tensors only
    assert call(count=-1) == -1
    assert call(tensors=[]) == 0 and call(tensors=[dict(n=0)]) == 0  # nothing to do
    assert call(tensors=[dict(ok, n=-1)]) == -1
    assert call(tensors=[dict(ok, n=(1 << 35) + 1)]) == -2
    assert call(p_dtype=2) == -2 and call(g_dtype=2) == -2 and call(moments_dtype=3) == -2
    assert call(stochastic=1) == -1
    for key in ("p", "g", "m", "v"):
        assert call(tensors=[dict(ok, **{key: 0})]) == -1
        assert call(tensors=[dict(ok, **{key: 17})]) == -1  # off its element
    for key in ("m_scale", "v_scale"):
        assert call(tensors=[dict(ok, **{key: 0})], moments_dtype=i8) == -1
        assert call(tensors=[dict(ok, **{key: 18})], moments_dtype=i8) == -1
    assert call(tensors=[ok, dict(ok, master=16)], p_dtype=1) == -1  # a master for all or for none
    assert call(tensors=[dict(ok, master=16)]) == -1  # of an fp32 parameter
    assert call("gl_adam_values") == -1  # fp32 moments are their values
    assert call("gl_adam_values", tensors=[], moments_dtype=i8) == 0
