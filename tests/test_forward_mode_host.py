"""Forward-mode differentiation is refused, with and without operands that require grad: no tangent is dropped in silence."""
import pytest
import torch
from torch.autograd import forward_ad

from granulelayer_amd import cross_entropy, dense, dense_cross_entropy, dense_projection, layer_norm, norm


class Zeros:
    """Takes the backend's place."""

    def norm_forward(self, x, w, b, eps, out_dtype, keep):
        return torch.zeros_like(x, dtype=out_dtype), torch.zeros(2 * len(x)) if keep else None

    def dense_forward(self, x, w, b, residual, activation, keep):
        return torch.zeros(len(x), len(w)), None, None

    def ce_forward(self, x, w, b, target, reduction, ignore_index, keep, piece_bytes=0):
        return torch.zeros(()), torch.zeros(4 + 5 * len(x), dtype=torch.int32) if keep else None, None


def _norm(x, w):
    return layer_norm(x, w[0], w[1])


def _dense(x, w):
    return dense_projection(x, w)


def _loss(x, w):
    return dense_cross_entropy(x, w, torch.zeros(len(x), dtype=torch.int64))


@pytest.fixture(autouse=True)
def backend(monkeypatch):
    for module in (norm, dense, cross_entropy):
        monkeypatch.setattr(module, "backend_for", lambda device: Zeros())


@pytest.mark.parametrize("call", [_norm, _dense, _loss])
@pytest.mark.parametrize("of", ["x", "w"])
@pytest.mark.parametrize("grad", ["none", "required", "off"])
def test_a_tangent_is_refused(call, of, grad):
    x, w = torch.randn(3, 4), torch.randn(2, 4)
    if grad == "required":
        x.requires_grad_(True)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad != "off"):
        dual = {"x": x, "w": w}
        dual[of] = forward_ad.make_dual(dual[of], torch.ones_like(dual[of]))
        with pytest.raises(NotImplementedError):
            call(**dual)


@pytest.mark.parametrize("call", [_norm, _dense, _loss])
def test_operands_without_a_tangent_go_on(call):
    x, w = torch.randn(3, 4), torch.randn(2, 4)
    with forward_ad.dual_level():
        y = call(x, w)
        assert not y.requires_grad and forward_ad.unpack_dual(y).tangent is None
    assert call(x, w).shape == y.shape
    assert call(x.requires_grad_(True), w).requires_grad
    with torch.no_grad():
        assert not call(x, w).requires_grad


@pytest.mark.parametrize("call", [_norm, _dense, _loss])
def test_transforms_are_refused(call):
    x, w = torch.randn(3, 4), torch.randn(2, 4)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: call(t, w), (x,), (x,))
