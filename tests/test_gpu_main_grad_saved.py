"""Gradients reach ``main_grad`` also where saved tensors come back as other tensors: under activation checkpointing, kept on the
host, and when the buffers are attached between the passes."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

from conftest import gpu_available

from granulelayer_amd import DenseCrossEntropy, DenseProjection, FusedAdamW, LayerNorm, SparsePoolingLayer

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a ROCm GPU")]
DEV = "cuda"
F = torch.float32


def _layers():
    level = dict(type="mean", activation="relu")
    return {
        "norm": lambda: LayerNorm(64, device=DEV),
        "norm without bias": lambda: LayerNorm(64, bias=False, device=DEV),
        "dense": lambda: DenseProjection(64, 32, "gelu", dtype=F, device=DEV),
        "dense in 8 bits": lambda: DenseProjection(64, 32, "gelu", dtype=F, activation_checkpoint="int8", device=DEV),
        "loss": lambda: DenseCrossEntropy(64, 100, bias=True, dtype=F, device=DEV),
        "sparse": lambda: SparsePoolingLayer(64, 512, 16, shared_neurons=None, pooling="mean", dtype=F, device=DEV),
        "two levels": lambda: SparsePoolingLayer(64, 1024, 8, shared_neurons=None, dtype=F, device=DEV,
                                                 pooling=dict(levels=[dict(level, neurons_per_shard=32), dict(type="sum")])),
    }


@pytest.mark.parametrize("kind", list(_layers()))
@pytest.mark.parametrize("how", ["checkpoint", "host", "late"])
def test_gradients_go_to_main_grad(kind, how):
    torch.manual_seed(0)
    lay = _layers()[kind]()
    x = torch.randn(300, 64, device=DEV, requires_grad=True)
    args = (x, torch.randint(0, 100, (300,), device=DEV)) if kind == "loss" else (x,)

    def backward(y):
        y.square().sum().backward()
        out = [p.main_grad.clone() for p in lay.parameters() if getattr(p, "main_grad", None) is not None]
        grads, x.grad = x.grad, None
        return out, grads

    lay.enable_main_grad()
    want, want_x = backward(lay(*args))
    assert all(w.any() for w in want)
    lay.zero_main_grad()
    if how == "checkpoint":
        y = checkpoint(lay, *args, use_reentrant=False)
    elif how == "host":
        with torch.autograd.graph.save_on_cpu():
            y = lay(*args)
    else:
        buffers = [p.main_grad for p in lay.parameters()]
        for p in lay.parameters():
            del p.main_grad
        y = lay(*args)
        for p, b in zip(lay.parameters(), buffers):
            p.main_grad = b
    got, got_x = backward(y)
    assert torch.equal(got_x, want_x)
    for p, a, b in zip(lay.parameters(), got, want):
        assert p.grad is None and torch.equal(a, b)


def test_a_checkpointed_training_step_moves_the_parameters():
    torch.manual_seed(0)
    lay = DenseProjection(64, 64, "relu", dtype=F, device=DEV)
    lay.enable_main_grad()
    opt = FusedAdamW(lay.parameters(), lr=1e-2, moments="fp32")
    was = [p.detach().clone() for p in lay.parameters()]
    checkpoint(lay, torch.randn(100, 64, device=DEV), use_reentrant=False).sum().backward()
    opt.step()
    assert all(not torch.equal(p, w) for p, w in zip(lay.parameters(), was))


def test_a_computed_weight_is_not_held():
    import weakref

    from granulelayer_amd import dense_cross_entropy, dense_projection, layer_norm

    x = torch.randn(20, 64, device=DEV)
    for call in (lambda w, b: dense_projection(x, w, b), lambda w, b: layer_norm(x, w[0], b), lambda w, b: dense_cross_entropy(
            x, w, torch.zeros(20, device=DEV, dtype=torch.int64), b)):
        w, b = torch.randn(64, 64, device=DEV, requires_grad=True), torch.randn(64, device=DEV, requires_grad=True)
        w2, b2 = w * 2, b * 2
        y = call(w2, b2)
        gone = weakref.ref(w2)
        del w2, b2
        y.sum().backward()
        assert gone() is None and w.grad.any()
