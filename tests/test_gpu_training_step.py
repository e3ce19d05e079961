"""The norm, the layers, the loss and the optimizer together, as a training step uses them."""
import numpy as np
import pytest
import torch
from torch import nn

from conftest import gpu_available, rel_err

from granulelayer_amd import (DenseCrossEntropy, DenseProjection, FusedAdamW, LayerNorm, SparsePoolingLayer,
                              dense_cross_entropy, layer_norm)

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a ROCm GPU")]
DEV = "cuda"
BF, F = torch.bfloat16, torch.float32
CLASSES, WIDTH, POOLS = 1000, 128, 96


class Block(nn.Module):
    """An fp32 residual stream: norm -> projection (gelu) -> sparse pooling layer -> projection back onto the stream."""

    def __init__(self, seed):
        super().__init__()
        self.norm = LayerNorm(WIDTH, out_dtype=BF, device=DEV)
        self.up = DenseProjection(WIDTH, 64, "gelu", device=DEV, seed=seed, bias_std=0.1)
        self.pool = SparsePoolingLayer(64, 3000, POOLS, shared_neurons=None, pooling="mean", dtype=F, device=DEV, seed=seed,
                                       bias_std=0.2)
        self.down = DenseProjection(POOLS, WIDTH, device=DEV, seed=seed + 1)

    def forward(self, x):
        return self.down(self.pool(self.up(self.norm(x)).float()).to(BF), x)


class Model(nn.Module):
    def __init__(self):
        super().__init__()
        self.blocks = nn.ModuleList(Block(10 * i) for i in range(2))
        self.norm = LayerNorm(WIDTH, out_dtype=BF, device=DEV)
        self.head = DenseCrossEntropy(WIDTH, CLASSES, bias=True, device=DEV, seed=5)

    def forward(self, x, target):
        for b in self.blocks:
            x = b(x)
        return self.head(self.norm(x), target)


def batch(seed, tokens=(3, 150)):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(*tokens, WIDTH, generator=g, device=DEV)
    target = torch.randint(0, CLASSES, tokens, generator=g, device=DEV)
    target[:, -20:] = -100
    return x, target


@pytest.mark.parametrize("moments", ["fp32", "bf16", "int8"])
@pytest.mark.parametrize("main", [False, True])
def test_steps_run_and_move_every_parameter(moments, main):
    torch.manual_seed(0)
    model = Model()
    if main:
        for m in model.modules():
            if hasattr(m, "enable_main_grad"):
                m.enable_main_grad()
    params = list(model.parameters())
    opt = FusedAdamW(params, lr=1e-3, moments=moments, weight_decay=0.01)
    for step in range(4):
        was = [p.detach().clone() for p in params]
        loss = model(*batch(step))
        assert loss.dtype == F and torch.isfinite(loss)
        loss.backward()
        opt.step()
        for p, w in zip(params, was):
            assert torch.isfinite(p).all() and not torch.equal(p.detach(), w)
            assert p.grad is None and (not main or not p.main_grad.any())
    for m, v in opt.moment_values():
        assert torch.isfinite(m).all() and (v >= 0).all()


def test_gradients_of_norm_and_head_through_each_other():
    """x -> norm -> head in one graph against float64; roundings: the norm's result (bf16) meets the head's weight, so
    dx carries 2^-8 from it, from dz, and from the gradient at the norm's result (bf16): at most 3 x 2^-8 in all, less
    than half of it on average."""
    g = torch.Generator(device=DEV).manual_seed(1)
    M, K, N = 700, 96, 1500
    x = torch.randn(M, K, generator=g, device=DEV)
    nw, nb = 1 + 0.2 * torch.randn(K, generator=g, device=DEV), 0.1 * torch.randn(K, generator=g, device=DEV)
    w = (0.2 * torch.randn(N, K, generator=g, device=DEV)).to(BF)
    target = torch.randint(0, N, (M,), generator=g, device=DEV)
    target[::5] = -100
    leaves = [t.requires_grad_(True) for t in (x, nw, nb, w)]
    loss = dense_cross_entropy(layer_norm(x, nw, nb, out_dtype=BF), w, target)
    got = torch.autograd.grad(loss, leaves)
    ref = [t.detach().cpu().double().requires_grad_(True) for t in leaves]
    h = torch.nn.functional.layer_norm(ref[0], (K,), ref[1], ref[2])
    want = torch.nn.functional.cross_entropy(h @ ref[3].t(), target.cpu())
    assert abs(float(loss.detach()) - float(want.detach())) < 2.0 ** -8 * float(want.detach())
    for a, b in zip(got, torch.autograd.grad(want, ref)):
        assert rel_err(a.detach().cpu().float().numpy(), b.numpy()) < 3 * 2.0 ** -8


def test_a_captured_step_replays():
    """Forward, backward into main_grad and the update in one graph, with eager work between the replays."""
    torch.manual_seed(0)
    model, other = Model(), Model()
    other.load_state_dict(model.state_dict())
    for net in (model, other):
        for m in net.modules():
            if hasattr(m, "enable_main_grad"):
                m.enable_main_grad()
    x, target = batch(7)
    sx, st = x.clone(), target.clone()

    def passes(net, a, b):
        loss = net(a, b)
        loss.backward()
        return loss.detach()

    for net in (model, other):  # schedules and edge lists are built on the first call
        passes(net, sx, st)
        for m in net.modules():
            if hasattr(m, "zero_main_grad"):
                m.zero_main_grad()
            elif hasattr(m, "enable_main_grad"):
                for p in m.parameters():
                    p.main_grad.zero_()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = passes(model, sx, st)
    for k in range(3):
        a, b = batch(20 + k)
        sx.copy_(a)
        st.copy_(b)
        graph.replay()
        want = passes(other, a, b)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        for p, q in zip(model.parameters(), other.parameters()):
            assert torch.equal(p.main_grad, q.main_grad)
