"""Forward, backward into main_grad and FusedAdamW's step captured into one graph."""
import pytest
import torch

from conftest import gpu_available

from granulelayer_amd import FusedAdamW
from test_gpu_training_step import Model, batch

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a ROCm GPU")]


def _make(moments):
    torch.manual_seed(0)
    model = Model()
    for m in model.modules():
        if hasattr(m, "enable_main_grad"):
            m.enable_main_grad()
    return model, FusedAdamW(list(model.parameters()), lr=1e-3, moments=moments, weight_decay=0.01)


def _pass(model, opt, x, target):
    loss = model(x, target)
    loss.backward()
    opt.step()
    return loss.detach()


@pytest.mark.parametrize("moments", ["fp32", "bf16", "int8"])
def test_a_captured_step_with_its_update_replays(moments):
    """A replay has the corrections and seeds of its capture, so the eager step beside it is set back to them."""
    model, opt = _make(moments)
    other, beside = _make(moments)
    x, target = batch(7)
    sx, st = x.clone(), target.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # schedules, edge lists and states are made on the first call
        _pass(model, opt, sx, st)
    torch.cuda.current_stream().wait_stream(side)
    _pass(other, beside, x, target)
    torch.cuda.synchronize()
    seed = opt._seed
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = _pass(model, opt, sx, st)
    assert all(s["step"] == 2 for s in opt.state.values())
    for k in range(4):
        a, b = batch(20 + k)
        sx.copy_(a)
        st.copy_(b)
        graph.replay()
        beside._seed = seed
        for s in beside.state.values():
            s["step"] = 1
        want = _pass(other, beside, a, b)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        for p, q in zip(model.parameters(), other.parameters()):
            assert torch.equal(p, q) and not p.main_grad.any() and not q.main_grad.any()
            for key, value in opt.state[p].items():
                assert key == "step" or torch.equal(value, beside.state[q][key]), (k, key)


def test_replayed_8bit_moments_decay():
    """Steps replayed from one capture draw anew: moments of gradients that stopped go on decaying.  Codes of 120 and more are
    off by sqrt(10 / 120) at most, sqrt(10 / 120) / sqrt(4096) = 0.45% of their mean; five times."""
    n = 8192
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    opt = FusedAdamW([p], moments="int8", lr=1e-3)
    stopped = torch.arange(n, device="cuda") % 2 == 1
    p.main_grad = torch.zeros(n, device="cuda")
    exact = torch.zeros(n, device="cuda", dtype=torch.float64)
    for _ in range(200):
        p.main_grad.fill_(1.0)
        opt.step()
        exact.mul_(0.999).add_(0.001)
    grad = torch.where(stopped, 0.0, 1.0)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        p.main_grad.copy_(grad)
        opt.step()
    for _ in range(1500):
        graph.replay()
        exact.mul_(0.999).add_(0.001 * grad.double())
    m, v = opt.moment_values()[0]
    assert not m[stopped].any()
    assert abs(float(v.double()[stopped].mean() / exact[stopped].mean()) - 1) < 0.0226
