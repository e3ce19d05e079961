"""The exponentials that the cross entropy's forward keeps are saved tensors: what checkpoints and hooks make of them, and when
their memory goes."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

from conftest import gpu_available

from granulelayer_amd import dense_cross_entropy
from test_gpu_cross_entropy import check, definition, inputs

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a ROCm GPU")]
DEV = "cuda"
BF, F = torch.bfloat16, torch.float32
M, K, N = 1500, 520, 20000  # 60 MB of bf16 exponentials
EXPS = M * N * 2


def _leaves(t):
    return [t[k].detach().requires_grad_(True) for k in "xwb"]


def _held(f):
    """f's result and the bytes that it left allocated."""
    torch.cuda.synchronize()
    was = torch.cuda.memory_allocated()
    out = f()
    torch.cuda.synchronize()
    return out, torch.cuda.memory_allocated() - was


def _check(t, grads):
    want = definition(t, "mean", torch.ones((), device=DEV))
    for v, name in zip(grads, ("dx", "dw", "db")):
        check(v, want, name)


def test_a_checkpointed_loss_holds_no_exponentials():
    t = inputs(M, K, N, BF)
    leaves = _leaves(t)
    plain, held = _held(lambda: dense_cross_entropy(leaves[0], leaves[1], t["target"], leaves[2]))
    assert held > EXPS
    want = torch.autograd.grad(plain, leaves)
    del plain
    loss, held = _held(lambda: checkpoint(dense_cross_entropy, leaves[0], leaves[1], t["target"], leaves[2], use_reentrant=False))
    assert held < EXPS // 8
    torch.cuda.reset_peak_memory_stats()
    was = torch.cuda.memory_allocated()
    got = torch.autograd.grad(loss, leaves)
    peak = torch.cuda.max_memory_allocated() - was
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    # one place of exponentials, gradients and the forward's and backward's own workspaces
    assert peak < EXPS + 3 * (N * K + M * K) * 2 + (64 << 20)


@pytest.mark.parametrize("dtype", [BF, F])
def test_hooks_on_saved_tensors(dtype):
    """Kept on the host, at another address, and cut out of a buffer with something else in it."""
    t = inputs(300, K, 900, dtype)
    leaves = _leaves(t)
    want = torch.autograd.grad(dense_cross_entropy(leaves[0], leaves[1], t["target"], leaves[2]), leaves)
    packed = []

    def to_host(x):
        packed.append(x.numel() * x.element_size())
        return x.cpu()

    def off(x):  # 8 bytes from where allocations begin, others' values around
        flat = torch.full((x.numel() + 32,), 7, device=x.device, dtype=x.dtype)
        n = 16 if x.dtype == torch.uint8 else 8
        flat[n:n + x.numel()] = x.reshape(-1)
        return flat, n, x.shape

    buffers = []

    def on(saved):
        flat, n, shape = saved
        buffers.append((flat, n, shape.numel()))
        return flat[n:n + shape.numel()].view(shape)

    for pack, unpack in ((to_host, lambda x: x.to(DEV)), (off, on)):
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            loss = dense_cross_entropy(leaves[0], leaves[1], t["target"], leaves[2])
        got = torch.autograd.grad(loss, leaves)
        if pack is to_host:
            assert max(packed) >= 300 * 900 * (2 if dtype == BF else 4)  # the exponentials are among them
            for a, b in zip(got, want):
                assert torch.equal(a, b)
        else:
            _check(t, got)
            for flat, n, size in buffers:
                assert (flat[:n] == 7).all() and (flat[n + size:] == 7).all()


def test_a_retained_graph_lets_go_of_them():
    t = inputs(M, K, N, BF)
    leaves = _leaves(t)
    (loss, held) = _held(lambda: dense_cross_entropy(leaves[0], leaves[1], t["target"], leaves[2]))
    grads, more = _held(lambda: torch.autograd.grad(loss, leaves, retain_graph=True))
    assert held > EXPS and more < (N * K + M * K + N) * 2 - EXPS + (4 << 20)
    _check(t, grads)
    for _ in range(2):
        _check(t, torch.autograd.grad(loss, leaves, retain_graph=True))


def test_a_checkpoint_backward_twice():
    t = inputs(300, K, 900, BF)
    leaves = _leaves(t)
    loss = checkpoint(dense_cross_entropy, leaves[0], leaves[1], t["target"], leaves[2], use_reentrant=False)
    for last in (False, False, True):
        _check(t, torch.autograd.grad(loss, leaves, retain_graph=not last))


def test_a_captured_checkpointed_pass():
    t = inputs(300, K, 900, BF)
    x, w, b = leaves = _leaves(t)
    target = t["target"].clone()

    def passes():
        loss = checkpoint(dense_cross_entropy, x, w, target, b, use_reentrant=False, preserve_rng_state=False)
        return (loss.detach(), *torch.autograd.grad(loss, leaves))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        passes()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = passes()
    for k in range(3):
        other = inputs(300, K, 900, BF, seed=k)
        with torch.no_grad():
            x.copy_(other["x"])
        target.copy_(other["target"])
        graph.replay()
        want = passes()
        torch.cuda.synchronize()
        for a, c in zip(out, want):
            assert torch.equal(a, c)
