"""Layer norm on the GPU against the definition in float64, element by element within bounds of its roundings."""
import numpy as np
import pytest
import torch

from conftest import gpu_available

from granulelayer_amd import LayerNorm, layer_norm

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a ROCm GPU")]
DEV = "cuda"
E = 2.0 ** -24  # half a last place of fp32
BF, F = torch.bfloat16, torch.float32
HALF = {BF: 2.0 ** -8, F: E}


def make(M, D, dtype, par, out, seed=0, pitch=0):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*s):
        return torch.randn(*s, generator=g, device=DEV)

    x = (normal(M, D + pitch) * torch.exp(normal(1, D + pitch)) + normal(1, D + pitch)).to(dtype)[:, :D]
    return x, (1 + 0.3 * normal(D)).to(par), (0.2 * normal(D)).to(par), normal(M, D).to(out)


def definition(x, w, b, dy, eps):
    """(name -> (value, bound of an fp32 evaluation's error)) in float64 on the CPU."""
    x, dy = x.detach().cpu().double().numpy(), dy.detach().cpu().double().numpy()
    M, D = x.shape
    w = np.ones(D) if w is None else w.detach().cpu().double().numpy()
    b = np.zeros(D) if b is None else b.detach().cpu().double().numpy()
    n = 40 + D / 1024  # additions in a row that a term of a row's sum goes through
    mean = x.mean(1, keepdims=True)
    r = 1 / np.sqrt(((x - mean) ** 2).mean(1, keepdims=True) + eps)
    h = (x - mean) * r
    # the mean: n sums, 1 / D and its product; r: its sum, square, products and root, a square root halves what is
    # before it; x - mean and its product with r one each
    d_mean = (n + 3) * E * np.abs(x).mean(1, keepdims=True)
    d_r = ((n + 6) / 2 + 3) * E
    d_h = r * d_mean + np.abs(h) * (d_r + 2 * E)
    y = h * w + b
    g = dy * w
    s0, s1 = g.mean(1, keepdims=True), (g * h).mean(1, keepdims=True)
    d_s0 = (n + 3) * E * np.abs(g).mean(1, keepdims=True)
    d_s1 = (n + 4) * E * np.abs(g * h).mean(1, keepdims=True) + (np.abs(g) * d_h).mean(1, keepdims=True)
    dx = r * (g - s0 - h * s1)
    d_dx = (r * (E * np.abs(g) + d_s0 + np.abs(h) * d_s1 + np.abs(s1) * d_h + 3 * E * (np.abs(g) + np.abs(s0) + np.abs(h * s1)))
            + np.abs(dx) * (d_r + E))
    nr = M + 60  # and of a column's
    return {"y": (y, np.abs(w) * d_h + E * (np.abs(h * w) + np.abs(y))), "dx": (dx, d_dx),
            "dw": ((dy * h).sum(0), (np.abs(dy) * d_h).sum(0) + nr * E * np.abs(dy * h).sum(0)),
            "db": (dy.sum(0), nr * E * np.abs(dy).sum(0))}


def check(got, want, name):
    value, bound = want[name]
    tol = bound + HALF[got.dtype] * (np.abs(value) + bound) + 1e-38
    off = np.abs(got.detach().cpu().double().numpy() - value) / tol
    assert off.max() <= 1, f"{name}: {off.max():.2f} of the bound at {np.unravel_index(off.argmax(), off.shape)}"


SHAPES = [(1, 1), (5, 1), (3, 2), (1, 7), (9, 8), (33, 64), (257, 131), (65, 511), (7, 512), (6, 513), (777, 1001),
          (4, 1024), (3, 1025), (130, 2048), (5, 2049), (1, 4096), (66, 4095), (5, 4097), (9, 8192), (3, 8193), (4, 16384),
          (3, 16385), (2, 70001)]


@pytest.mark.parametrize("dtype,par,out", [(F, F, F), (BF, BF, BF), (F, F, BF), (F, BF, BF), (BF, F, F)])
@pytest.mark.parametrize("M,D", SHAPES)
def test_forward_and_gradients(M, D, dtype, par, out):
    x, w, b, dy = make(M, D, dtype, par, out, seed=M + D)
    x, w, b = (t.requires_grad_(True) for t in (x, w, b))
    y = layer_norm(x, w, b, 1e-5, out)
    assert y.dtype == out and y.shape == x.shape
    grads = torch.autograd.grad(y, (x, w, b), dy)
    want = definition(x, w, b, dy, 1e-5)
    check(y, want, "y")
    for g, t, name in zip(grads, (x, w, b), ("dx", "dw", "db")):
        assert g.dtype == t.dtype and g.shape == t.shape
        check(g, want, name)
    with torch.no_grad():
        assert torch.equal(layer_norm(x, w, b, 1e-5, out), y)


@pytest.mark.parametrize("D", [300, 3000, 20000])
def test_many_rows(D):
    """More rows than workgroups at a time."""
    M = 40_000_000 // D // 8
    x, w, b, dy = make(M, D, BF, BF, BF, seed=1)
    x, w, b = (t.requires_grad_(True) for t in (x, w, b))
    y = layer_norm(x, w, b)
    grads = torch.autograd.grad(y, (x, w, b), dy)
    want = definition(x, w, b, dy, 1e-5)
    for g, name in zip((y, *grads), ("y", "dx", "dw", "db")):
        check(g, want, name)


@pytest.mark.parametrize("pitch", [1, 3, 8])
@pytest.mark.parametrize("dtype", [F, BF])
def test_strided_rows_and_gradients(pitch, dtype):
    x, w, b, _ = make(50, 777, dtype, F, dtype, seed=2, pitch=pitch)
    wide = torch.randn(50, 777 * 2, device=DEV).to(dtype)
    for dy in (wide[:, :777], wide[:, ::2], wide[:1, :777].expand(50, 777), torch.ones((), device=DEV, dtype=dtype).expand(50, 777)):
        xs, ws, bs = x.detach().requires_grad_(True), w.detach().requires_grad_(True), b.detach().requires_grad_(True)
        assert xs.stride(0) == 777 + pitch
        grads = torch.autograd.grad(layer_norm(xs, ws, bs), (xs, ws, bs), dy)
        want = definition(x, w, b, dy, 1e-5)
        for g, name in zip(grads, ("dx", "dw", "db")):
            check(g, want, name)


def test_views_dimensions_and_missing_parameters():
    x, w, b, dy = make(24, 96, F, F, F, seed=3)
    want = definition(x, w, b, dy, 1e-5)
    y = layer_norm(x.view(2, 3, 4, 96), w, b)
    assert y.shape == (2, 3, 4, 96)
    check(y.view(24, 96), want, "y")
    check(layer_norm(x.t().contiguous().t(), w, b), want, "y")  # features a stride apart
    check(layer_norm(x[5], w, b)[None], {"y": tuple(v[5:6] for v in want["y"])}, "y")
    check(layer_norm(x, w), definition(x, w, None, dy, 1e-5), "y")
    check(layer_norm(x, None, b), definition(x, None, b, dy, 1e-5), "y")
    check(layer_norm(x), definition(x, None, None, dy, 1e-5), "y")
    assert layer_norm(x[:0], w, b).shape == (0, 96)
    neg = torch._neg_view(-x)
    assert neg.is_neg() and torch.equal(layer_norm(neg, w, b), layer_norm(x, w, b))
    for names in ("x", "w", "b", "xw", "xb", "wb"):
        t = {"x": x, "w": w, "b": b}
        t = {k: v.detach().requires_grad_(k in names) for k, v in t.items()}
        grads = torch.autograd.grad(layer_norm(t["x"], t["w"], t["b"]), [t[k] for k in names], torch._neg_view(-dy))
        for k, g in zip(names, grads):
            check(g, want, "d" + k)
    e = x[:0].detach().requires_grad_(True)
    ws = w.detach().requires_grad_(True)
    gx, gw = torch.autograd.grad(layer_norm(e, ws).sum(), (e, ws))
    assert gx.shape == (0, 96) and not gw.any()


def test_gradient_against_differences():
    x, w, b, dy = make(6, 200, F, F, F, seed=4)
    t = [v.requires_grad_(True) for v in (x, w, b)]
    grads = torch.autograd.grad(layer_norm(*t), t, dy)
    gen = torch.Generator(device=DEV).manual_seed(5)
    step = 2.0 ** -7
    for i, g in enumerate(grads):
        u = torch.randn(t[i].shape, generator=gen, device=DEV)
        sides = []
        for s in (step, -step):
            moved = [v.detach() for v in t]
            moved[i] = moved[i] + s * u
            sides.append((layer_norm(*moved).double() * dy.double()).sum())
        slope, want = float(sides[0] - sides[1]) / (2 * step), float((g.double() * u.double()).sum())
        # rounding of y: 2^-23 |y dy| summed over 1200 terms and two sides, over 2 x step: about 0.01; the third
        # derivative's share step^2 / 6 times some r^3 |u|^3: below 1e-3 of |g| |u|
        assert abs(slope - want) < 0.02 + 2e-3 * float(g.norm() * u.norm())


def test_rows_that_are_no_numbers_or_constant():
    x, w, b, dy = make(8, 600, F, F, F, seed=6)
    clean = layer_norm(x, w, b)
    x2 = x.clone()
    x2[2, 5], x2[4, 0], x2[6, 599] = float("nan"), float("inf"), float("-inf")
    xs = x2.requires_grad_(True)
    y = layer_norm(xs, w, b)
    dx, = torch.autograd.grad(y, xs, dy)
    bad = torch.tensor([2, 4, 6], device=DEV)
    good = torch.tensor([0, 1, 3, 5, 7], device=DEV)
    assert torch.isnan(y[bad]).all() and torch.isnan(dx[bad]).all()
    assert torch.equal(y[good], clean[good]) and torch.isfinite(dx[good]).all()
    const = torch.full((3, 600), 7.0, device=DEV)
    assert torch.equal(layer_norm(const, w, b), b.expand(3, 600))  # sums of 600 sevens are whole: the mean is 7


def test_a_graph_of_the_backward_is_refused_where_it_is_used():
    x, w, b, dy = make(9, 300, F, F, F, seed=9)
    xs = x.detach().requires_grad_(True)
    dx, = torch.autograd.grad(layer_norm(xs, w, b), xs, dy, create_graph=True)
    check(dx, definition(x, w, b, dy, 1e-5), "dx")
    with pytest.raises(RuntimeError):
        dx.sum().backward()


def test_main_grad_is_added_to():
    lay = LayerNorm(300, device=DEV, out_dtype=BF)
    x, _, _, dy = make(40, 300, F, F, BF, seed=7)
    with torch.no_grad():
        lay.weight.uniform_(0.5, 1.5)
        lay.bias.uniform_(-1, 1)
    lay.enable_main_grad()
    lay.weight.main_grad.fill_(2.0)
    xs = x.requires_grad_(True)
    for _ in range(2):
        lay(xs).backward(dy)
    assert lay.weight.grad is None and lay.bias.grad is None
    want = definition(x, lay.weight, lay.bias, dy, 1e-5)
    twice = {k: (2 * v, 2 * t + 4 * E * (2 + np.abs(v))) for k, (v, t) in want.items()}
    check(lay.weight.main_grad - 2.0, twice, "dw")
    check(lay.bias.main_grad, twice, "db")
    lay.zero_main_grad()
    assert not lay.weight.main_grad.any()


def test_a_captured_training_pass_and_another_stream():
    x, w, b, dy = make(300, 1500, BF, F, BF, seed=8)
    t = [v.requires_grad_(True) for v in (x, w, b)]

    def passes():
        y = layer_norm(*t)
        return (y, *torch.autograd.grad(y, t, dy))

    eager = passes()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = passes()
    torch.cuda.current_stream().wait_stream(side)
    for a, c in zip(eager, other):
        assert torch.equal(a, c)
    del other, a, c
    eager = [v.detach().clone() for v in eager]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = passes()
    for k in range(3):
        for o in out:
            o.detach().zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(eager, out):
            assert torch.equal(a, c.detach())


def test_rows_past_32_bits():
    """2^16 + 3 rows of 2^15 features of bf16: 4.3 GB, element offsets past 32 bits."""
    M, D = 2 ** 16 + 3, 2 ** 15
    x = torch.zeros(M, D, device=DEV, dtype=BF)
    x[:, ::2] = 2.0  # mean 1, variance 1
    w = torch.full((D,), 3.0, device=DEV, requires_grad=True)
    x.requires_grad_(True)
    y = layer_norm(x, w, None, 0.0)
    assert bool((y.detach()[-5:, ::2] == 3).all()) and bool((y.detach()[-5:, 1::2] == -3).all()) and bool((y[:3, ::2] == 3).all())
    dy = torch.ones(1, device=DEV, dtype=BF).expand(M, D)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert not dx[-5:].any() and not dx[:5].any()  # equal gradients of a row cancel
    assert bool((dw[::2] == M).all()) and bool((dw[1::2] == -M).all())
