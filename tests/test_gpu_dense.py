"""The dense projection and its backward against float64, with bounds from the arithmetic.

Sums of n products in fp32, in any order, are within n 2^-24 sum|terms| of the exact ones (each of at most n
roundings is half a step of at most the terms' sum); twice that covers roundings inside the matrix instructions.
A result rounded to bf16 is within 2^-8 of itself (fp32: 2^-24).  The backward rounds dz to the operands'
type (bf16: 2^-8 of each term); erf and exp are good to a few units in the last place, 1e-6 of gelu's range."""
import math

import pytest
import torch

from granulelayer_amd import DenseProjection, FusedAdamW, dense_projection, pack_activation
from granulelayer_amd.backend import backend_for

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24
HALF = {BF: 2.0 ** -8, F32: 2.0 ** -24}


def act64(z, act):
    return {"identity": lambda: z, "relu": lambda: z.clamp(min=0),
            "gelu": lambda: 0.5 * z * torch.special.erfc(-z / math.sqrt(2))}[act]()


def dact64(z, act):
    if act == "gelu":
        return 0.5 * torch.special.erfc(-z / math.sqrt(2)) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return torch.ones_like(z)


def within(got, want, bound, what):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    err = (got.double() - want).abs()
    bad = ~(err <= bound)
    if bool(bad.any()):
        i = int(torch.where(bad, err, -1.0).nan_to_num(nan=1e300).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside the bound; worst at {i}: got "
                             f"{float(got.reshape(-1)[i])!r} want {float(want.reshape(-1)[i])!r} bound "
                             f"{float(bound.reshape(-1)[i])!r}")


def inputs(M, K, N, dtype, res=None, seed=0):
    gen = torch.Generator().manual_seed(seed + 7 * M + 11 * K + 13 * N)

    def normal(*s):
        return torch.randn(*s, generator=gen).to(DEV)

    t = dict(x=normal(M, K).to(dtype), w=(normal(N, K) / math.sqrt(K)).to(dtype), b=normal(N).to(dtype),
             dy=normal(M, N), res=None if res is None else normal(M, N).to(res))
    t["dy"] = t["dy"].to(torch.promote_types(dtype, res or dtype))
    return t


def check_forward(y, x, w, b, res, act):
    """y against float64 of the same inputs; returns (z, bound of z's error)."""
    x64, w64 = x.double(), w.double()
    K = x.shape[-1]
    z = x64 @ w64.t()
    mag = x64.abs() @ w64.abs().t()
    if b is not None:
        z, mag = z + b.double(), mag + b.double().abs()
    ez = 2 * (K + 2) * U * mag
    want = act64(z, act)
    # |gelu'| <= 1.13; its own error; residual's addition
    bound = 1.13 * ez + (1e-6 * z.abs() if act == "gelu" else 0)
    if res is not None:
        want = want + res.double()
        bound = bound + U * want.abs()
    within(y, want, bound * (1 + HALF[y.dtype]) + HALF[y.dtype] * want.abs() + 1e-37, "y")
    return z, ez


def check_gradients(got, t, act, z_kept, x_kept, positive):
    """dx, dw, db against float64 at what was kept."""
    dtype = t["x"].dtype
    g = t["dy"].double()
    if act == "relu":
        dz, e = torch.where(positive, g, 0.0), torch.zeros_like(g)
    else:
        dz, e = g * dact64(z_kept, act), g.abs() * (1e-6 * (1 + z_kept.abs()) if act == "gelu" else 0.0)
    M, N = dz.shape
    K = t["x"].shape[1]
    r = e + (HALF[dtype] * dz.abs() if act != "identity" or dtype != t["dy"].dtype else 0.0)
    for name, a, ea, b, n in (("dx", dz, r, t["w"].double(), N), ("dw", dz.t(), r.t(), x_kept.double(), M)):
        if got.get(name) is None:
            continue
        want, mag = a @ b, a.abs() @ b.abs()
        bound = ea @ b.abs() + 2 * (n + 2) * U * mag
        h = HALF[got[name].dtype]
        within(got[name], want, bound * (1 + h) + h * want.abs() + 1e-37, name)
    if got.get("db") is not None:
        want = dz.sum(0)
        h = HALF[got["db"].dtype]
        bound = e.sum(0) + 2 * (M + 2) * U * dz.abs().sum(0)
        within(got["db"], want, bound * (1 + h) + h * want.abs() + 1e-37, "db")


def run_training(t, act, ckpt, residual=True):
    leaves = {k: t[k].detach().requires_grad_(True) for k in ("x", "w", "b") if t[k] is not None}
    res = t["res"].detach().requires_grad_(True) if t["res"] is not None else None
    y = dense_projection(leaves["x"], leaves["w"], leaves.get("b"), res, act, activation_checkpoint=ckpt)
    saved = y.grad_fn.saved_tensors
    names = list(leaves) + (["res"] if res is not None else [])
    grads = dict(zip(["d" + n for n in names], torch.autograd.grad(y, list(leaves.values()) + ([res] if res is not None else []),
                                                                   t["dy"])))
    return y.detach(), grads, saved


def check_training(t, act, ckpt):
    y, grads, (x, xq, xe, w, b, z, ze) = run_training(t, act, ckpt)
    z64, ez = check_forward(y, t["x"], t["w"], t["b"], t["res"], act)
    N, K = t["w"].shape
    be = backend_for(y.device)
    if ckpt == "int8":
        x_kept = be.unpack8(xq, xe, K, F32)
        assert torch.equal(x_kept, pack_activation(t["x"]).unpack(F32)) and x is None
    else:
        x_kept = x
    z_kept, positive = None, None
    if act == "relu":
        bits = torch.stack([(z >> i) & 1 for i in range(32)], -1).reshape(z.shape[0], -1)
        positive = bits[:, :N].bool()
        sure = z64.abs() > ez
        assert torch.equal(positive[sure], (z64 > 0)[sure])
        assert not bool(bits[:, N:].any())
    elif act == "gelu":
        if ckpt == "int8":
            z_kept = be.unpack8(z, ze, N, F32).double()
            # half a step of a block: a step is below 1/63.75 of its largest magnitude
            nb = -(-N // 32)
            top = torch.nn.functional.pad(z64.abs() + ez, (0, nb * 32 - N)).reshape(-1, nb, 32).amax(-1)
            half = (top / 63.75 / 2).repeat_interleave(32, 1)[:, :N]
            within(z_kept, z64, ez + half, "kept z")
        else:
            z_kept = z[:, :N].double()
            within(z_kept, z64, ez + HALF[t["x"].dtype] * (z64.abs() + ez), "kept z")
    elif act == "identity":
        z_kept = z64
    check_gradients(grads, t, act, z_kept, x_kept, positive)
    if t["res"] is not None:
        assert torch.equal(grads["dres"], t["dy"].to(t["res"].dtype))
    for name, leaf in (("dx", "x"), ("dw", "w"), ("db", "b")):
        if name in grads:
            assert grads[name].dtype == t[leaf].dtype


SMALL = [(1, 1, 1), (1, 33, 17), (3, 8, 5), (16, 256, 48), (17, 40, 64), (33, 130, 31), (64, 128, 96), (65, 64, 33),
         (129, 257, 255), (300, 1001, 77), (128, 4096, 256), (70, 96, 1001)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("act", ["identity", "relu", "gelu"])
@pytest.mark.parametrize("M,K,N", SMALL)
def test_inference(M, K, N, act, dtype):
    for res, bias in ((None, True), (dtype, False), (F32, True), (BF, True)):
        t = inputs(M, K, N, dtype, res)
        with torch.no_grad():
            b = t["b"] if bias else None
            y = dense_projection(t["x"], t["w"], b, t["res"], act)
        assert y.dtype == torch.promote_types(dtype, res or dtype)
        check_forward(y, t["x"], t["w"], b, t["res"], act)


@pytest.mark.parametrize("ckpt", ["exact", "int8"])
@pytest.mark.parametrize("act", ["identity", "relu", "gelu"])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("M,K,N", SMALL)
def test_training(M, K, N, dtype, act, ckpt):
    check_training(inputs(M, K, N, dtype), act, ckpt)


@pytest.mark.parametrize("dtype,res", [(BF, BF), (BF, F32), (F32, F32), (F32, BF)])
@pytest.mark.parametrize("ckpt", ["exact", "int8"])
def test_training_with_a_residual(dtype, res, ckpt):
    check_training(inputs(100, 72, 130, dtype, res), "gelu", ckpt)


# every tile of every product: tiles past the edges, whole tiles, sums split over the reduction
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("M,K,N", [(4099, 200, 4104), (4099, 4104, 200), (200, 4099, 4104), (2048, 512, 1024),
                                   (1000, 1001, 1255), (20000, 64, 72), (130, 20000, 264)])
def test_large(M, K, N, dtype):
    check_training(inputs(M, K, N, dtype), "gelu", "int8")


@pytest.mark.parametrize("dtype", [BF, F32])
def test_strides_and_alignment(dtype):
    """Rows of wider tensors, at odd addresses, transposed, expanded: all against the contiguous copies'
    results, bit for bit."""
    M, K, N = 150, 200, 136
    gen = torch.Generator().manual_seed(3)

    def wide(r, c):
        return torch.randn(r, c, generator=gen).to(dtype).to(DEV)

    for few in (False, True):
        m = 9 if few else M
        X, W, R = wide(m, K + 40), wide(N, K + 40), wide(m, N + 9)
        b = wide(1, N + 3)[0]
        for o in (0, 1, 8):
            x, w, r, bias = X[:, o:o + K], W[:, o:o + K], R[:, o:o + N], b[min(o, 3):min(o, 3) + N]
            want = dense_projection(x.contiguous(), w.contiguous(), bias.clone(), r.contiguous(), "gelu")
            assert torch.equal(dense_projection(x, w, bias, r, "gelu"), want)
            lv = [v.detach().requires_grad_(True) for v in (x, w, bias, r)]
            lc = [v.detach().clone(memory_format=torch.contiguous_format).requires_grad_(True) for v in (x, w, bias, r)]
            dy = wide(m, N + 8)[:, o:o + N]
            for ga, gb in zip(torch.autograd.grad(dense_projection(*lv, "gelu", "int8"), lv, dy),
                              torch.autograd.grad(dense_projection(*lc, "gelu", "int8"), lc, dy.contiguous())):
                assert torch.equal(ga, gb)
        xt, wt = wide(K, m).t(), wide(K, N).t()
        assert torch.equal(dense_projection(xt, wt), dense_projection(xt.contiguous(), wt.contiguous()))
        one = wide(1, N)
        x, w = X[:, :K], W[:, :K]
        assert torch.equal(dense_projection(x, w, None, one.expand(m, N)),
                           dense_projection(x, w, None, one.expand(m, N).contiguous()))
        rows = wide(1, K).expand(m, K)
        assert torch.equal(dense_projection(rows, w), dense_projection(rows.contiguous(), w))
        # gradients that arrive expanded (sum) and transposed
        xa = x.detach().requires_grad_(True)
        y = dense_projection(xa, w, None, None, "relu")
        g1, = torch.autograd.grad(y.sum(), xa, retain_graph=True)
        g2, = torch.autograd.grad(y, xa, torch.ones_like(y))
        assert torch.equal(g1, g2)


def test_leading_dimensions_and_empty_batches():
    t = inputs(24, 40, 56, BF, BF)
    flat = dense_projection(t["x"], t["w"], t["b"], t["res"], "gelu")
    y = dense_projection(t["x"].view(2, 3, 4, 40), t["w"], t["b"], t["res"].view(2, 3, 4, 56), "gelu")
    assert y.shape == (2, 3, 4, 56) and torch.equal(y.view(24, 56), flat)
    assert torch.equal(dense_projection(t["x"][0], t["w"], t["b"], t["res"][0], "gelu"), flat[0])
    for ckpt in ("exact", "int8"):
        x = t["x"][:0].detach().requires_grad_(True)
        w, b = t["w"].detach().requires_grad_(True), t["b"].detach().requires_grad_(True)
        y = dense_projection(x, w, b, None, "gelu", ckpt)
        assert y.shape == (0, 56)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
        assert dx.shape == (0, 40) and not bool(dw.any()) and not bool(db.any()) and dw.shape == w.shape


def test_only_the_gradients_that_are_asked_for():
    t = inputs(90, 64, 72, BF, BF)
    full = run_training(t, "gelu", "exact")[1]
    for asked in (("x",), ("w",), ("b",), ("res",), ("x", "b"), ("w", "b")):
        leaves = {k: t[k].detach().requires_grad_(k in asked) for k in ("x", "w", "b", "res")}
        y = dense_projection(leaves["x"], leaves["w"], leaves["b"], leaves["res"], "gelu")
        y.backward(t["dy"])
        for k, v in leaves.items():
            assert (v.grad is not None) == (k in asked)
            if k in asked:
                assert torch.equal(v.grad, full["d" + k]), k


def test_one_tensor_in_two_places():
    """x that is the residual too, and a weight used twice: gradients are sums."""
    t = inputs(80, 64, 64, F32)
    x, w = t["x"].detach().requires_grad_(True), t["w"].detach().requires_grad_(True)
    y = dense_projection(x, w, None, x, "gelu")
    y = dense_projection(y, w, None, y, "gelu")
    gx, gw = torch.autograd.grad(y, (x, w), t["dy"])
    x6, w6 = t["x"].double().requires_grad_(True), t["w"].double().requires_grad_(True)
    h = act64(x6 @ w6.t(), "gelu") + x6
    h = act64(h @ w6.t(), "gelu") + h
    ex, ew = torch.autograd.grad(h, (x6, w6), t["dy"].double())
    # two products deep: relative to the gradients' size, 64 products each at 2^-24
    for g, e in ((gx, ex), (gw, ew)):
        assert float((g.double() - e).norm() / e.norm()) < 64 * 4 * U


def test_gradients_against_differences():
    """The backward's gradients along a direction against central differences of the forward in fp32.  Along a
    direction that moves z by s dz, the difference over 2 h is off from the slope by at most h^2 / 6 times the sum
    of |dy| |g| |dz|^3, g = phi(z) (z^3 - 4 z) gelu's third derivative, below 0.78 everywhere, and by y's rounding
    over h."""
    t = inputs(66, 48, 40, F32, F32)
    for act in ("gelu", "identity"):
        leaves = [t[k].detach().requires_grad_(True) for k in ("x", "w", "b", "res")]
        y = dense_projection(*leaves, act)
        grads = torch.autograd.grad(y, leaves, t["dy"])
        gen = torch.Generator().manual_seed(5)
        for i, (v, g) in enumerate(zip(leaves, grads)):
            d = torch.randn(v.shape, generator=gen).to(DEV)
            h = 2.0 ** -7

            def f(s):
                args = [a.detach() for a in leaves]
                args[i] = args[i] + s * h * d
                return (dense_projection(*args, act).double() * t["dy"].double()).sum()

            num, ana = (f(1) - f(-1)) / (2 * h), (g.double() * d.double()).sum()
            dz = {0: lambda: d @ t["w"].t(), 1: lambda: t["x"] @ d.t(), 2: lambda: d.expand(66, 40),
                  3: lambda: torch.zeros(66, 40, device=DEV)}[i]().double()
            third = 0.78 if act == "gelu" else 0.0
            # rounding of y: 2^-24 each of ~50 products deep, at random over the outputs
            scale = (float(t["dy"].double().norm()) * 50 * U * 3 / h
                     + h * h / 6 * third * float((t["dy"].double().abs() * dz.abs() ** 3).sum()))
            assert abs(float(num - ana)) < scale, (act, i, float(num), float(ana), scale)


def test_main_grad_and_the_optimizer():
    """fp32 main_grad buffers take both backward passes' sums; FusedAdamW then steps bf16 parameters."""
    for bias in (True, False):
        lay = DenseProjection(96, 80, "gelu", bias=bias, dtype=BF, activation_checkpoint="int8", device=DEV, seed=1,
                              bias_std=0.5)
        x, dy = torch.randn(130, 96, device=DEV).bfloat16(), torch.randn(130, 80, device=DEV).bfloat16()
        lay(x).backward(dy)
        auto = [p.grad.clone() for p in lay.parameters()]
        lay.zero_grad(set_to_none=True)
        lay.enable_main_grad()
        lay(x).backward(dy)
        once = [p.main_grad.clone() for p in lay.parameters()]
        assert all(p.grad is None for p in lay.parameters())
        for a, o in zip(auto, once):
            assert torch.equal(a, o.bfloat16())  # the same sums, unrounded
        lay(x).backward(dy)
        for o, p in zip(once, lay.parameters()):
            assert torch.equal(p.main_grad, o + o)
        before = [p.detach().clone() for p in lay.parameters()]
        FusedAdamW(lay.parameters(), lr=1e-2, stochastic_rounding=False).step()
        for p, was in zip(lay.parameters(), before):
            assert not bool(p.main_grad.any()) and not torch.equal(p, was)
        lay.zero_main_grad()


def test_repeats_have_the_same_bits():
    t = inputs(700, 520, 392, BF, BF)
    first = run_training(t, "gelu", "int8")
    again = run_training(t, "gelu", "int8")
    assert torch.equal(first[0], again[0])
    for k in first[1]:
        assert torch.equal(first[1][k], again[1][k])


def test_infinities_and_nan():
    """They reach the outputs of their own row (forward), and their own rows and columns (backward), no others."""
    M, K, N = 200, 136, 152
    for few in (False, True):
        m = 20 if few else M
        t = inputs(m, K, N, BF)
        t["x"][3, 5], t["x"][11, 135] = float("nan"), float("inf")
        y = dense_projection(t["x"], t["w"], t["b"], None, "gelu")
        clean = torch.ones(m, dtype=torch.bool, device=DEV)
        clean[3] = clean[11] = False
        assert bool(y[clean].isfinite().all()) and not bool(y[3].isfinite().any())
    t["dy"][7, 9] = float("nan")
    for ckpt, cols in (("exact", [5, 135]), ("int8", list(range(32)) + list(range(128, 136)))):
        _, g, _ = run_training(t, "identity", ckpt)
        dx = torch.ones(m, dtype=torch.bool, device=DEV)
        dx[7] = False
        assert bool(g["dx"][dx].isfinite().all()) and bool(g["dx"][7].isnan().all())
        dw = torch.ones(N, K, dtype=torch.bool, device=DEV)
        dw[9] = False
        dw[:, cols] = False
        assert bool(g["dw"][dw].isfinite().all())
        assert bool(g["db"][torch.arange(N, device=DEV) != 9].isfinite().all()) and bool(g["db"][9].isnan())


def test_another_stream_and_two_at_once():
    t = inputs(600, 264, 520, BF)
    want = dense_projection(t["x"], t["w"], t["b"], None, "gelu")
    grads = run_training(t, "gelu", "int8")[1]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = []
    for s in streams:
        with torch.cuda.stream(s):
            outs.append((dense_projection(t["x"], t["w"], t["b"], None, "gelu"), run_training(t, "gelu", "int8")[1]))
    torch.cuda.synchronize()
    for y, g in outs:
        assert torch.equal(y, want)
        for k in grads:
            assert torch.equal(g[k], grads[k])


@pytest.mark.parametrize("M", [1, 40, 300])
def test_captured_and_replayed(M):
    """Forward and backward in one graph, replayed with new inputs and eager work between the replays."""
    t = inputs(M, 264, 136, BF, BF)
    x, w, b, res, dy = (t[k] for k in ("x", "w", "b", "res", "dy"))

    def step():
        leaves = [v.detach().requires_grad_(True) for v in (x, w, b, res)]
        y = dense_projection(*leaves, "gelu", "int8")
        with torch.no_grad():
            served = dense_projection(x, w, b, res, "gelu")
        return [y.detach(), served, *torch.autograd.grad(y, leaves, dy)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for seed in range(3):
        fresh = inputs(M, 264, 136, BF, BF, seed=100 + seed)
        for k, v in (("x", x), ("w", w), ("b", b), ("res", res), ("dy", dy)):
            v.copy_(fresh[k])
        g.replay()
        eager = step()
        torch.cuda.synchronize()
        for a, e in zip(out, eager):
            assert torch.equal(a, e)


def test_refusals_on_the_gpu():
    t = inputs(8, 16, 24, BF)
    x, w = t["x"], t["w"].detach().requires_grad_(True)
    with pytest.raises(ValueError, match="weight on cpu"):
        dense_projection(x, t["w"].cpu())
    y = dense_projection(x, w, None, None, "gelu")
    with torch.no_grad():
        w.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward(t["dy"])
    xa = x.detach().requires_grad_(True)
    g, = torch.autograd.grad(dense_projection(xa, t["w"], None, None, "gelu"), xa, t["dy"].requires_grad_(True),
                             create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()  # no second derivatives
    w2 = t["w"].detach().requires_grad_(True)
    w2.main_grad = torch.zeros(24, 16, device=DEV, dtype=BF)
    with pytest.raises(ValueError, match="main_grad"):
        dense_projection(x, w2).backward(t["dy"])


@pytest.mark.parametrize("ckpt", ["exact", "int8"])
def test_gelu_over_the_whole_line(ckpt):
    """gelu and its derivative by themselves: a product with one weight of 1 hands every fp32 z through (exactly, 1 z
    has one term), from subnormals to the largest numbers, infinities and NaN."""
    f = torch.finfo(F32)
    z = torch.cat([torch.linspace(-15, 15, 200001), torch.tensor([0.0, -0.0, f.tiny, -f.tiny, 1e-40, 7.99, 8.01, -8.01, 6.49, 6.51,
                   -6.51, 40.0, -40.0, 1e4, -1e4, 1e19, -1e19, f.max, -f.max, float("inf"), float("-inf"), float("nan")])])
    z = z.to(DEV).reshape(-1, 1).requires_grad_(True)
    one = torch.ones(1, 1, device=DEV)
    y = dense_projection(z, one, None, None, "gelu", ckpt)
    served = dense_projection(z.detach()[:50], one, None, None, "gelu")
    assert torch.equal(served, y.detach()[:50])
    z6 = z.detach().double()
    want = torch.where(z6 == float("-inf"), 0.0, act64(z6, "gelu"))
    fine = ~want.isnan()
    assert bool(want[:-1].isnan().logical_not().all()) and bool(y[-1].isnan())
    # the last place of z (z - a Q(a) is rounded there) and 1e-7 of the polynomial
    err = (y.detach().double() - want).abs()[fine & want.isfinite()]
    assert bool((err <= 2 * U * z6.abs()[fine & want.isfinite()] + 1e-7).all())
    assert float(y.detach()[-3]) == float("inf")
    g, = torch.autograd.grad(y, z, torch.ones_like(y))
    if ckpt == "exact":
        w = torch.where(z6.abs() > 1e3, (z6 > 0).double(), dact64(z6, "gelu"))
        assert bool(((g.double() - w).abs()[:-1] <= 4e-7).all()) and bool(g[-1].isnan())
    else:
        assert bool(g[-3:].isnan().all()) and bool(g[:-3].isfinite().all())


def test_past_32_bits():
    """Rows whose elements and bytes are past 2^31 and 2^32 of x, y, z and dy.  dy is zero but on those rows, and sums
    with zeros are exact, so the gradients' bounds are those of the rows alone."""
    M, K, N = 2 ** 21 + 3, 1032, 2056
    x = torch.randn(M, K, device=DEV, dtype=BF)
    t = inputs(1, K, N, BF)
    rows = torch.tensor(sorted({0, 1, 255, 256, M - 1, M - 4, *(e // n + d for e in (2 ** 30, 2 ** 31, 2 ** 32) for n in (K, N)
                                                                for d in (-1, 0, 1) if e // n + d < M)}), device=DEV)
    dy = torch.zeros(M, N, device=DEV, dtype=BF)
    dy[rows] = torch.randn(len(rows), N, device=DEV).to(BF)
    leaves = [x.requires_grad_(True), t["w"].requires_grad_(True), t["b"].requires_grad_(True)]
    y = dense_projection(*leaves, None, "gelu", "int8")
    xq, xe, z, ze = (y.grad_fn.saved_tensors[i] for i in (1, 2, 5, 6))
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    x, w, b, y = x.detach(), t["w"].detach(), t["b"].detach(), y.detach()
    check_forward(y[rows], x[rows], w, b, None, "gelu")
    be = backend_for(y.device)
    kept = [be.unpack8(q[rows], e[rows], n, F32) for q, e, n in ((xq, xe, K), (z, ze, N))]
    assert torch.equal(kept[0], pack_activation(x[rows]).unpack(F32))
    sub = dict(x=x[rows], w=w, b=b, dy=dy[rows])
    check_gradients(dict(dx=dx[rows], dw=dw, db=db), sub, "gelu", kept[1].double(), kept[0], None)
    others = torch.ones(M, dtype=torch.bool, device=DEV)
    others[rows] = False
    assert not bool(dx[others].any())


# Sizes whose forward product takes each tile, whole and with its reduction split (the rest of them are in the tests above);
# dX and dW take it with the sizes in turn.
TILES = [
    (BF, "256 x 256 split", 8200, 8200, 1001), (BF, "256 x 128", 4104, 520, 1001), (BF, "256 x 128 split", 8200, 3001, 130),
    (BF, "128 x 128", 1001, 100, 4104), (BF, "128 x 128 split", 777, 8200, 3001), (BF, "deep", 8200, 1001, 130),
    (BF, "deep split", 3001, 8200, 257),
    (F32, "128 x 128", 1001, 100, 4104), (F32, "128 x 128 split", 8200, 1001, 130), (F32, "deep", 2500, 130, 777),
    (F32, "deep split", 4104, 777, 130),
]


@pytest.mark.parametrize("turn", ["forward", "dx", "dw"])
@pytest.mark.parametrize("dtype,tile,M,K,N", TILES, ids=[f"{str(t[0])[6:]} {t[1]}" for t in TILES])
def test_every_tile_of_every_product(dtype, tile, M, K, N, turn):
    """The products are M x N over K, M x K over N and N x K over M."""
    size = {"forward": (M, K, N), "dx": (M, N, K), "dw": (K, N, M)}[turn]
    check_training(inputs(*size, dtype), "gelu", "int8")


@pytest.mark.parametrize("asked", ["w", "b", "wb", "xwb"])
def test_computed_parameters(asked):
    """bf16 parameters cast from fp32 ones: the gradients of the cast ones, cast; the bias may change before the backward."""
    t = inputs(70, 48, 40, BF)
    leaves = {k: t[k].float().requires_grad_(k in asked) for k in "xwb"}
    cast = {k: v.bfloat16() for k, v in leaves.items()}
    y = dense_projection(cast["x"], cast["w"], cast["b"], None, "gelu")
    with torch.no_grad():
        cast["b"].add_(1)
    got = torch.autograd.grad(y, [leaves[k] for k in asked], t["dy"])
    want = run_training(t, "gelu", "exact")[1]
    for k, g in zip(asked, got):
        assert g.dtype == F32 and torch.equal(g, want["d" + k].float())


def test_gelu_in_the_negative_tail():
    """Relative to gelu, down to z = -4: the fit's 2e-5, and the last places of a log2 of magnitude 15 (2e-6)."""
    z = torch.linspace(-4, -1e-3, 100001).to(DEV).reshape(-1, 1)
    y = dense_projection(z, torch.ones(1, 1, device=DEV), None, None, "gelu")
    want = act64(z.double(), "gelu")
    assert bool(((y.double() - want).abs() <= 2.5e-5 * want.abs()).all())
    below = torch.tensor([[-9.0], [-1e4], [float("-inf")]], device=DEV)
    y = dense_projection(below, torch.ones(1, 1, device=DEV), None, None, "gelu")
    assert bool((y.abs() < 1e-14).all())
