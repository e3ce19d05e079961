"""Cross entropy of a dense head on the GPU against the definition in float64, element by element within bounds of its
roundings and as a whole within what roundings that are independent of each other leave."""
import math

import pytest
import torch

from conftest import gpu_available

from granulelayer_amd import DenseCrossEntropy, dense_cross_entropy

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a ROCm GPU")]
DEV = "cuda"
E = 2.0 ** -24  # half a last place of fp32
BF, F = torch.bfloat16, torch.float32
HALF = {BF: 2.0 ** -8, F: E}
IGNORED = -100


def inputs(M, K, N, dtype, bias=True, ignored=0.3, seed=0, scale=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed + M + K + N)

    def normal(*s):
        return torch.randn(*s, generator=g, device=DEV)

    t = dict(x=normal(M, K).to(dtype), w=(scale / math.sqrt(K) * normal(N, K)).to(dtype))
    t["b"] = normal(N).to(dtype) if bias else None
    target = torch.randint(0, N, (M,), generator=g, device=DEV)
    t["target"] = torch.where(torch.rand(M, generator=g, device=DEV) < ignored, IGNORED, target)
    t["g"] = torch.rand(M, generator=g, device=DEV) + 0.1
    return t


def definition(t, reduction, g):
    """name -> (value, bound of the errors of fp32 arithmetic, dz rounded to the operands' type) in float64."""
    x, w = t["x"].detach().double(), t["w"].detach().double()
    b = 0 if t["b"] is None else t["b"].detach().double()
    target = t["target"]
    M, K = x.shape
    N = w.shape[0]
    on = target != IGNORED
    at = torch.where(on, target, 0)[:, None]
    z = x @ w.t() + b
    d_z = (K + 3) * E * (x.abs() @ w.abs().t() + (0 if t["b"] is None else b.abs()))
    lse = torch.logsumexp(z, 1)
    # sums of exponentials: errors of their logits (no more than the largest) and two of each exponential; up to 70
    # additions in a row and the tiles' rescalings; the log and the statistics' own places
    d_lse = d_z.amax(1) + 4 * E * z.abs().amax(1) + 100 * E + 2 * E * lse.abs()
    loss = torch.where(on, lse - z.gather(1, at)[:, 0], 0.0)
    d_loss = torch.where(on, d_lse + (d_z + 4 * E * z.abs()).gather(1, at)[:, 0] + 3 * E * (lse.abs() + z.abs().amax(1)), 0.0)
    n = max(1, int(on.sum()))
    c = {"none": lambda: g.double(), "sum": lambda: g.double(), "mean": lambda: g.double() / n}[reduction]().expand(M)
    c = torch.where(on, c, 0.0)[:, None]
    p = torch.exp(z - lse[:, None])
    # an exponential below the least normal number, 2^-126, is 0
    d_p = p * (d_z + d_lse[:, None] + 4 * E * (z.abs() + lse.abs()[:, None]) + 3 * E) + 2.0 ** -126
    if x.shape[1] >= 512 and t["x"].dtype == BF:
        # exponentials are kept in 16 bits: 10 of them the mantissa's, 6 the exponent's, down to 2^-63 of the largest of 64
        d_p = d_p + 2.0 ** -11 * p + 2.0 ** -62 * p.amax(1, keepdim=True)
    dz = c * p.scatter_add(1, at, -torch.ones_like(at, dtype=torch.float64))
    d_dz = c.abs() * d_p + 3 * E * dz.abs()
    d_dzr = d_dz + HALF[t["x"].dtype] * (dz.abs() + d_dz)
    out = {"dx": (dz @ w, d_dzr @ w.abs() + (N + 10) * E * (dz.abs() @ w.abs())),
           "dw": (dz.t() @ x, d_dzr.t() @ x.abs() + (M + 10) * E * (dz.abs().t() @ x.abs())),
           "db": (dz.sum(0), d_dz.sum(0) + (M + 10) * E * dz.abs().sum(0))}
    if reduction == "none":
        out["loss"] = loss, d_loss
    else:
        k = n if reduction == "mean" else 1
        out["loss"] = loss.sum() / k, d_loss.sum() / k + 2 * E * loss.sum() / k
    return out


def check(got, want, name, whole=True):
    value, bound = want[name]
    got = got.detach()
    tol = bound + HALF[got.dtype] * (value.abs() + bound) + 1e-38
    off = (got.double() - value).abs()
    worst = float((off / tol).max()) if off.numel() else 0.0
    assert worst <= 1, f"{name}: {worst:.2f} of the bound"
    if whole and value.dim() and float(value.norm()):
        # independent roundings: of dz and of the result, 2^-8 each at most and less than half of that on average; fp32
        # sums' and the statistics' errors stay below 1e-5 of it
        assert float(off.norm() / value.norm()) <= (2.0 ** -8 if got.dtype == BF else 1e-5), name


def run(t, reduction, budget=None, **kw):
    leaves = {k: t[k].detach().requires_grad_(True) for k in "xwb" if t[k] is not None}
    loss = dense_cross_entropy(leaves["x"], leaves["w"], t["target"], leaves.get("b"), reduction, IGNORED, budget)
    g = t["g"] if reduction == "none" else torch.tensor(1.7, device=DEV)
    grads = torch.autograd.grad(loss, list(leaves.values()), g)
    return g, dict({"d" + k: v for k, v in zip(leaves, grads)}, loss=loss)


def compare(t, reduction, budget=None):
    g, got = run(t, reduction, budget)
    want = definition(t, reduction, g)
    for name, v in got.items():
        if name != "loss":
            leaf = t[name[1]]
            assert v.dtype == leaf.dtype and v.shape == leaf.shape
        check(v, want, name)
    assert got["loss"].dtype == F
    with torch.no_grad():
        assert torch.equal(dense_cross_entropy(t["x"], t["w"], t["target"], t["b"], reduction), got["loss"])
    return got


SHAPES = [(1, 16, 2), (1, 1, 1), (3, 7, 5), (16, 64, 130), (64, 1024, 1000), (1, 130, 5000), (128, 100, 257), (129, 100, 300), (256, 100, 257), (257, 100, 300),
          (300, 128, 2049), (777, 1001, 555), (1000, 72, 4097), (2, 8192, 33), (600, 33, 1), (4100, 40, 9)]


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_loss_and_gradients(M, K, N, dtype, reduction):
    compare(inputs(M, K, N, dtype, bias=(M + N) % 2 == 0), reduction)


# sizes whose products take each tile, whole and with its reduction split
TILES = ([(BF, *s) for s in ((300, 40, 130), (2100, 40, 2500), (8200, 40, 8200), (777, 2500, 2500), (4104, 2500, 1255),
                             (520, 8200, 777), (1300, 130, 33000), (16390, 130, 8200), (16390, 130, 130),
                             (4104, 130, 16500), (520, 4104, 8200))]
         + [(F, *s) for s in ((300, 40, 130), (520, 40, 8200), (520, 130, 16500), (300, 8200, 257), (16390, 40, 1255),
                              (16390, 130, 130), (777, 40, 16500))])


@pytest.mark.parametrize("dtype,M,K,N", TILES)
def test_every_tile(dtype, M, K, N):
    compare(inputs(M, K, N, dtype, ignored=0.1), "mean")


@pytest.mark.parametrize("K", [130, 520])
@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("M", [40, 700])
def test_pieces(K, dtype, M):
    """1001 classes in pieces of 256 and of 512 and whole."""
    t = inputs(M, K, 1001, dtype)
    es = 2 if dtype == BF else 4
    whole = compare(t, "mean")
    for columns in (1, 300, 512, 1001):
        got = compare(t, "mean", budget=M * es * columns)
        # a piece's columns of dw and db do not depend on the others but for how their sums over the rows are split
        assert torch.equal(got["loss"], whole["loss"])


@pytest.mark.parametrize("K", [64, 520])
@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("M", [1, 256, 257, 5000])
@pytest.mark.parametrize("kept", ["none", "first", "last", "one in the middle"])
def test_ignored_rows(K, dtype, M, kept):
    t = inputs(M, K, 300, dtype, ignored=0.0)
    on = {"none": [], "first": [0], "last": [M - 1], "one in the middle": [M // 2]}[kept]
    target = torch.full_like(t["target"], IGNORED)
    target[on] = t["target"][on]
    t["target"] = target
    got = compare(t, "mean")
    if not on:
        assert got["loss"] == 0 and not any(got["d" + k].any() for k in "xwb")
    off = torch.ones(M, dtype=torch.bool, device=DEV)
    off[on] = False
    assert not got["dx"][off].any()
    each = run(t, "none")[1]["loss"]
    assert not each[off].any()


@pytest.mark.parametrize("K", [200, 520])
@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("M", [100, 900])
def test_what_ignored_rows_hold_does_not_matter(K, dtype, M):
    t = inputs(M, K, 500, dtype, ignored=0.4)
    off = t["target"] == IGNORED
    clean = run(t, "mean")[1]
    for value in (float("nan"), float("inf"), torch.finfo(dtype).max):
        dirty = dict(t, x=t["x"].clone())
        dirty["x"][off] = value
        got = run(dirty, "mean")[1]
        for k, v in clean.items():
            assert torch.equal(got[k], v), k
        assert not got["dx"][off].any()


@pytest.mark.parametrize("K", [72, 520])
@pytest.mark.parametrize("M", [60, 600])
def test_classes_that_take_no_part(K, M):
    """A bias of -inf: a padded vocabulary, whole tiles of it among them."""
    t = inputs(M, K, 700, F, ignored=0.2)
    t["b"][300:] = float("-inf")
    t["target"] = torch.where(t["target"] == IGNORED, IGNORED, t["target"] % 300)
    got = run(t, "mean")[1]
    part = dict(t, w=t["w"][:300].contiguous(), b=t["b"][:300].contiguous())
    want = definition(part, "mean", torch.tensor(1.7, device=DEV))
    check(got["loss"], want, "loss")
    check(got["dx"], want, "dx")
    check(got["dw"][:300], want, "dw")
    check(got["db"][:300], want, "db")
    assert not got["dw"][300:].any() and not got["db"][300:].any()
    t["b"].fill_(torch.finfo(F).min)  # the type's lowest everywhere: a shift of all logits, no mask
    got = run(t, "mean")[1]
    assert abs(float(got["loss"].detach()) - math.log(700)) < 1e-5 and all(torch.isfinite(v).all() for v in got.values())
    # x w is lost against it: every class has 1 / 700, so db is 1.7 / 700 - 1.7 times the class' share of the targets
    share = torch.bincount(t["target"][t["target"] != IGNORED], minlength=700) / int((t["target"] != IGNORED).sum())
    assert torch.allclose(got["db"], 1.7 * (1 / 700 - share), rtol=1e-5, atol=1e-7)


@pytest.mark.parametrize("K", [48, 520])
@pytest.mark.parametrize("M", [60, 600])
@pytest.mark.parametrize("bad", [-1, 300, 2 ** 40, -2 ** 63])
def test_targets_that_are_no_class(K, M, bad):
    t = inputs(M, K, 300, BF, ignored=0.2)
    row = int((t["target"] != IGNORED).nonzero()[1])
    clean = run(t, "none")[1]
    t["target"][row] = bad
    got = run(t, "none")[1]
    assert torch.isnan(got["loss"][row]) and torch.isnan(got["dx"][row]).all()
    others = torch.arange(M, device=DEV) != row
    assert torch.equal(got["loss"][others], clean["loss"][others]) and torch.equal(got["dx"][others], clean["dx"][others])
    assert torch.isnan(dense_cross_entropy(t["x"], t["w"], t["target"], t["b"]))


@pytest.mark.parametrize("K", [48, 520])
def test_rows_that_are_no_numbers(K):
    t = inputs(600, K, 300, F, ignored=0.0)
    clean = run(t, "none")[1]
    t["x"][7, 3], t["x"][500, 0] = float("nan"), float("inf")
    got = run(t, "none")[1]
    bad = torch.tensor([7, 500], device=DEV)
    good = torch.ones(600, dtype=torch.bool, device=DEV)
    good[bad] = False
    assert torch.isnan(got["loss"][bad]).all() and torch.isnan(got["dx"][bad]).all()
    assert torch.equal(got["loss"][good], clean["loss"][good]) and torch.equal(got["dx"][good], clean["dx"][good])


@pytest.mark.parametrize("M", [100, 700])
def test_a_class_as_the_ignored_index(M):
    t = inputs(M, 520, 300, BF, ignored=0.0)
    t["target"][::3] = 7
    other = dict(t, target=torch.where(t["target"] == 7, IGNORED, t["target"]))
    want = run(other, "mean")[1]
    leaves = [t[k].detach().requires_grad_(True) for k in "xwb"]
    loss = dense_cross_entropy(*leaves[:2], t["target"], leaves[2], ignore_index=7)
    assert torch.equal(loss, want["loss"])
    for k, v in zip("xwb", torch.autograd.grad(loss, leaves, torch.tensor(1.7, device=DEV))):
        assert torch.equal(v, want["d" + k])


def test_a_graph_of_the_backward_is_refused_where_it_is_used():
    t = inputs(300, 32, 64, F)
    x = t["x"].detach().requires_grad_(True)
    dx, = torch.autograd.grad(dense_cross_entropy(x, t["w"], t["target"], t["b"]), x, create_graph=True)
    check(dx, definition(t, "mean", torch.ones((), device=DEV)), "dx")
    with pytest.raises(RuntimeError):
        dx.sum().backward()


@pytest.mark.parametrize("dtype,K", [(F, 64), (F, 520), (BF, 520)])
def test_large_logits(dtype, K):
    """Logits of several hundreds: exponentials that overflow without the largest taken off."""
    t = inputs(500, K, 900, dtype, scale=200.0)
    got = run(t, "none")
    want = definition(t, "none", got[0])
    for name, v in got[1].items():
        check(v, want, name, whole=False)


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("M", [100, 500])
def test_strides_views_and_types(dtype, M):
    t = inputs(M, 130, 333, dtype)
    g = torch.tensor(1.7, device=DEV)
    want = definition(t, "mean", g)
    wide_x = torch.zeros(M, 150, device=DEV, dtype=dtype)
    wide_w = torch.zeros(333, 143, device=DEV, dtype=dtype)
    wide_b = torch.zeros(666, device=DEV, dtype=dtype)
    for first in (0, 1, 8):
        wide_x[:, first:first + 130] = t["x"]
        wide_w[:, first:first + 130] = t["w"]
        wide_b[::2] = t["b"]
        wide_target = torch.stack([t["target"], t["target"] + 7], 1)
        leaves = [v.detach().requires_grad_(True) for v in (wide_x[:, first:first + 130], wide_w[:, first:first + 130], wide_b[::2])]
        assert leaves[0].stride(0) == 150 and leaves[1].stride(0) == 143
        loss = dense_cross_entropy(leaves[0], leaves[1], wide_target[:, 0], leaves[2])
        check(loss, want, "loss")
        for v, name in zip(torch.autograd.grad(loss, leaves, g), ("dx", "dw", "db")):
            check(v, want, name)
    loss = dense_cross_entropy(t["x"].view(5, -1, 130), t["w"], t["target"].view(5, -1).int(), t["b"], "none")
    assert loss.shape == (5, M // 5)
    check(loss.reshape(-1), definition(t, "none", t["g"]), "loss")
    x1 = t["x"][:1]
    one = dict(t, x=x1, target=t["target"].clamp(min=0)[:1], g=t["g"][:1])
    check(dense_cross_entropy(x1[0], t["w"], one["target"][0], t["b"], "none").view(1), definition(one, "none", one["g"]), "loss")
    neg = torch._neg_view(-t["x"])
    assert torch.equal(dense_cross_entropy(neg, t["w"], t["target"], t["b"]), dense_cross_entropy(t["x"], t["w"], t["target"], t["b"]))


@pytest.mark.parametrize("K", [64, 520])
@pytest.mark.parametrize("M", [100, 500])
def test_gradients_asked_for_alone_and_upstream_strides(K, M):
    t = inputs(M, K, 222, BF)
    for names in ("x", "w", "b", "xw", "xb", "wb"):
        leaves = {k: t[k].detach().requires_grad_(k in names) for k in "xwb"}
        loss = dense_cross_entropy(leaves["x"], leaves["w"], t["target"], leaves["b"], "none")
        for g in (t["g"], torch.stack([t["g"], t["g"]], 1)[:, 0], torch._neg_view(-t["g"]), torch.full((1,), 0.5, device=DEV).expand(M)):
            want = definition(t, "none", g.resolve_neg())
            for k, v in zip(names, torch.autograd.grad(loss, [leaves[k] for k in names], g, retain_graph=True)):
                check(v, want, "d" + k)


def test_no_rows():
    t = inputs(4, 32, 50, BF)
    x = t["x"][:0].detach().requires_grad_(True)
    w, b = (t[k].detach().requires_grad_(True) for k in "wb")
    for reduction in ("mean", "sum", "none"):
        loss = dense_cross_entropy(x, w, t["target"][:0], b, reduction)
        assert loss.shape == ((0,) if reduction == "none" else ()) and not loss.any()
        grads = torch.autograd.grad(loss.sum(), (x, w, b))
        assert grads[0].shape == (0, 32) and not grads[1].any() and not grads[2].any()


def test_gradient_against_differences():
    t = inputs(300, 40, 130, F, ignored=0.2)
    g, got = run(t, "sum")
    gen = torch.Generator(device=DEV).manual_seed(5)
    step = 2.0 ** -6
    for k in "xwb":
        u = torch.randn(t[k].shape, generator=gen, device=DEV)
        u = u / u.norm()
        sides = [float(dense_cross_entropy(*(t[n] + (s * u if n == k else 0) for n in "xw"), t["target"],
                                           t["b"] + (s * u if k == "b" else 0), "none").double().sum()) for s in (step, -step)]
        slope, want = 1.7 * (sides[0] - sides[1]) / (2 * step), float((got["d" + k].double() * u.double()).sum())
        # losses of up to 10 are within 5e-6 each, 300 of them at random 1e-4, over 2 x step: 4e-3; the third derivative of a
        # unit direction is below a few times the gradient's norm, step^2 / 6 of it 1e-4
        assert abs(slope - want) < 1e-2 + 1e-3 * float(got["d" + k].norm())


@pytest.mark.parametrize("M", [100, 700])
def test_main_grad_is_added_to(M):
    lay = DenseCrossEntropy(64, 500, bias=True, device=DEV, seed=3)
    t = inputs(M, 64, 500, BF)
    lay.enable_main_grad()
    lay.weight.main_grad.fill_(2.0)
    x = t["x"].detach().requires_grad_(True)
    for _ in range(2):
        lay(x, t["target"]).backward()
    assert lay.weight.grad is None and lay.bias.grad is None
    want = definition(dict(t, w=lay.weight, b=lay.bias), "mean", torch.ones((), device=DEV))
    twice = {k: (2 * v, 2 * b + 4 * E * (2 + v.abs())) for k, (v, b) in want.items()}
    check(lay.weight.main_grad - 2.0, twice, "dw", whole=False)
    check(lay.bias.main_grad, twice, "db", whole=False)
    lay.zero_main_grad()
    assert not lay.weight.main_grad.any()


@pytest.mark.parametrize("K", [96, 520])
@pytest.mark.parametrize("M", [100, 700])
def test_a_captured_training_pass_and_another_stream(K, M):
    t = inputs(M, K, 1000, BF)
    leaves = [t[k].detach().requires_grad_(True) for k in "xwb"]
    target = t["target"].clone()

    def passes():
        loss = dense_cross_entropy(leaves[0], leaves[1], target, leaves[2], "mean", IGNORED, M * 2 * 400)
        return (loss.detach(), *torch.autograd.grad(loss, leaves))

    eager = passes()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = passes()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    del other
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = passes()
    gen = torch.Generator(device=DEV).manual_seed(1)
    for k in range(4):  # other numbers of rows that count
        new = torch.randint(0, 1000, (M,), generator=gen, device=DEV)
        target.copy_(torch.where(torch.rand(M, generator=gen, device=DEV) < 0.3 * k, IGNORED, new))
        for o in out:
            o.zero_()
        graph.replay()
        got = [o.clone() for o in out]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(passes(), got))


def test_a_second_backward_and_one_without_the_first():
    """The kept exponentials serve one backward; another of the same graph makes them again."""
    t = inputs(700, 520, 900, BF)
    leaves = [t[k].detach().requires_grad_(True) for k in "xwb"]
    want = definition(t, "mean", torch.ones((), device=DEV))
    loss = dense_cross_entropy(leaves[0], leaves[1], t["target"], leaves[2])
    for last in (False, False, True):
        for v, name in zip(torch.autograd.grad(loss, leaves, retain_graph=not last), ("dx", "dw", "db")):
            check(v, want, name)
    dense_cross_entropy(leaves[0], leaves[1], t["target"], leaves[2])  # its graph goes without a backward
    from torch.utils.checkpoint import checkpoint

    loss = checkpoint(dense_cross_entropy, leaves[0], leaves[1], t["target"], leaves[2], use_reentrant=False)
    for v, name in zip(torch.autograd.grad(loss, leaves), ("dx", "dw", "db")):
        check(v, want, name)


@pytest.mark.parametrize("reduction", ["mean", "sum"])
@pytest.mark.parametrize("K", [64, 520])
@pytest.mark.parametrize("M", [100, 700])
@pytest.mark.parametrize("upstream", [float("inf"), float("nan")])
def test_an_upstream_gradient_that_is_no_number(upstream, M, K, reduction):
    """It reaches the rows that count and no others."""
    t = inputs(M, K, 300, BF)
    off = t["target"] == IGNORED
    for target in (t["target"], torch.full_like(t["target"], IGNORED)):
        leaves = [t[k].detach().requires_grad_(True) for k in "xwb"]
        loss = dense_cross_entropy(leaves[0], leaves[1], target, leaves[2], reduction)
        dx, dw, db = torch.autograd.grad(loss, leaves, torch.full((), upstream, device=DEV))
        if target is t["target"]:
            assert not dx[off].any() and not dx[~off].isfinite().all(1).any() and not dw.isfinite().all() and not db.isfinite().all()
        else:
            assert not dx.any() and not dw.any() and not db.any()


def test_a_captured_backward_without_its_forward():
    """A graph of the backward alone is replayed as often as one likes; one forward serves all of them."""
    t = inputs(700, 520, 900, BF)
    leaves = [t[k].detach().requires_grad_(True) for k in "xwb"]
    want = definition(t, "mean", torch.ones((), device=DEV))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        loss = dense_cross_entropy(leaves[0], leaves[1], t["target"], leaves[2])
        torch.autograd.grad(loss, leaves)
        loss = dense_cross_entropy(leaves[0], leaves[1], t["target"], leaves[2])
        one = torch.ones((), device=DEV)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = torch.autograd.grad(loss, leaves, one, retain_graph=True)
    for _ in range(3):
        for o in out:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for v, name in zip(out, ("dx", "dw", "db")):
            check(v, want, name)


def test_a_capture_has_a_number():
    from granulelayer_amd.backend import backend_for

    be, dev, x = backend_for(torch.device(DEV)), torch.device(DEV), torch.zeros(4, device=DEV)
    seen = [be.capture_id(dev)]
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for g in graphs:
        with torch.cuda.graph(g):
            x.add_(1)
            seen += [be.capture_id(dev), be.capture_id(dev)]
    seen.append(be.capture_id(dev))
    assert seen[0] == seen[5] == 0 and seen[1] == seen[2] != 0 and seen[3] == seen[4] != 0 and seen[1] != seen[3]


def test_operands_may_not_change_before_the_backward():
    t = inputs(300, 32, 64, BF)
    for name in ("x", "w", "b", "target"):
        leaves = {k: t[k].clone().requires_grad_(True) for k in "xwb"}
        leaves["target"] = t["target"].clone()
        loss = dense_cross_entropy(leaves["x"], leaves["w"], leaves["target"], leaves["b"])
        with torch.no_grad():
            leaves[name].add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            loss.backward()


def test_the_same_bits_twice():
    t = inputs(3000, 200, 5000, BF)
    a, b = run(t, "mean")[1], run(t, "mean")[1]
    assert all(torch.equal(a[k], b[k]) for k in a)


def test_past_32_bits():
    """70000 rows of 32768 classes, 2.3e9 logits, in pieces and whole: every logit is 0, so dz is 1 / classes but for the
    target's."""
    M, K, N = 70_000, 8, 32768
    x = torch.zeros(M, K, device=DEV, dtype=BF)
    x[:, 0] = 1.0
    w = torch.zeros(N, K, device=DEV, dtype=BF)
    w[:, 1] = 1.0  # x has 0 there
    target = torch.zeros(M, dtype=torch.int64, device=DEV)
    target[-1] = N - 1
    for budget in (None, 16 << 30):
        xs, ws = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        loss = dense_cross_entropy(xs, ws, target, None, "sum", IGNORED, budget)
        assert abs(float(loss.detach()) / (M * 15 * math.log(2)) - 1) < 1e-6
        dx, dw = torch.autograd.grad(loss, (xs, ws))
        # sum over the classes of w[:, 1] dz: (N - 1) / N - (N - 1) / N; dz of the target rounded to bf16 is -1
        assert not dx[:, 0].any() and float(dx[:, 1].abs().max()) <= 2.0 ** -8
        assert float(dw[1, 0]) == float(torch.tensor(M / N).bfloat16()) and float(dw[N - 1, 0]) == float(torch.tensor((M - 1) / N - 1).bfloat16())
        assert not dw[:, 1:].any()


def test_kept_exponentials_past_32_bits():
    """70000 rows of 32768 classes, whose exponentials are 4.6 GB: every logit is 0 but that of each row's own class, 1."""
    M, K, N = 70_000, 512, 32768
    x = torch.zeros(M, K, device=DEV, dtype=BF)
    rows = torch.arange(M, device=DEV)
    x[rows, rows % K] = 1.0
    w = torch.zeros(N, K, device=DEV, dtype=BF)
    own = torch.arange(K, device=DEV)
    w[64 * own, own] = 1.0  # row m's own class is 64 (m % K)
    target = (64 * (rows % K) + 1) % N  # its neighbour
    target[-1] = N - 1
    xs, ws = x.requires_grad_(True), w.requires_grad_(True)
    loss = dense_cross_entropy(xs, ws, target, None, "none", IGNORED, 16 << 30)
    Z = N - 1 + math.e
    assert float((loss.detach() - math.log(Z)).abs().max()) < 1e-5
    dx, dw = torch.autograd.grad(loss, (xs, ws), torch.ones(M, device=DEV))
    # dx[m, c] = dz[m, 64 c]: e / Z at the row's own, 1 / Z elsewhere, rounded to bf16 as dz and as dx (2^-7 for both)
    for m in (0, 1, 32_767, 32_768, 65_536, M - 1):
        want = torch.full((K,), 1 / Z, device=DEV)
        want[m % K] = math.e / Z
        assert float((dx[m].float() / want - 1).abs().max()) <= 2.0 ** -7 + 1e-4
    # dw[n, c] = sum over the rows whose own is c of dz[m, n]: of the neighbour of another's class, 1 / Z each
    c = 5
    count = len(range(c, M, K))
    assert abs(float(dw[1, c]) / (count / Z) - 1) <= 2.0 ** -7 + 1e-4
    assert abs(float(dw[64 * c, c]) / (count * math.e / Z) - 1) <= 2.0 ** -7 + 1e-4
    assert abs(float(dw[64 * c + 1, c]) / (count * (1 / Z - 1)) - 1) <= 2.0 ** -7 + 1e-4
    # rows the last of all: (M - 1) % K's column holds its target's -1
    last = (M - 1) % K
    assert abs(float(dw[N - 1, last]) / (len(range(last, M, K)) / Z - 1) - 1) <= 2.0 ** -7 + 1e-4
