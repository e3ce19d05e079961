"""Activations in 8 bits on the GPU, bit for bit against the definition in float64: the smallest power of
two, from 2^-126 to 2^121, in which a block's values round to integers of magnitude 127 or less (values next to
the largest number are cut to 127 of the largest step)."""
import numpy as np
import pytest
import torch

from granulelayer_amd import PackedActivation, pack_activation
from granulelayer_amd.backend import backend_for

pytestmark = pytest.mark.gpu
DEV = "cuda"


def want8(x):
    """The values of x's 8-bit form, in float64 (numpy; blocks of 32 along the rows)."""
    x = np.asarray(x, np.float64)
    out = np.empty_like(x)
    for c in range(0, x.shape[1], 32):
        b = x[:, c:c + 32]
        top = np.abs(b).max(1, keepdims=True)
        with np.errstate(all="ignore"):
            p = np.floor(np.log2(np.where(np.isfinite(top) & (top > 0), top, 1.0))) - 6
            p = np.where(top == 0, -126, p)
            p = np.clip(np.where(np.abs(top) / 2.0 ** p >= 127.5, p + 1, p), -126, 121)
            q = np.clip(np.rint(b / 2.0 ** p), -127, 127) * 2.0 ** p
        out[:, c:c + 32] = np.where(np.isfinite(top), q, np.nan)
    return out


def check(x):
    p = pack_activation(x)
    rows, nb = x.numel() // x.shape[-1], -(-x.shape[-1] // 32)
    assert p.codes.shape == (rows, nb * 32) and p.exponents.shape == (rows, nb)
    assert p.nbytes == rows * nb * 33
    want = want8(x.detach().float().reshape(rows, -1).cpu().numpy())
    for dt in (torch.float32, torch.bfloat16):
        got = p.unpack(dt)
        assert got.dtype == dt and got.shape == x.shape and got.is_contiguous()
        np.testing.assert_array_equal(got.double().reshape(rows, -1).cpu().numpy(), want)
    assert p.unpack().dtype == x.dtype
    assert not bool(p.codes.reshape(rows, nb * 32)[:, x.shape[-1]:].any())  # zeros behind the features
    return p


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 31), (1, 32), (3, 33), (5, 64), (2, 97), (7, 255), (4, 256), (63, 513),
                                       (1, 16385), (300, 1001), (2, 2080), (1030, 8)])
def test_values(dtype, rows, cols):
    gen = torch.Generator().manual_seed(rows * 131 + cols)
    x = torch.randn(rows, cols, generator=gen) * torch.exp(2 * torch.randn(rows, cols, generator=gen))
    check(x.to(dtype).to(DEV))


def test_borders():
    """Maxima on both sides of every border of the exponent's rule, ties of the rounding, subnormals, the
    largest numbers, zero blocks, infinities and NaN."""
    f = torch.finfo(torch.float32)
    one = []
    for top in (1.0, 127.49999, 127.5, 127.50001, 127.99999, 128.0, 63.999996, 64.0, f.max, f.tiny, f.tiny / 2 ** 20,
                2.0 ** -149, 2.0 ** -120, 2.0 ** -119, 2.0 ** -120 * 127.5 / 64):
        b = torch.linspace(-1, 1, 32) * top
        b[3], b[7], b[11] = top, top / 2, -top
        one.append(b)
    one.append(torch.arange(32).float() + 0.5)                          # ties, step 1/2
    one.append(torch.cat([torch.arange(31).float() * 2 + 0.5, torch.tensor([100.0])]))  # ties at step 1
    one.append(torch.zeros(32))
    one.append(-torch.zeros(32))
    for bad in (float("inf"), float("-inf"), float("nan")):
        b = torch.randn(32)
        b[5] = bad
        one.append(b)
    x = torch.cat(one)
    check(x.reshape(1, -1).to(DEV))
    check(torch.stack(one).to(DEV))
    check(torch.stack(one).to(DEV).bfloat16())


def test_a_second_time_changes_nothing():
    x = torch.randn(50, 333, device=DEV)
    v = pack_activation(x).unpack()
    assert torch.equal(pack_activation(v).unpack(), v)
    assert torch.equal(pack_activation(v.bfloat16()).unpack(torch.float32), v)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_shapes(dtype):
    base = torch.randn(40, 301, device=DEV).to(dtype)
    for x in (base[:, 1:], base[:, 3:260], base[::2, 2:], base.t(), base[:, ::2], base[5:6], base[:, :1],
              base[0].expand(6, 301), base[:, 7], base.reshape(4, 10, 301)[:, 1:], torch.imag(torch.randn(4, 9, device=DEV,
              dtype=torch.complex64).conj()).to(dtype)):
        check(x)
    assert pack_activation(base[:0]).unpack().shape == (0, 301)
    x = base.clone().requires_grad_(True)
    assert not pack_activation(x).unpack().requires_grad


def test_past_32_bits_of_elements():
    """Rows past 2^32 elements: the first and last rows against the definition."""
    cols = 4096
    rows = 2 ** 32 // cols + 5
    x = torch.zeros(rows, cols, device=DEV, dtype=torch.bfloat16)
    for r in (0, 1, rows - 6, rows - 1):
        x[r] = torch.randn(cols, device=DEV).bfloat16()
    v = pack_activation(x).unpack()
    for r in (0, 1, rows - 6, rows - 5, rows - 1):
        np.testing.assert_array_equal(v[r:r + 1].double().cpu().numpy(), want8(x[r:r + 1].double().cpu().numpy()))


def test_on_another_stream_and_replayed():
    s = torch.cuda.Stream()
    x = torch.randn(70, 100, device=DEV)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        p = pack_activation(x)
        v = p.unpack()
    s.synchronize()
    np.testing.assert_array_equal(v.double().cpu().numpy(), want8(x.cpu().numpy()))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        w = pack_activation(x).unpack()
    for seed in range(3):
        x.copy_(torch.randn(70, 100, generator=torch.Generator().manual_seed(seed)))
        g.replay()
        eager = pack_activation(x).unpack()
        torch.cuda.synchronize()
        assert torch.equal(w, eager)


def test_refusals_of_codes():
    p = pack_activation(torch.randn(4, 40, device=DEV))
    with pytest.raises(TypeError):
        p.unpack(torch.float16)
    be = backend_for(torch.device(DEV))
    with pytest.raises(ValueError):
        be.unpack8(p.codes[:, :32], p.exponents, 40, torch.float32)
    with pytest.raises(ValueError):
        be.unpack8(p.codes, p.exponents[:3], 40, torch.float32)
    with pytest.raises(ValueError):
        PackedActivation(p.codes, p.exponents, (4, 100), torch.float32).unpack()


# ---- the sparse layers' input in 8 bits -----------------------------------------------------------------
def sparse_layer(kind, ckpt):
    import granulelayer_amd as G

    if kind == "cover":
        gen = torch.Generator().manual_seed(2)
        L = G.cover_topk16.EnvelopeLayout(256, 4096, 8, 64, 256)
        w = torch.randn(L.weight_shape, generator=gen) / 8
        b = torch.randn(L.bias_shape, generator=gen)
        cand = torch.stack([torch.randperm(256, generator=gen)[:64].sort().values for _ in range(int(np.prod(L.index_shape[:2])))])
        return G.CoverTopK16Layer.from_envelope(w.to(DEV), b.to(DEV), cand.view(L.index_shape).to(DEV), input_dim=256,
                                                hidden_dim=4096, output_dim=8, device=DEV, activation_checkpoint=ckpt)
    pooling, policy = {
        "mean": ("mean", "auto"), "gelu": (dict(type="sum", activation="gelu"), "auto"),
        "bf16": ("mean", "auto"),
        "max": ("max", "recompute_stats"), "topk": (dict(type="topk_mean", k=4), "recompute_stats"),
        "lme": (dict(type="logmeanexp", activation="gelu"), "recompute_stats"),
        "two": (dict(levels=[dict(type="mean", neurons_per_shard=128), dict(type="logmeanexp")],
                     level1_checkpoint="recompute"), "auto"),
    }[kind]
    return G.SparsePoolingLayer(250, 6144, 12, shared_neurons=None, pooling=pooling, checkpoint_policy=policy,
                                dtype=torch.bfloat16 if kind == "bf16" else torch.float32, device=DEV, seed=4, bias_std=0.3,
                                activation_checkpoint=ckpt)


@pytest.mark.parametrize("kind", ["mean", "gelu", "bf16", "max", "topk", "lme", "two", "cover"])
def test_sparse_layers_backward_at_the_kept_input(kind):
    """The output has the exact input's bits; the gradients have the bits of an exact layer whose input are the
    kept values (where nothing but the input is kept)."""
    exact, eight = sparse_layer(kind, "exact"), sparse_layer(kind, "int8")
    D = 256 if kind == "cover" else 250
    x = torch.randn(3, 17, D, generator=torch.Generator().manual_seed(1)).to(DEV)
    if kind == "bf16":
        x = x.bfloat16()
    xe = x.clone().requires_grad_(True)
    xk = pack_activation(x).unpack().requires_grad_(True)
    y = eight(xe)
    assert eight.last_info["input_checkpoint_bytes"] == 51 * 8 * 33
    assert torch.equal(y, exact(x)) and exact.last_info["input_checkpoint_bytes"] == x.numel() * x.element_size()
    dy = torch.randn(y.shape, generator=torch.Generator().manual_seed(6)).to(DEV)
    got = torch.autograd.grad(y, [xe, eight.weight, eight.bias], dy)
    want = torch.autograd.grad(exact(xk), [xk, exact.weight, exact.bias], dy)
    for g, w in zip(got, want):
        assert g.dtype == w.dtype and torch.equal(g, w)


def test_sparse_layer_keeps_bits_and_winners_of_the_exact_input():
    """Kept ReLU bits and kept winners come from the forward, so only what multiplies the input sees the kept values:
    dX of those layers has the exact layer's bits."""
    import granulelayer_amd as G

    for kw in (dict(pooling="mean", plan=G.PhysicalPlan(relu_bits="keep")), dict(pooling="max")):
        lay = [G.SparsePoolingLayer(200, 4096, 8, shared_neurons=None, dtype=torch.float32, device=DEV, seed=1, bias_std=0.2,
                                    activation_checkpoint=c, **kw) for c in ("exact", "int8")]
        x = torch.randn(37, 200, device=DEV)
        dy = torch.randn(37, 8, device=DEV)
        grads = []
        for m in lay:
            xl = x.clone().requires_grad_(True)
            grads.append(torch.autograd.grad(m(xl), [xl, m.weight], dy))
        if "plan" not in kw:  # the dX pass of the ReLU sums recomputes z
            assert torch.equal(grads[0][0], grads[1][0])
        # dW is a sum of dz x over the tokens: off by the input's half steps, below 1/126 of a block's maximum
        rel = float((grads[0][1] - grads[1][1]).norm() / grads[0][1].norm())
        assert 0 < rel < 4 / 126
    with torch.no_grad():
        lay[1](x)
        assert lay[1].last_info["input_checkpoint_bytes"] == x.numel() * 4  # nothing is put away without a backward


def test_a_block_of_layers_trains_in_8_bits():
    """Dense projection -> sparse layer -> dense projection back onto the stream, all keeping 8 bits: gradients
    near the exact ones, parameters stepped by the fused optimizer."""
    from granulelayer_amd import DenseProjection, FusedAdamW, SparsePoolingLayer

    def model(ckpt):
        up = DenseProjection(192, 256, "gelu", dtype=torch.bfloat16, device=DEV, seed=1, activation_checkpoint=ckpt)
        mid = SparsePoolingLayer(256, 16384, 64, shared_neurons=None, pooling=dict(type="mean", activation="gelu"),
                                 dtype=torch.bfloat16, device=DEV, seed=2, activation_checkpoint=ckpt)
        down = DenseProjection(64, 192, dtype=torch.bfloat16, device=DEV, seed=3, activation_checkpoint=ckpt)
        return torch.nn.ModuleList([up, mid, down])

    def loss(m, x):
        up, mid, down = m
        return (down(mid(up(x)), x).float() ** 2).mean()

    x = torch.randn(4, 40, 192, generator=torch.Generator().manual_seed(0)).to(DEV).bfloat16()
    grads = {}
    for ckpt in ("exact", "int8"):
        m = model(ckpt)
        for layer in m:
            layer.enable_main_grad()
        xl = x.clone().requires_grad_(True)
        loss(m, xl).backward()
        grads[ckpt] = [xl.grad.float()] + [p.main_grad.clone() for p in m.parameters()]
    for a, b in zip(grads["exact"], grads["int8"]):
        # kept values are within 1/127 of their block's maximum (here below 4 deviations: 3% of a deviation, and
        # uniform in their step: half of that), once in the input and once in z, over three layers
        assert float((a - b).norm() / a.norm()) < 0.1
    opt = FusedAdamW(m.parameters(), lr=1e-3)
    opt.step()
    assert all(not bool(p.main_grad.any()) for p in m.parameters())


SMOOTH = {
    "lme": dict(type="logmeanexp"),
    "lme cold": dict(type="logmeanexp", temperature=0.05),
    "lme gelu": dict(type="logmeanexp", temperature=0.1, activation="gelu", out_activation="gelu"),
    "softmax": dict(type="softmax_weighted", beta=10.0),
    "softmax gelu": dict(type="softmax_weighted", activation="gelu"),
    "power": dict(type="power_mean", p=4.0),
    "power odd": dict(type="power_mean", p=2.5),
    "two": dict(levels=[dict(type="softmax_weighted", beta=10.0, neurons_per_shard=128), dict(type="logmeanexp")],
                level1_checkpoint="save"),
    "two power": dict(levels=[dict(type="power_mean", p=4.0, neurons_per_shard=128, out_activation="gelu"), dict(type="sum")],
                      level1_checkpoint="save"),
}


@pytest.mark.parametrize("large", [False, True])
@pytest.mark.parametrize("pooling", SMOOTH.values(), ids=SMOOTH.keys())
def test_smooth_pools_take_their_normalisers_from_the_kept_input(pooling, large):
    """A smooth pool's gradient divides by what its forward summed: with an input kept in 8 bits, that of the kept
    values, also under the default policy, which keeps the exact input's.  The gradients have the bits of an exact layer at the
    kept values that recomputes its statistics; one large feature a block makes the kept values coarse."""
    import granulelayer_amd as G

    def layer(ckpt, pooling, **kw):
        return G.SparsePoolingLayer(250, 6144, 12, shared_neurons=None, pooling=pooling, dtype=torch.float32, device=DEV,
                                    seed=4, bias_std=0.3, activation_checkpoint=ckpt, **kw)

    eight = layer("int8", pooling)
    if "levels" in pooling:
        exact = layer("exact", dict(pooling, level1_checkpoint="recompute"))
    else:
        exact = layer("exact", pooling, checkpoint_policy="recompute_stats")
    x = torch.randn(3, 17, 250, generator=torch.Generator().manual_seed(1)).to(DEV)
    if large:
        x[..., ::32] *= 30
    xe = x.clone().requires_grad_(True)
    xk = pack_activation(x).unpack().requires_grad_(True)
    y = eight(xe)
    assert torch.equal(y, exact(x))
    dy = torch.randn(y.shape, generator=torch.Generator().manual_seed(6)).to(DEV)
    got = torch.autograd.grad(y, [xe, eight.weight, eight.bias], dy)
    want = torch.autograd.grad(exact(xk), [xk, exact.weight, exact.bias], dy)
    for g, w in zip(got, want):
        assert g.dtype == w.dtype and torch.equal(g, w)


@pytest.mark.parametrize("pool", ["mean", "sum"])
def test_kept_relu_bits_are_the_mask_of_every_gradient(pool):
    """PhysicalPlan(relu_bits="keep") with an input in 8 bits: the exact input's bits mask dW, db and dX alike.  dX and db do
    not multiply the input, so they have the exact layer's bits; dW is dz^T x over those neurons, in the kept x."""
    import granulelayer_amd as G

    D, H, U = 200, 4096, 8
    lay = [G.SparsePoolingLayer(D, H, U, shared_neurons=None, pooling=pool, dtype=torch.float32, device=DEV, seed=1,
                                bias_std=0.2, activation_checkpoint=c, plan=G.PhysicalPlan(relu_bits="keep"))
           for c in ("exact", "int8")]
    x = torch.randn(37, D, generator=torch.Generator().manual_seed(2)).to(DEV)
    dy = torch.randn(37, U, generator=torch.Generator().manual_seed(3)).to(DEV)
    grads = []
    for m in lay:
        xl = x.clone().requires_grad_(True)
        grads.append(torch.autograd.grad(m(xl), [xl, m.weight, m.bias], dy))
        assert m.last_info["backward_relu_mask"]
    assert torch.equal(grads[0][0], grads[1][0]) and torch.equal(grads[0][2], grads[1][2])
    m = lay[1]
    idx = m.indices.reshape(-1, 8).long()
    w6, b6 = m.weight.detach().double().reshape(-1, 8), m.bias.detach().double().reshape(-1)
    z = torch.stack([(x[t].double()[idx] * w6).sum(-1) + b6 for t in range(37)])  # [37, slots]
    slots = z.shape[1] // U
    counts = m.layout.counts_tensor(DEV).double()
    there = torch.arange(slots, device=DEV).repeat(U) < counts.repeat_interleave(slots)
    c1 = (dy.double() / (counts if pool == "mean" else 1.0)).repeat_interleave(slots, 1)
    dz = torch.where((z > 0) & there, c1, 0.0)
    # neurons with a z within its rounding of 0 (9 roundings of at most the terms' sum) may go either way: a few at most
    mag = torch.stack([(x[t].double()[idx] * w6).abs().sum(-1) + b6.abs() for t in range(37)])
    sure = ~((z.abs() <= 9 * 2.0 ** -24 * mag) & there).any(0)
    assert float(sure.double().mean()) > 0.99
    xk = pack_activation(x).unpack().double()
    want = torch.stack([(dz[:, :, None] * v[:, idx]).sum(0) for v in (x.double(), xk)])
    # 37 products of fp32 added in fp32, from a coefficient that is rounded once
    bound = 40 * 2.0 ** -24 * (dz.abs()[:, :, None] * xk[:, idx].abs()).sum(0)
    got = grads[1][1].double().reshape(-1, 8)
    assert bool(((got - want[1]).abs() <= bound)[sure].all())
    assert bool(((got - want[0]).abs() > bound)[sure].any())  # and the kept x's, not the exact one's


@pytest.mark.parametrize("kind", ["mean", "lme", "two", "cover"])
@pytest.mark.parametrize("ckpt", ["exact", "int8"])
def test_layers_under_activation_checkpointing(kind, ckpt):
    from torch.utils.checkpoint import checkpoint

    lay = sparse_layer(kind, ckpt)
    x = torch.randn(9, 256 if kind == "cover" else 250, device=DEV, requires_grad=True)
    leaves = [x, lay.weight, lay.bias]
    want = torch.autograd.grad(lay(x).square().sum(), leaves)
    got = torch.autograd.grad(checkpoint(lay, x, use_reentrant=False).square().sum(), leaves)
    for g, w in zip(got, want):
        assert torch.equal(g, w)
