"""8-bit moments whose codes are drawn (FusedAdamW's default): right on average in one step and after thousands of them.

Sums of errors are compared with five times their own standard deviation, which follows from the probabilities that keep a value on
average: between codes lo and hi a value x has the variance (hi - x)(x - lo)."""
import numpy as np
import pytest
import torch

from conftest import gpu_available

from granulelayer_amd import FusedAdamW
from granulelayer_amd.backend import HipBackend, adam_row

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a ROCm GPU")]
DEV = "cuda"
B1, B2 = 0.9, 0.999


def _state(n, seed):
    rng = np.random.default_rng(seed)
    nb = -(-n // 256)
    return dict(m=rng.integers(-127, 128, n).astype(np.int8), v=rng.integers(1, 256, n).astype(np.uint8),
                m_scale=np.exp(rng.standard_normal(nb)).astype(np.float32) / 127 ** 2,
                v_scale=np.exp(rng.standard_normal(nb)).astype(np.float32) / 255 ** 2)


def _step(state, g, t, p, pdt=torch.float32):
    """State of a parameter after a step from ``state``."""
    p = torch.nn.Parameter(torch.from_numpy(p).to(DEV, pdt))
    opt = FusedAdamW([p], moments="int8", betas=(B1, B2), lr=1e-3)
    opt.state[p] = dict(step=t - 1, **{k: torch.from_numpy(a.copy()).to(DEV) for k, a in state.items()})
    p.main_grad = torch.from_numpy(g).to(DEV)
    opt.step()
    return {k: a.cpu().numpy() for k, a in opt.state[p].items() if k != "step"}


def _exact(state, g):
    of = np.arange(g.size) // 256
    m, v, g = state["m"].astype(np.float64), state["v"].astype(np.float64), g.astype(np.float64)
    m = B1 * m * np.abs(m) * state["m_scale"].astype(np.float64)[of] + (1 - B1) * g
    v = B2 * (v * v * state["v_scale"].astype(np.float64)[of]) ** 2 + (1 - B2) * g * g
    return m, v


def _drawn(codes, q, power, most):
    """Checks codes of the quotients q = code^power; the share of the way up of each and whether it was taken, of those
    between two codes."""
    root = lambda x: np.floor(x ** (1.0 / power))  # noqa: E731
    least, top = np.minimum(root(q * (1 - 2.0 ** -20)), most - 1), np.minimum(root(q * (1 + 2.0 ** -20)) + 1, most)
    assert ((codes >= least) & (codes <= top)).all()
    lo = np.minimum(root(q), most - 1)
    share = (q - lo ** power) / ((lo + 1) ** power - lo ** power)
    between = (share > 2.0 ** -10) & (share < 1 - 2.0 ** -10)
    return lo, share, codes > lo, between


@pytest.mark.parametrize("n", [1 << 18, 1001])
def test_codes_are_neighbours_and_right_on_average(n):
    rng = np.random.default_rng(1)
    state, g = _state(n, 2), (0.3 * rng.standard_normal(n)).astype(np.float32)
    p = rng.standard_normal(n).astype(np.float32)
    m, v = _exact(state, g)
    got = _step(state, g, 5, p)
    of = np.arange(n) // 256
    tops = np.stack([np.maximum.reduceat(np.abs(x).astype(np.float32), np.arange(0, n, 256)) for x in (m, v)]).astype(np.float64)
    np.testing.assert_array_equal(got["m_scale"], (tops[0] / 127 ** 2).astype(np.float32))
    np.testing.assert_array_equal(got["v_scale"], (np.sqrt(tops[1]) / 255 ** 2).astype(np.float32))
    assert (got["m"] * m >= 0).all()
    taken = []
    for codes, q, power, most in (
            (np.abs(got["m"].astype(np.float64)), np.abs(m) / got["m_scale"].astype(np.float64)[of], 2, 127),
            (got["v"].astype(np.float64), v / got["v_scale"].astype(np.float64)[of] ** 2, 4, 255)):
        lo, share, up, between = _drawn(codes, q, power, most)
        if power == 4:
            assert (codes >= 1).all()
            between &= lo >= 1
        for a, b in ((0, 4), (4, 16), (16, 64), (64, 256)):
            k = between & (lo >= a) & (lo < b)
            assert abs((up - share)[k].sum()) <= 5 * np.sqrt((share * (1 - share))[k].sum()), (power, a)
        taken.append(np.where(between, (up - share) / np.sqrt(np.maximum(share * (1 - share), 1e-9)), 0.0))
    # the draws of m and v, of neighbours, and of elements a vector, a half and a block apart have nothing to do with each other
    pairs = [(taken[0], taken[1])] + [(t[:-d], t[d:]) for t in taken for d in (1, 2, 3, 4, 128, 256)]
    for a, b in pairs:
        assert abs((a * b).sum()) <= 5 * np.sqrt((a * a * b * b).sum())


def test_draws_of_steps_differ_and_of_equal_calls_do_not():
    n = 1 << 16
    rng = np.random.default_rng(3)
    state, g = _state(n, 4), (0.3 * rng.standard_normal(n)).astype(np.float32)
    p = rng.standard_normal(n).astype(np.float32)
    a, b = _step(state, g, 5, p), _step(state, g, 5, p)
    for k in a:
        np.testing.assert_array_equal(a[k], b[k])
    others = [_step(state, g, 6, p), _step(state, g, 5, p + 1)]  # another step; another parameter
    m, v = _exact(state, g)
    of = np.arange(n) // 256
    for c in others:
        for key, x, power, most in (("m", np.abs(m) / a["m_scale"].astype(np.float64)[of], 2, 127),
                                    ("v", v / a["v_scale"].astype(np.float64)[of] ** 2, 4, 255)):
            ea, ec = ((np.abs(s[key].astype(np.float64)), x, power, most) for s in (a, c))
            lo, share, up, between = _drawn(*ea)
            _, _, up2, _ = _drawn(*ec)
            z = ((up - share) * (up2 - share) / np.maximum(share * (1 - share), 1e-9))[between & (lo >= 1)]
            assert abs(z.sum()) <= 5 * np.sqrt((z * z).sum())


@pytest.mark.parametrize("pdt,master", [(torch.float32, False), (torch.bfloat16, False), (torch.bfloat16, True)])
def test_every_kind_of_parameter_draws(pdt, master):
    n = 1 << 16
    rng = np.random.default_rng(5)
    p = torch.nn.Parameter(torch.zeros(n, device=DEV, dtype=pdt))
    opt = FusedAdamW([p], moments="int8", betas=(B1, B2), master_weights=master)
    p.grad = torch.from_numpy(rng.standard_normal(n).astype(np.float32)).to(DEV, pdt)
    g = p.grad.float().cpu().numpy()
    opt.step()
    st = {k: a.cpu().numpy() for k, a in opt.state[p].items() if k != "step"}
    m = (1 - B1) * g.astype(np.float64)
    lo, share, up, between = _drawn(np.abs(st["m"].astype(np.float64)), np.abs(m) / st["m_scale"].astype(np.float64)[np.arange(n) // 256], 2, 127)
    assert abs((up - share)[between].sum()) <= 5 * np.sqrt((share * (1 - share))[between].sum())


def _follow(phases, n, lr=1e-3, b2=B2):
    """fp32 and 8-bit moments over the same gradients; phases: (scale of every element, steps, gradients of one sign)."""
    gen = torch.Generator(device=DEV).manual_seed(6)
    ps = [torch.nn.Parameter(torch.zeros(n, device=DEV)) for _ in range(2)]
    opts = [FusedAdamW([p], moments=k, lr=lr, betas=(B1, b2)) for p, k in zip(ps, ("fp32", "int8"))]
    was = []
    for scale, steps, constant in phases:
        was = [p.detach().clone() for p in ps]
        for _ in range(steps):
            g = scale if constant else scale * (0.3 + torch.randn(n, generator=gen, device=DEV))
            for p, o in zip(ps, opts):
                p.grad = g.clone()
                o.step()
    ways = [p.detach() - w for p, w in zip(ps, was)]
    (_, v32), (m8, v8) = (o.moment_values()[0] for o in opts)
    return v32.double(), m8, v8.double(), [w.double() for w in ways]


def test_moments_decay_where_gradients_get_small_or_stop():
    """5,000 steps after part of every block's gradients fell to a hundredth or to nothing.  A step moves v by about 1 / 1000 of
    itself and the block's scale by less than 4 / 1000, between codes 4 / c of v apart, and forgets 1 / 1000 of what it was off by: a
    variance of 0.005 (4 / c) / 0.002 = 10 / c of v^2 at most.  Codes here are 20 and more: of 512 elements' mean, 0.71 / sqrt(512)
    = 3.1%, of 4096, 1.1%; bounds of five times that.  What a parameter goes is off by half of v's share at most, 0.35."""
    n = 8192
    i = torch.arange(n, device=DEV) % 256
    one = torch.ones(n, device=DEV)
    scale = torch.where(i % 2 == 0, 1.0, 0.01)
    scale[i % 16 == 1] = 0.0
    v32, m8, v8, ways = _follow([(one, 500, False), (scale, 5000, False)], n)
    for s in (1.0, 0.01, 0.0):
        k = scale == s
        bound = 5 * 0.71 / float(k.sum()) ** 0.5
        assert abs(float(v8[k].mean() / v32[k].mean()) - 1) < bound, s
        if s:
            assert float((ways[1][k] - ways[0][k]).norm() / ways[0][k].norm()) < 0.35, s
    assert not m8[scale == 0].any()


def test_moments_decay_beside_constant_gradients():
    n = 8192
    one = torch.ones(n, device=DEV)
    stopped = torch.arange(n, device=DEV) % 2 == 1
    v32, m8, v8, _ = _follow([(one, 200, True), (torch.where(stopped, 0.0, one), 1500, True)], n)
    # codes of 120 and more: sqrt(10 / 120) / sqrt(4096) = 0.45%, five times
    assert abs(float(v8[stopped].mean() / v32[stopped].mean()) - 1) < 0.0226
    assert not m8[stopped].any()
    assert float((v8 / v32 - 1)[~stopped].abs().max()) < 2.0 ** -6  # each the largest of its block


def test_moments_decay_beside_constant_gradients_after_the_corrections():
    """b2 = 0.95: when gradients stop, 600 equal steps have made moments, scales and corrections constants.  A step moves v by 0.05 of
    itself between codes 4 / c apart, and forgets as much: a variance of 0.05 (4 / c) / 0.1 = 2 / c of v^2, c = 5 after 300
    steps: sqrt(0.4) / sqrt(4096) = 1%, five times; and 1 / c^4 where v may not fall below the code 1."""
    n = 8192
    one = torch.ones(n, device=DEV)
    stopped = torch.arange(n, device=DEV) // 4 % 2 == 1  # all that a draw is made of
    v32, m8, v8, _ = _follow([(one, 600, True), (torch.where(stopped, 0.0, one), 300, True)], n, b2=0.95)
    assert abs(float(v8[stopped].mean() / v32[stopped].mean()) - 1) < 0.05 + 0.0016
    assert not m8[stopped].any()


def test_slow_second_moments_decay():
    """b2 = 0.9999, gradients that fall to nearly nothing: a step takes 1 / 4000 of the way to the next code where c = 10.  Of v that the
    steps leave alone but for the share 1 - b2, variances are 2 / c of v^2; codes of 20 and more after 20,000 steps (v is 0.135 of
    what it was, 1e-4 of the others'): sqrt(0.1) / sqrt(4096) = 0.5%, five times; twice that for the block's scale, which moves."""
    n = 8192
    one = torch.ones(n, device=DEV)
    small = torch.arange(n, device=DEV) // 4 % 2 == 1
    first = torch.where(small, 0.03, one)
    v32, _, v8, _ = _follow([(first, 3000, False), (torch.where(small, 1e-5, one), 20000, False)], n, b2=0.9999)
    assert abs(float(v8[small].mean() / v32[small].mean()) - 1) < 0.05
    assert abs(float(v8[~small].mean() / v32[~small].mean()) - 1) < 0.0226


def test_like_gradients_keep_their_moments():
    """Codes of 60 and more for nearly all: sqrt(10 / 60) / sqrt(8192) = 0.45%, five times."""
    n = 8192
    v32, _, v8, ways = _follow([(torch.ones(n, device=DEV), 3000, False)], n)
    assert abs(float(v8.mean() / v32.mean()) - 1) < 0.0226
    assert float((ways[1] - ways[0]).norm() / ways[0].norm()) < 0.2


def test_values_of_more_elements_than_a_launch_takes():
    """2^34 elements, 2^32 threads in all: 32 rows of one tensor's codes, most of them into one place (each writes the same)."""
    n = 1 << 29
    codes = torch.arange(256, device=DEV, dtype=torch.int32)
    m, v = codes.to(torch.int8).repeat(n // 256), codes.to(torch.uint8).repeat(n // 256)
    scales = [torch.rand(n // 256, device=DEV) + 0.5 for _ in range(2)]
    places = {i: [torch.zeros(n, device=DEV) for _ in range(2)] for i in (0, 15, 16, 31)}
    rows = [adam_row(places.get(i, places[0])[1].data_ptr(), places.get(i, places[0])[0].data_ptr(), m.data_ptr(), v.data_ptr(), 0,
                     scales[0].data_ptr(), scales[1].data_ptr(), n, 0, 1.0, 1.0) for i in range(32)]
    HipBackend.get().adam_values(m.device, rows)
    torch.cuda.synchronize()
    for k in (0, 1, n // 512, n // 256 - 1):
        part = slice(256 * k, 256 * k + 256)
        cm, cv = m[part].double(), v[part].double()
        wm, wv = (cm * cm.abs() * scales[0][k].double()).float(), (cv * cv * scales[1][k].double()).square().float()
        for pm, pv in places.values():
            assert torch.equal(pm[part], wm) and torch.equal(pv[part], wv)
    for pm, pv in places.values():
        assert torch.equal(pm, places[0][0]) and torch.equal(pv, places[0][1])
