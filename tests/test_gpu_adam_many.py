"""FusedAdamW over many tensors at once and its 8-bit moments on the GPU.

fp32 and bf16 moments: bit for bit the single-tensor step, whatever the tensors' number, sizes, places and kinds of
gradients.  8-bit moments: codes and scales equal to a restatement in float64; parameters within the roundings of
an fp32 update."""
import numpy as np
import pytest
import torch

from conftest import gpu_available

from granulelayer_amd import FusedAdamW
from granulelayer_amd.backend import HipBackend, adam_row

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a ROCm GPU")]
DEV = "cuda"
HP = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)
SIZES = [1, 3, 4, 255, 256, 257, 1000, 4095, 4096, 4097, 12345]


def _at(n, dtype, offset, gen, scale=1.0):
    """n values ``offset`` elements into a buffer."""
    buf = torch.randn(n + offset + 8, generator=gen, device=DEV) * scale
    return buf.to(dtype)[offset:offset + n]


# ---- fp32 and bf16 moments --------------------------------------------------------------------------------
@pytest.mark.parametrize("moments", ["fp32", "bf16"])
@pytest.mark.parametrize("kind", ["fp32", "nearest", "master", "stochastic"])
@pytest.mark.parametrize("main", [False, True])
def test_many_tensors_equal_single_steps(moments, kind, main):
    gen = torch.Generator(device=DEV).manual_seed(3)
    pdt = torch.float32 if kind == "fp32" else torch.bfloat16
    sizes = SIZES * 5  # 55 tensors: two launches
    params = [torch.nn.Parameter(torch.randn(n, generator=gen, device=DEV).to(pdt)) for n in sizes]
    opt = FusedAdamW(params, moments=moments, master_weights=kind == "master", stochastic_rounding=kind == "stochastic", **HP)
    mdt = torch.float32 if moments == "fp32" else torch.bfloat16
    want = [dict(p=p.detach().clone(), m=torch.zeros(p.shape, device=DEV, dtype=mdt),
                 v=torch.zeros(p.shape, device=DEV, dtype=mdt),
                 master=p.detach().float() if kind == "master" else None) for p in params]
    b1, b2 = HP["betas"]
    seed = 0
    for t in (1, 2, 3):
        grads = [torch.randn(n, generator=gen, device=DEV).to(torch.float32 if main else pdt) for n in sizes]
        for p, g in zip(params, grads):
            if main:
                p.main_grad = g.clone()
            else:
                p.grad = g.clone()
        opt.step()
        for w, g in zip(want, grads):
            seed += 1
            HipBackend.get().adam(w["p"], g.float(), w["m"], w["v"], HP["lr"], b1, b2, HP["eps"], HP["weight_decay"],
                                  1 - b1 ** t, 1 - b2 ** t, master=w["master"], stochastic=kind == "stochastic", seed=seed)
    for p, w in zip(params, want):
        st = opt.state[p]
        assert st["step"] == 3
        assert torch.equal(p.detach(), w["p"]) and torch.equal(st["m"], w["m"]) and torch.equal(st["v"], w["v"])
        if kind == "master":
            assert torch.equal(st["master"], w["master"])
        if main:
            assert not p.main_grad.any()
        else:
            assert p.grad is None


def test_values_next_to_a_tensor_stay():
    """Tensors in the middle of buffers, at addresses of one element's alignment."""
    gen = torch.Generator(device=DEV).manual_seed(4)
    for pdt in (torch.float32, torch.bfloat16):
        for moments in ("fp32", "bf16", "int8"):
            bufs, params = [], []
            for n in (5, 256, 259, 4099):
                for off in (1, 2, 3):
                    buf = torch.randn(n + 16, generator=gen, device=DEV).to(pdt)
                    bufs.append((buf, buf.clone(), off, n))
                    params.append(torch.nn.Parameter(buf[off:off + n]))
            opt = FusedAdamW(params, moments=moments, **HP)
            for p in params:
                p.grad = _at(p.numel(), pdt, 1, gen)
            opt.step()
            for buf, was, off, n in bufs:
                assert torch.equal(buf[:off], was[:off]) and torch.equal(buf[off + n:], was[off + n:])
                assert not torch.equal(buf[off:off + n], was[off:off + n])


def test_gradients_of_both_kinds_and_none():
    p = [torch.nn.Parameter(torch.ones(300, device=DEV, dtype=dt)) for dt in (torch.float32, torch.bfloat16) * 2]
    p[0].main_grad = torch.ones(300, device=DEV)
    p[1].grad = torch.ones(300, device=DEV, dtype=torch.bfloat16)
    p[2].grad = torch.ones(600, device=DEV)[::2]  # strided
    opt = FusedAdamW(p, stochastic_rounding=False, lr=0.5, moments="fp32")
    opt.step()
    for q in p[:3]:
        np.testing.assert_allclose(q.detach().float().cpu(), 0.5, rtol=2 ** -8)  # the first step is lr
    assert torch.equal(p[3].detach(), torch.ones_like(p[3])) and p[3] not in opt.state


@pytest.mark.filterwarnings("ignore:optimizer contains a parameter group with duplicate")
def test_a_parameter_that_is_there_twice():
    """Two steps of it one after the other: the second has no gradient left (p.grad), or a zeroed one (main_grad)."""
    for main in (False, True):
        p, q = (torch.nn.Parameter(torch.ones(3000, device=DEV)) for _ in range(2))
        opt = FusedAdamW([p, q, p], moments="fp32", lr=0.5, betas=(0.5, 0.5))
        for t in (p, q):
            if main:
                t.main_grad = torch.ones(3000, device=DEV)
            else:
                t.grad = torch.ones(3000, device=DEV)
        opt.step()
        assert opt.state[p]["step"] == (2 if main else 1) and opt.state[q]["step"] == 1
        # m = 1/2 then 1/4, v the same; corrected by 1 - 1/2 and 1 - 1/4: steps of 1/2 and of 1/2 (1/3) / sqrt(1/3)
        want = 0.5 - (0.5 * 3 ** -0.5 if main else 0.0)
        np.testing.assert_allclose(p.detach().cpu(), want, rtol=0, atol=2 ** -20)
        np.testing.assert_allclose(q.detach().cpu(), 0.5, rtol=0, atol=2 ** -20)


# ---- 8-bit moments ----------------------------------------------------------------------------------------
@pytest.mark.parametrize("shared", ["storage", "main_grad"])
def test_parameters_that_share_memory_step_one_after_the_other(shared):
    n = 300_000
    gen = torch.Generator(device=DEV).manual_seed(4)
    data = torch.randn(2, n, device=DEV, generator=gen)
    grads = torch.randn(2, n, device=DEV, generator=gen)

    def make(together):
        a, b = data.clone()
        ps = [torch.nn.Parameter(a), torch.nn.Parameter(a if shared == "storage" else b)]
        gs = grads.clone()
        for p, g in zip(ps, (gs[0], gs[0] if shared == "main_grad" else gs[1])):
            p.main_grad = g
        groups = [dict(params=ps)] if together else [dict(params=[p]) for p in ps]
        return ps, FusedAdamW(groups, lr=1e-2, moments="fp32", weight_decay=0.1)

    (got, one), (want, two) = make(True), make(False)
    for opt in (one, two):
        for _ in range(3):
            opt.step()
    for p, q in zip(got, want):
        assert torch.equal(p, q) and not p.main_grad.any()
        assert torch.equal(one.state[p]["m"], two.state[q]["m"]) and one.state[p]["step"] == 3


def test_a_state_whose_memory_moved():
    """A state's tensor that has other memory under it is read and written there."""
    p, q = (torch.nn.Parameter(torch.full((1000,), 0.5, device=DEV, dtype=torch.bfloat16)) for _ in range(2))
    opts = [FusedAdamW([t], lr=1e-2, moments="int8", master_weights=True) for t in (p, q)]
    for k in range(4):
        for t, opt in zip((p, q), opts):
            t.grad = torch.full_like(t, 0.25 + k)
            opt.step()
        st = opts[1].state[q]
        for key in ("master", "m_scale", "v_scale", "m", "v"):
            st[key].data = st[key].data.clone()
    a, b = opts[0].state[p], opts[1].state[q]
    assert torch.equal(p, q) and all(torch.equal(a[k], b[k]) for k in ("master", "m_scale", "v_scale", "m", "v"))


def _values(cm, sm, cv, sv, n):
    of = np.arange(n) // 256
    m = cm.astype(np.float64) * np.abs(cm.astype(np.float64)) * sm.astype(np.float64)[of]
    v = (cv.astype(np.float64) ** 2 * sv.astype(np.float64)[of]) ** 2
    return m, v


def _encode(m, v):
    n = m.size
    nb = -(-n // 256)
    cm, cv = np.zeros(n, np.int8), np.zeros(n, np.uint8)
    sm, sv = np.zeros(nb, np.float32), np.zeros(nb, np.float32)
    for b in range(nb):
        k = slice(256 * b, min(n, 256 * b + 256))
        with np.errstate(over="ignore"):
            top, vtop = np.abs(m[k]).astype(np.float32).max(), v[k].astype(np.float32).max()
        if not np.isfinite(top):
            sm[b] = np.nan
        elif top >= 2.0 ** -100:
            sm[b] = np.float32(np.float64(top) / 127 ** 2)
            cm[k] = np.copysign(np.floor(np.sqrt(np.abs(m[k]) / np.float64(sm[b])) + 0.5), m[k]).astype(np.int8)
        if not np.isfinite(vtop):
            sv[b] = np.nan
        elif vtop >= 2.0 ** -126:
            sv[b] = np.float32(np.sqrt(np.float64(vtop)) / 255 ** 2)
            c = np.floor(np.sqrt(np.sqrt(v[k]) / np.float64(sv[b])) + 0.5)
            cv[k] = np.where((c == 0) & (v[k] > 0), 1, c).astype(np.uint8)
    return cm, sm, cv, sv


class Reference8:
    """A tensor's step with 8-bit moments in float64."""

    def __init__(self, p):
        n = p.size
        self.p = p.astype(np.float64)
        self.state = (np.zeros(n, np.int8), np.zeros(-(-n // 256), np.float32), np.zeros(n, np.uint8),
                      np.zeros(-(-n // 256), np.float32))

    def step(self, g, t, p_from):
        """p after a step from ``p_from`` (the parameter as it is stored), and how far an fp32 update may be off."""
        (b1, b2), lr = HP["betas"], HP["lr"]
        m, v = _values(*self.state, g.size)
        g = g.astype(np.float64)
        with np.errstate(over="ignore", invalid="ignore"):
            m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
            upd = (m / (1 - b1 ** t)) / (np.sqrt(v / (1 - b2 ** t)) + HP["eps"])
            self.state = _encode(m, v)
            p = p_from.astype(np.float64) * (1 - lr * HP["weight_decay"]) - lr * upd
        # In halves of a last place, 2^-24.  p: its product with 1 - lr wd (itself off by lr, wd, their product and the
        # difference), 5, and the last sum, of p.  upd: m, v under a root, 1 / bc1 and 1 / bc2 (each as fp32 and its
        # quotient; the second's root with half of them), lr and five products or sums, 12, and an estimated root and
        # quotient of two each: 16
        tol = 2.0 ** -24 * (5 * np.abs(p_from) + 16 * lr * np.abs(upd) + np.abs(p))
        return p, tol


def _state8(st):
    return (st["m"].cpu().numpy().reshape(-1), st["m_scale"].cpu().numpy(), st["v"].cpu().numpy().reshape(-1),
            st["v_scale"].cpu().numpy())


@pytest.mark.parametrize("pdt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("main", [False, True])
def test_8bit_moments_equal_float64(pdt, main):
    gen = torch.Generator(device=DEV).manual_seed(5)
    params = [torch.nn.Parameter(torch.randn(n, generator=gen, device=DEV).to(pdt)) for n in SIZES]
    opt = FusedAdamW(params, moments="int8", stochastic_rounding=False, **HP)
    refs = [Reference8(p.detach().float().cpu().numpy()) for p in params]
    for t in range(1, 6):
        was = [p.detach().float().cpu().numpy() for p in params]
        grads = []
        for i, p in enumerate(params):
            g = torch.randn(p.numel(), generator=gen, device=DEV) * torch.exp(3 * torch.randn(p.numel(), generator=gen, device=DEV))
            if t == 3:
                g[::7] = 0
            if t == 4:
                g.mul_(1e-12)
            g = g.to(torch.float32 if main else pdt)
            grads.append(g.float().cpu().numpy())
            if main:
                p.main_grad = g
            else:
                p.grad = g
        opt.step()
        for p, ref, g, w in zip(params, refs, grads, was):
            want, tol = ref.step(g, t, w)
            for got, exp, name in zip(_state8(opt.state[p]), ref.state, ("m", "m_scale", "v", "v_scale")):
                np.testing.assert_array_equal(got, exp, err_msg=f"{name} of {p.numel()} at step {t}")
            got = p.detach().float().cpu().numpy().astype(np.float64)
            if pdt == torch.bfloat16:
                tol = tol + 2.0 ** -8 * np.abs(want) + 2.0 ** -133
            assert (np.abs(got - want) <= tol).all()
    for (m, v), ref, p in zip(opt.moment_values(), refs, params):
        wm, wv = _values(*ref.state, p.numel())
        np.testing.assert_array_equal(m.cpu().numpy(), wm.astype(np.float32))
        np.testing.assert_array_equal(v.cpu().numpy(), wv.astype(np.float32))


def test_8bit_moments_that_are_no_numbers_or_nothing():
    n = 1024
    p = torch.nn.Parameter(torch.ones(n, device=DEV))
    g = torch.zeros(n, device=DEV)
    g[3] = float("nan")           # block 0
    g[256 + 9] = float("inf")     # block 1
    g[512:768] = 1e-36            # block 2: m below its least scale, v below fp32
    g[768] = 3e38                 # block 3: v past fp32
    opt = FusedAdamW([p], moments="int8", **HP)
    ref = Reference8(np.ones(n, np.float32))
    p.grad = g.clone()
    opt.step()
    ref.step(g.cpu().numpy(), 1, np.ones(n, np.float32))
    for got, exp in zip(_state8(opt.state[p]), ref.state):
        np.testing.assert_array_equal(got, exp)
    s = opt.state[p]
    assert torch.isnan(s["m_scale"]).tolist() == [True, True, False, False]
    assert torch.isnan(s["v_scale"]).tolist() == [True, True, False, True]
    assert s["m_scale"][2] == 0 and s["v_scale"][2] == 0
    q = p.detach().cpu()
    assert torch.isnan(q[[3, 256 + 9]]).all() and torch.isfinite(q[[0, 255, 256, 511, 512, 767, 769]]).all()
    p.grad = torch.zeros(n, device=DEV)
    opt.step()
    m, v = opt.moment_values()[0]
    assert torch.isnan(m[:512]).all() and torch.isnan(v[:512]).all() and not m[512:768].any() and not v[512:768].any()


def test_8bit_moments_follow_fp32_moments():
    """A step takes unrounded moments, so one step from equal moments differs by nothing but fp32 roundings; over 50
    steps the parameters stay within a share of their way: each step's m and sqrt(v) are off by at most half a code,
    1 / c of themselves, and a decayed sum of such errors is no larger than the terms' own."""
    gen = torch.Generator(device=DEV).manual_seed(6)
    n = 5000
    start = torch.randn(n, generator=gen, device=DEV)
    ps = [torch.nn.Parameter(start.clone()) for _ in range(2)]
    opts = [FusedAdamW([p], moments=k, lr=1e-3) for p, k in zip(ps, ("fp32", "int8"))]
    scale = 0.1 + torch.rand(n, generator=gen, device=DEV)
    for _ in range(50):
        g = scale * (1 + torch.randn(n, generator=gen, device=DEV))
        for p, o in zip(ps, opts):
            p.grad = g.clone()
            o.step()
    way, apart = (ps[0] - start).norm(), (ps[1] - ps[0]).norm()
    assert apart < 0.05 * way


def test_hundreds_of_tensors_and_an_empty_one():
    gen = torch.Generator(device=DEV).manual_seed(7)
    sizes = [1 + 37 * i % 900 for i in range(300)]
    sizes[17] = 0
    for moments in ("fp32", "int8"):
        params = [torch.nn.Parameter(torch.randn(n, generator=gen, device=DEV)) for n in sizes]
        was = [p.detach().clone() for p in params]
        for p in params:
            p.grad = torch.randn(p.shape, generator=gen, device=DEV)
        signs = [p.grad.sign() for p in params]
        FusedAdamW(params, moments=moments, lr=0.5, eps=1e-30).step()
        # The first step is lr against the gradient's sign.  With fp32 moments the betas are fp32: 0.999 is off by up to
        # 2^-25, so 1 - 0.999 by 2^-25 / 0.001 = 3.0e-5 of itself, the root by half of that, and lr = 0.5 times it is 7.5e-6;
        # 0.9 adds 0.5 x 2^-25 / 0.1 = 1.5e-7
        atol = 2 ** -20 + (7.7e-6 if moments == "fp32" else 0.0)
        for p, w, s in zip(params, was, signs):
            np.testing.assert_allclose(p.detach().cpu(), (w - 0.5 * s).cpu(), rtol=2 ** -20, atol=atol)


@pytest.mark.parametrize("moments", ["fp32", "bf16", "int8"])
@pytest.mark.parametrize("master", [False, True])
def test_state_dict_round_trip(moments, master):
    gen = torch.Generator(device=DEV).manual_seed(8)

    def make():
        g = torch.Generator(device=DEV).manual_seed(9)
        return [torch.nn.Parameter(torch.randn(n, generator=g, device=DEV).to(torch.bfloat16)) for n in (700, 33)]

    a = make()
    one = FusedAdamW(a, moments=moments, master_weights=master, stochastic_rounding=False, **HP)
    grads = [[torch.randn(p.shape, generator=gen, device=DEV).to(torch.bfloat16) for p in a] for _ in range(3)]

    def step(opt, params, gs):
        for p, g in zip(params, gs):
            p.grad = g.clone()
        opt.step()

    step(one, a, grads[0])
    step(one, a, grads[1])
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    two = FusedAdamW(b, moments=moments, master_weights=master, stochastic_rounding=False, **HP)
    two.load_state_dict(one.state_dict())
    step(one, a, grads[2])
    step(two, b, grads[2])
    for p, q in zip(a, b):
        assert torch.equal(p.detach(), q.detach())
        for key, value in one.state[p].items():
            got = two.state[q][key]
            if torch.is_tensor(value):
                assert got.dtype == value.dtype and torch.equal(got, value) and got.data_ptr() != value.data_ptr()
            else:
                assert got == value


def test_another_stream_and_a_graph():
    gen = torch.Generator(device=DEV).manual_seed(10)
    n = 3000
    ps = [torch.nn.Parameter(torch.randn(n, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)) for _ in range(2)]
    opts = [FusedAdamW([p], moments="int8", **HP) for p in ps]
    g = torch.randn(n, generator=gen, device=DEV)
    for p in ps:
        p.main_grad = torch.zeros(n, device=DEV)
    side = torch.cuda.Stream()
    for p, o in zip(ps, opts):  # a first step makes the state; the second on another stream
        p.main_grad.copy_(g)
        o.step()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ps[0].main_grad.copy_(g)
        opts[0].step()
    torch.cuda.current_stream().wait_stream(side)
    ps[1].main_grad.copy_(g)
    opts[1].step()
    torch.cuda.synchronize()
    assert torch.equal(ps[0].detach(), ps[1].detach())
    # a captured call replays its own numbers; here the same as an eager call's of the third step
    st = opts[0].state[ps[0]]
    b1, b2 = HP["betas"]
    row = adam_row(ps[0].data_ptr(), ps[0].main_grad.data_ptr(), st["m"].data_ptr(), st["v"].data_ptr(), 0,
                   st["m_scale"].data_ptr(), st["v_scale"].data_ptr(), n, 0, 1 - b1 ** 3, 1 - b2 ** 3)

    def call():
        HipBackend.get().adam_many(ps[0].device, [row], torch.float32, torch.float32, torch.int8, HP["lr"], b1, b2,
                                   HP["eps"], HP["weight_decay"], clear=True)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for _ in range(3):
        ps[0].main_grad.copy_(g)
        ps[1].main_grad.copy_(g)
        graph.replay()
        opts[1].state[ps[1]]["step"] = 2
        opts[1].step()
        torch.cuda.synchronize()
        assert torch.equal(ps[0].detach(), ps[1].detach()) and not ps[0].main_grad.any()


def test_a_tensor_past_32_bits_of_bytes():
    """2^31 + 5 elements of bf16 parameters with 8-bit moments: 4.3 GB of parameters, offsets past 32 bits."""
    n = 2 ** 31 + 5
    p = torch.nn.Parameter(torch.zeros(n, device=DEV, dtype=torch.bfloat16))
    p.grad = torch.full((n,), 2.0, device=DEV, dtype=torch.bfloat16)
    p.grad[-3] = -2.0
    opt = FusedAdamW([p], moments="int8", lr=0.5, stochastic_rounding=False)
    opt.step()
    st = opt.state[p]
    assert p.detach()[-3] == 0.5 and p.detach()[-1] == -0.5 and p.detach()[0] == -0.5
    assert st["m"][-3] == -127 and bool((st["v"][-5:] == 255).all()) and bool((st["v"][:5] == 255).all())
    assert int((p.detach() == -0.5).sum()) == n - 1
