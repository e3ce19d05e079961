"""Cross entropy of a dense head, CPU side: what the function, the module and the C entry points refuse before any device
use, and how workspaces follow the budget."""
import ctypes

import pytest
import torch

from granulelayer_amd import DenseCrossEntropy, dense_cross_entropy
from granulelayer_amd import _native as N


def test_arguments_are_checked():
    x, w, t, b = torch.zeros(4, 8), torch.zeros(5, 8), torch.zeros(4, dtype=torch.int64), torch.zeros(5)

    def call(x=x, w=w, t=t, b=b, **kw):
        return dense_cross_entropy(x, w, t, b, **kw)

    for bad in (dict(reduction="avg"), dict(w=torch.zeros(5)), dict(w=torch.zeros(0, 8)), dict(x=torch.zeros(4, 7)),
                dict(x=torch.zeros(())), dict(t=torch.zeros(3, dtype=torch.int64)), dict(t=t[:, None]), dict(b=torch.zeros(4)),
                dict(workspace_budget=0), dict(workspace_budget=1.5), dict(workspace_budget=True),
                dict(w=torch.zeros(5, 8, device="meta"))):
        with pytest.raises(ValueError):
            call(**bad)
    for bad in (dict(x=x.bfloat16()), dict(x=x.double(), w=w.double(), b=b.double()), dict(t=t.float()), dict(b=b.bfloat16())):
        with pytest.raises(TypeError):
            call(**bad)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        call()


def test_module():
    m = DenseCrossEntropy(6, 9, bias=True, dtype=torch.float32, seed=1)
    assert m.weight.shape == (9, 6) and m.bias.shape == (9,) and not m.bias.any()
    assert torch.equal(m.weight, DenseCrossEntropy(6, 9, dtype=torch.float32, seed=1).weight)
    table = torch.nn.Parameter(torch.randn(9, 6).bfloat16())
    assert DenseCrossEntropy(6, 9, weight=table).weight is table
    for bad in (dict(input_dim=0, classes=4), dict(input_dim=4, classes=0), dict(input_dim=4, classes=4, reduction="x"),
                dict(input_dim=6, classes=8, weight=table)):
        with pytest.raises(ValueError):
            DenseCrossEntropy(**bad)
    with pytest.raises(NotImplementedError):
        DenseCrossEntropy(4, 4, dtype=torch.float16)


def test_the_c_entry_points_refuse():
    lib = N.library()
    out = ctypes.c_size_t()
    base = dict(X=4096, sx=64, W=4096, sw=64, target=4096, M=300, N=1000, K=64, dtype=1, reduction=1)

    def fwd(query=False, **kw):
        a = N.GlCeArgs(**{**base, "loss": 4096, **kw})
        return lib.lib.gl_ce_fwd_workspace(ctypes.byref(a), ctypes.byref(out)) if query else lib.lib.gl_ce_fwd(ctypes.byref(a), None)

    def bwd(query=False, **kw):
        a = N.GlCeBwdArgs(**{**base, "kept": 4096, "dloss": 4096, "dX": 4096, "dW": 4096, "db": 4096, "g_dtype": 1, **kw})
        return lib.lib.gl_ce_bwd_workspace(ctypes.byref(a), ctypes.byref(out)) if query else lib.lib.gl_ce_bwd(ctypes.byref(a), None)

    assert lib.lib.gl_ce_fwd(None, None) == -1 and lib.lib.gl_ce_bwd(None, None) == -1
    for f in (fwd, bwd):
        assert f() == -3 and f(ws=16, ws_bytes=1 << 40) == -1  # too little; off 256 bytes
        assert f(M=0) == 0 and f(True, M=0) == 0 and out.value == 0
        assert f(True) == 0 and out.value > 0
        for bad in (dict(M=-1), dict(N=0), dict(K=0), dict(X=0), dict(W=0), dict(target=0), dict(target=4100), dict(sx=63),
                    dict(sw=63), dict(X=4097), dict(W=4097), dict(bias=4097), dict(reduction=3), dict(reduction=-1)):
            assert f(**bad) == -1 and f(True, **bad) == -1, bad
        for bad in (dict(N=(1 << 20) + 1), dict(K=(1 << 20) + 1), dict(M=(1 << 24) + 1), dict(dtype=2)):
            assert f(**bad) == -2 and f(True, **bad) == -2, bad
    assert fwd(loss=0) == -1 and fwd(loss=4098) == -1 and fwd(kept=4098) == -1
    for bad in (dict(kept=0), dict(dloss=0), dict(kept=4098), dict(dloss=4098), dict(sdl=-1), dict(dX=4097), dict(dW=4097),
                dict(db=4097), dict(accumulate=1)):
        assert bwd(**bad) == -1, bad
    assert bwd(g_dtype=2) == -2
    assert bwd(dX=0, dW=0, db=0) == 0


def test_workspace_follows_the_budget():
    lib = N.library()
    out = ctypes.c_size_t()

    def need(M, classes, budget, dtype=1, K=4096, exps=0):
        a = N.GlCeBwdArgs(X=4096, sx=K, W=4096, sw=K, target=4096, M=M, N=classes, K=K, dtype=dtype, reduction=1, kept=4096,
                          dloss=4096, dX=4096, dW=4096, g_dtype=dtype, piece_bytes=budget, exps=exps)
        assert lib.lib.gl_ce_bwd_workspace(ctypes.byref(a), ctypes.byref(out)) == 0
        return out.value

    M, V = 8192, 131072
    rest = M * 4096 * 2 + M * 16 + 256 + M * 4096 * 4  # x, the rows, their factor, dx in fp32 over the pieces
    for budget in (64 << 20, 256 << 20, 1 << 30):
        assert budget * 0.9 < need(M, V, budget) - rest <= budget + 256 * M * 2
    assert need(M, V, 0) == need(M, V, 4 << 30) and need(2 * M, 2 * V, 0) == need(2 * M, 2 * V, 4 << 30) > need(2 * M, 2 * V, 1 << 30)
    # pieces' gradients at the logits have the place of the kept exponentials
    assert need(M, V, 1 << 30, exps=4096) - rest <= 64 << 20
    assert need(M, V, 1) - rest <= 256 * M * 2 + (64 << 20)  # 256 classes at least (and their products' partial sums)


@pytest.mark.parametrize("dtype", [0, 1])
def test_pieces_stay_within_the_budget(dtype):
    """A piece's place, given as that of the exponentials kept for it: rows of whole 8 columns, and 4 bytes of every 64."""
    lib = N.library()
    out = ctypes.c_size_t()
    es = 4 >> dtype

    def place(M, classes, budget):
        a = N.GlCeArgs(X=4096, sx=1024, W=4096, sw=1024, target=4096, M=M, N=classes, K=1024, dtype=dtype, reduction=1,
                       loss=4096, kept=4096, piece_bytes=budget)
        assert lib.lib.gl_ce_exps_bytes(ctypes.byref(a), ctypes.byref(out)) == 0
        return out.value

    def bytes_of(M, columns):
        up = lambda n: -(-n // 256) * 256  # noqa: E731
        return up(M * (-(-columns // 8) * 8) * es) + up(M * -(-columns // 64) * 4)

    for M, classes in ((4096, 50000), (777, 12553), (1, 300), (129, 257), (6_000_000, 50000)):
        for columns in (1, 100, 255, 256, 257, 300, 511, 513, 1000, 12552, 12553, 12559, 12560, 30000, 49999, 50000):
            got = place(M, classes, M * es * columns)
            assert got <= max(bytes_of(M, columns // 8 * 8), bytes_of(M, 256)), (M, classes, columns)
            if columns >= -(-classes // 8) * 8:
                assert got == bytes_of(M, classes)
        for budget in (0, 1 << 20, (1 << 30) + 12345):
            most = (budget or 4 << 30) // (M * es)
            assert place(M, classes, budget) <= max(bytes_of(M, most // 8 * 8), bytes_of(M, 256))
