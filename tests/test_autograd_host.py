"""The autograd functions around the kernels, on the CPU with a backend in plain torch."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

from granulelayer_amd import LevelSpec, PhysicalPlan, PoolingConfig
from granulelayer_amd.autograd import Level1Runtime, SemanticPoolFunction, SparsePoolFunction
from granulelayer_amd.layout import SparseLayout, init_parameters


class _Sums:
    """pre = the input's sum (its statistics depend on the input), gradients of that; every forward's input and
    every backward's input and statistics are noted.  Eight bits are whole numbers here."""

    def __init__(self):
        self.forwards, self.backwards = [], []

    def forward(self, rt, x, w, b, track_ids=False):
        self.forwards.append(x.clone())
        pre = x.float().sum(1, keepdim=True).expand(-1, rt.units.U).contiguous()
        return {"pre": pre, "L2": 2 * pre}

    def backward(self, rt, x, w, b, g_pre, stats, dw_buf, db_buf):
        self.backwards.append((x.clone(), {k: v.clone() for k, v in stats.items()}))
        dw_buf += 1
        db_buf += 1
        return g_pre.sum(1, keepdim=True).expand_as(x).contiguous()

    def pack8(self, x):
        return x.round(), torch.zeros(len(x), 1)

    def unpack8(self, q, e, cols, dtype):
        assert q.shape[1] == cols
        return q.to(dtype)


def _layer(pooling, activation_checkpoint="exact"):
    cfg = PoolingConfig.parse(pooling)
    L = SparseLayout(24, 512, 4, 8, 8, False)
    idx, w, b = init_parameters(L, "cpu")
    be = _Sums()
    rt = Level1Runtime(L, idx, cfg.levels[0], PhysicalPlan(), cfg.levels[0].neurons_per_shard, backend=be)
    rt.activation_checkpoint = activation_checkpoint
    w.requires_grad_(True), b.requires_grad_(True)

    def call(x):
        if cfg.is_semantic_hierarchy:
            return SemanticPoolFunction.apply(x, w, b, rt, cfg, "minimal_stats", torch.float32, [])
        return SparsePoolFunction.apply(x, w, b, rt, "minimal_stats", torch.float32)

    return call, be, (w, b)


TWO = dict(levels=[dict(type="mean", neurons_per_shard=32), dict(type="mean")])


@pytest.mark.parametrize("eight", ["exact", "int8"])
@pytest.mark.parametrize("pooling", ["mean", TWO], ids=["one level", "two levels"])
def test_under_activation_checkpointing(pooling, eight):
    """torch.utils.checkpoint without re-entrant autograd lets a backward read its saved tensors once."""
    call, _, params = _layer(pooling, eight)
    x = torch.randn(5, 24, requires_grad=True)
    want = torch.autograd.grad(call(x).sum(), (x, *params))
    got = torch.autograd.grad(checkpoint(call, x, use_reentrant=False).sum(), (x, *params))
    for g, t in zip(got, want):
        assert torch.equal(g, t)


LEVELS = {"lme": dict(type="logmeanexp", temperature=0.05), "softmax": dict(type="softmax_weighted"),
          "power": dict(type="power_mean", p=4.0)}


@pytest.mark.parametrize("two", [False, True], ids=["one level", "two levels"])
@pytest.mark.parametrize("eight", ["exact", "int8"])
@pytest.mark.parametrize("level", LEVELS.values(), ids=LEVELS.keys())
def test_normalisers_and_terms_are_of_one_input(level, eight, two):
    """What a smooth pool's backward divides by was summed over the input that its terms are recomputed from."""
    pooling = dict(levels=[dict(level, neurons_per_shard=32), dict(type="sum")], level1_checkpoint="save") if two else level
    call, be, _ = _layer(pooling, eight)
    x = torch.randn(5, 24, requires_grad=True)
    call(x).sum().backward()
    (xb, stats), = be.backwards
    assert torch.equal(xb, x.detach().round() if eight == "int8" else x.detach())
    assert torch.equal(stats["pre"], xb.sum(1, keepdim=True).expand_as(stats["pre"]))
    if "L2" in stats:
        assert torch.equal(stats["L2"], 2 * stats["pre"])
    assert len(be.forwards) == (2 if eight == "int8" else 1)
