"""Cross entropy of a dense head on the GPU: logits that overflow, budgets below the least piece."""
import pytest
import torch

from conftest import gpu_available

from test_gpu_cross_entropy import compare, inputs, run

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a ROCm GPU")]
DEV = "cuda"
BF, F = torch.bfloat16, torch.float32


@pytest.mark.parametrize("K", [48, 520])  # exponentials made again, and kept
@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("M", [100, 600])
def test_a_target_whose_logit_overflows(M, dtype, K):
    """log sum exp - z is infinity less infinity, not 0, where only the target's logit is infinite."""
    t = inputs(M, K, 300, dtype, ignored=0.0)
    t["w"][11] = 2.0 ** 60
    t["target"][t["target"] == 11] = 12
    t["target"][7] = 11
    clean = run(t, "none")[1]
    t["x"][7] = 2.0 ** 70  # others' logits of the row are about 2^70
    got = run(t, "none")[1]
    good = torch.arange(M, device=DEV) != 7
    assert torch.isnan(got["loss"][7]) and torch.isnan(got["dx"][7]).all()
    assert torch.equal(got["loss"][good], clean["loss"][good]) and torch.equal(got["dx"][good], clean["dx"][good])
    assert torch.isnan(got["dw"]).all() and torch.isnan(got["db"]).all()
    for reduction in ("mean", "sum"):
        got = run(t, reduction)[1]
        assert torch.isnan(got["loss"]) and torch.isnan(got["dx"][7]).all() and torch.isfinite(got["dx"][good]).all()


@pytest.mark.parametrize("K", [48, 520])
@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("M", [100, 600])
def test_a_target_whose_bias_is_infinite(M, dtype, K):
    t = inputs(M, K, 300, dtype, ignored=0.0)
    t["b"][11] = float("inf")
    t["target"][::2] = 11
    got = run(t, "none")[1]
    assert torch.isnan(got["loss"]).all() and torch.isnan(got["dx"]).all()
    assert torch.isnan(got["dw"]).all() and torch.isnan(got["db"]).all()


@pytest.mark.parametrize("M", [3, 300])
def test_the_only_class(M):
    """One class: the loss is 0 and so are the gradients, unless its logit is no number."""
    t = inputs(M, 64, 1, F, ignored=0.0)
    got = run(t, "none")[1]
    assert not got["loss"].any() and not got["dx"].any() and not got["dw"].any() and not got["db"].any()
    for b in (float("inf"), float("-inf"), float("nan")):
        t["b"][0] = b
        got = run(t, "none")[1]
        assert torch.isnan(got["loss"]).all() and torch.isnan(got["dx"]).all()


@pytest.mark.parametrize("K", [48, 520])
@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("M", [100, 700])
@pytest.mark.parametrize("N", [5, 100, 255, 256, 300])
def test_a_budget_of_less_than_the_least_piece(N, M, dtype, K):
    """Fewer classes than a piece has at least, and a budget of fewer still."""
    t = inputs(M, K, N, dtype)
    whole = compare(t, "mean")
    for budget in (1, M * (N // 2)):
        got = compare(t, "mean", budget=budget)
        if N <= 256:  # the same single piece
            assert all(torch.equal(got[k], whole[k]) for k in whole)
