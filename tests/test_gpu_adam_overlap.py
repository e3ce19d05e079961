"""FusedAdamW over parameters and gradient buffers that meet partly in memory: as one step after the other."""
import pytest
import torch

from conftest import gpu_available

from granulelayer_amd import FusedAdamW

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a ROCm GPU")]
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("moments", ["fp32", "bf16"])
@pytest.mark.parametrize("kind", ["parameters", "main_grads", "chain"])
def test_tensors_that_meet_partly_step_one_after_the_other(dtype, moments, kind):
    n = 300_000
    gen = torch.Generator(device=DEV).manual_seed(4)
    data = torch.randn(3 * n, device=DEV, generator=gen).to(dtype)
    grads = torch.randn(3 * n, device=DEV, generator=gen)

    def make(together):
        buf, main = data.clone(), grads.clone()
        if kind == "main_grads":
            parts, mains = [(0, n), (n, 2 * n)], [(0, n), (n // 3, n // 3 + n)]
        else:
            parts, mains = [(0, n), (n - 1000, 2 * n - 1000)], [(0, n), (n, 2 * n)]
        if kind == "chain":
            parts.append((2 * n - 2000, 3 * n - 2000))
            mains.append((2 * n, 3 * n))
        ps = []
        for (a, b), (c, d) in zip(parts, mains):
            ps.append(torch.nn.Parameter(buf[a:b]))
            ps[-1].main_grad = main[c:d]
        groups = [dict(params=ps)] if together else [dict(params=[p]) for p in ps]
        return buf, main, FusedAdamW(groups, lr=1e-2, moments=moments, weight_decay=0.1), ps

    got, main, one, ps = make(True)
    want, _, two, qs = make(False)
    for _ in range(3):
        main.copy_(grads)
        two_main = qs[0].main_grad._base
        two_main.copy_(grads)
        one.step()
        two.step()
        assert torch.equal(got, want) and torch.equal(main, two_main)
    for p, q in zip(ps, qs):
        assert torch.equal(one.state[p]["m"], two.state[q]["m"]) and torch.equal(one.state[p]["v"], two.state[q]["v"])
