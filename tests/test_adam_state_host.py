"""What FusedAdamW keeps and loads, CPU side: state dicts and their hooks, and nothing alive that its state has let go."""
import gc
import weakref

import pytest
import torch

from granulelayer_amd import FusedAdamW, optim


def _loaded(moments="fp32", dtype=torch.bfloat16):
    p = torch.nn.Parameter(torch.zeros(300, dtype=dtype))
    opt = FusedAdamW([p], moments=moments, master_weights=True)
    st = opt._new_state(p)
    for t in st.values():
        if torch.is_tensor(t):
            t.copy_((torch.arange(t.numel()) % 100 + 1) / (128.0 if t.is_floating_point() else 1))
    opt.state[p] = dict(st, step=7)
    return opt


def _fresh(moments="fp32", dtype=torch.bfloat16):
    p = torch.nn.Parameter(torch.zeros(300, dtype=dtype))
    return p, FusedAdamW([p], moments=moments, master_weights=True)


def test_tensors_keep_their_types():
    for moments in ("fp32", "bf16", "int8"):
        source = _loaded(moments)
        want = next(iter(source.state.values()))
        p, opt = _fresh(moments)
        opt.load_state_dict(source.state_dict())
        for key, value in want.items():
            got = opt.state[p][key]
            if torch.is_tensor(value):
                assert got.dtype == value.dtype and torch.equal(got, value) and got.data_ptr() != value.data_ptr()
            else:
                assert got == value


def test_a_pre_hook_that_returns_another_dict():
    source = _loaded()
    p, opt = _fresh()

    def five(optimizer, state_dict):
        state = {i: {k: 5 * v if k == "m" else v for k, v in st.items()} for i, st in state_dict["state"].items()}
        return dict(state_dict, state=state)

    opt.register_load_state_dict_pre_hook(five)
    opt.load_state_dict(source.state_dict())
    want = next(iter(source.state.values()))
    got = opt.state[p]
    assert torch.equal(got["m"], 5 * want["m"]) and torch.equal(got["v"], want["v"]) and got["m"].dtype == torch.float32


def test_a_post_hook_sees_and_changes_the_loaded_state():
    source = _loaded()
    p, opt = _fresh()
    seen = []

    def three(optimizer):
        st = optimizer.state[p]
        seen.append((st["m"].dtype, st["m"].clone()))
        st["m"] = 3 * st["m"]

    opt.register_load_state_dict_post_hook(three)
    opt.load_state_dict(source.state_dict())
    want = next(iter(source.state.values()))["m"]
    assert seen[0][0] == torch.float32 and torch.equal(seen[0][1], want)
    assert torch.equal(opt.state[p]["m"], 3 * want)


def test_hooks_of_a_load_do_not_stay():
    p, opt = _fresh()
    calls = []
    opt.register_load_state_dict_pre_hook(lambda *_: calls.append("pre"))
    opt.register_load_state_dict_post_hook(lambda *_: calls.append("post"))
    for _ in range(2):
        opt.load_state_dict(_loaded().state_dict())
    try:
        opt.load_state_dict({"state": {}, "param_groups": []})
    except ValueError:
        pass
    opt.load_state_dict(_loaded().state_dict())
    assert calls == ["pre", "post"] * 2 + ["pre"] + ["pre", "post"]
    assert opt.state[p]["step"] == 7


class _Nothing:
    def adam_many(self, *args, **kw):
        pass


nothing = _Nothing()


def _stepped(monkeypatch, moments, dtype=torch.bfloat16, master=True):
    monkeypatch.setattr(optim, "backend_for", lambda device: nothing)
    p = torch.nn.Parameter(torch.zeros(300, dtype=dtype))
    opt = FusedAdamW([p], moments=moments, master_weights=master)
    for _ in range(2):
        p.grad = torch.zeros_like(p)
        opt.step()
    return p, opt


@pytest.mark.parametrize("moments", ["fp32", "bf16", "int8"])
def test_a_state_that_is_taken_away_is_freed(monkeypatch, moments):
    p, opt = _stepped(monkeypatch, moments)
    kept = [weakref.ref(t) for t in opt.state[p].values() if torch.is_tensor(t)]
    assert len(kept) == (5 if moments == "int8" else 3) and all(r() is not None for r in kept)
    opt.state.clear()
    gc.collect()
    assert all(r() is None for r in kept)


def test_a_state_that_is_replaced_is_freed(monkeypatch):
    p, opt = _stepped(monkeypatch, "fp32")
    kept = {k: weakref.ref(t) for k, t in opt.state[p].items() if torch.is_tensor(t)}
    for k in kept:
        opt.state[p][k] = opt.state[p][k].clone()
    gc.collect()
    assert all(r() is None for r in kept.values())


def test_a_parameter_that_is_taken_away_is_freed(monkeypatch):
    p, opt = _stepped(monkeypatch, "fp32")
    kept = weakref.ref(p)
    opt.param_groups.clear()
    opt.state.clear()
    del p
    gc.collect()
    assert kept() is None


@pytest.mark.parametrize("moments", ["fp32", "int8"])
def test_a_changed_state_is_looked_at_again(monkeypatch, moments):
    """Whatever changes between two steps is what the second works on."""
    rows = []
    monkeypatch.setattr(optim, "_ROW", lambda *fields: rows.append(fields) or fields)
    p, opt = _stepped(monkeypatch, moments, master=False)
    fields = dict(m=2, v=3, m_scale=5, v_scale=6)

    def step():
        p.grad = torch.zeros_like(p)
        opt.step()
        for key, i in fields.items():
            t = opt.state[p].get(key)
            assert rows[-1][i] == (0 if t is None else t.data_ptr())

    step()
    for key in fields:
        if key in opt.state[p]:
            was = opt.state[p][key]  # alive, so that the new one is elsewhere
            opt.state[p][key] = was.clone()
            step()
            opt.state[p][key].data = was.data.clone()
            step()
            opt.state[p][key] = torch.zeros(7, dtype=was.dtype)
            with pytest.raises(ValueError):
                step()
            opt.state[p][key] = was
            step()
    opt.state[p]["master"] = torch.zeros(300)
    step()
    assert rows[-1][4] == opt.state[p]["master"].data_ptr()
    del opt.state[p]["master"]
    step()
    assert rows[-1][4] == 0
