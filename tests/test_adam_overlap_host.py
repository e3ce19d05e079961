"""FusedAdamW over tensors that meet in memory, CPU side: which of them go into one launch."""
import random

import pytest
import torch

from granulelayer_amd import FusedAdamW, optim


class Recorder:
    """Takes the place of the backend; keeps the addresses (parameter, gradient) and seeds of every call."""

    def __init__(self, monkeypatch):
        self.calls = []
        monkeypatch.setattr(optim, "_ROW", lambda *fields: fields)
        monkeypatch.setattr(optim, "backend_for", lambda device: self)

    def adam_many(self, device, rows, *args, **kw):
        self.calls.append([(r[0], r[1], r[8]) for r in rows])


def _param(data, main=None, grad=None):
    p = torch.nn.Parameter(data)
    if main is not None:
        p.main_grad = main
    else:
        p.grad = torch.zeros_like(p) if grad is None else grad
    return p


def _step(monkeypatch, params, **kw):
    rec = Recorder(monkeypatch)
    opt = FusedAdamW(params, **kw)
    opt.step()
    at = [p.data_ptr() for p in params]
    return [[at.index(a) for a, _, _ in call] for call in rec.calls], rec, opt


def test_disjoint_parts_of_one_buffer_share_a_launch(monkeypatch):
    buf, main = torch.zeros(1000), torch.zeros(1000)
    parts = [(600, 1000), (0, 400), (400, 600)]
    calls, _, _ = _step(monkeypatch, [_param(buf[a:b], main[a:b]) for a, b in parts])
    assert calls == [[0, 1, 2]]


def test_parameters_that_meet_partly(monkeypatch):
    buf, other = torch.zeros(1000), torch.zeros(50)
    calls, _, opt = _step(monkeypatch, [_param(buf[:600]), _param(buf[400:]), _param(other)])
    assert calls == [[0, 2], [1]]
    assert all(st["step"] == 1 for st in opt.state.values())


def test_main_grads_that_meet_partly(monkeypatch):
    main = torch.zeros(1000)
    calls, _, _ = _step(monkeypatch, [_param(torch.zeros(600), main[400:]), _param(torch.zeros(500), main[:500])])
    assert calls == [[0], [1]]


def test_order_over_a_chain(monkeypatch):
    """The third meets only the second, which comes after the first."""
    buf = torch.zeros(1000)
    calls, _, _ = _step(monkeypatch, [_param(buf[:400]), _param(buf[300:700]), _param(buf[600:])])
    assert calls == [[0], [1], [2]]


@pytest.mark.parametrize("first", ["clears", "reads"])
def test_a_gradient_that_is_anothers_main_grad(monkeypatch, first):
    g = torch.zeros(300)
    ps = [_param(torch.zeros(300), g), _param(torch.zeros(300), grad=g)]
    calls, _, _ = _step(monkeypatch, ps if first == "clears" else ps[::-1])
    assert calls == [[0], [1]]


def test_a_gradient_that_several_read(monkeypatch):
    g = torch.zeros(300)
    calls, _, _ = _step(monkeypatch, [_param(torch.zeros(300), grad=g) for _ in range(3)])
    assert calls == [[0, 1, 2]]


def test_seeds_follow_the_parameters_order(monkeypatch):
    """Stochastic rounding's noise does not depend on which tensors meet."""
    buf = torch.zeros(1000, dtype=torch.bfloat16)
    _, rec, opt = _step(monkeypatch, [_param(buf[:600]), _param(buf[400:]), _param(torch.zeros(9, dtype=torch.bfloat16))])
    assert [[s for _, _, s in call] for call in rec.calls] == [[1, 3], [2]] and opt._seed == 3


@pytest.mark.filterwarnings("ignore:optimizer contains a parameter group with duplicate")
@pytest.mark.parametrize("main", [False, True])
def test_a_parameter_that_is_there_twice(monkeypatch, main):
    p = _param(torch.zeros(9), torch.zeros(9) if main else None)
    calls, _, opt = _step(monkeypatch, [p, p])
    assert calls == ([[0], [0]] if main else [[0]]) and opt.state[p]["step"] == opt._seed == len(calls)


def test_a_state_that_does_not_fit_stops_all_turns(monkeypatch):
    rec = Recorder(monkeypatch)
    buf = torch.zeros(1000)
    ps = [_param(buf[:600]), _param(buf[400:])]
    opt = FusedAdamW(ps)
    opt.state[ps[1]] = dict(opt._new_state(ps[1]), m=torch.zeros(3, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        opt.step()
    assert not rec.calls


def test_turns_against_pairs_looked_at_one_by_one():
    rng = random.Random(1)
    for _ in range(200):
        todo = []
        for k in range(rng.randint(1, 9)):
            n, m = rng.choice([0, 1, 5, 20]), rng.random() < 0.5
            p, g = torch.empty(n, device="meta"), torch.empty(n, device="meta")
            todo.append((p, g, torch.float32, m, rng.randint(0, 150), rng.randint(1000, 1100), n, p.dtype, -1))
        spans = [[(t[4], t[4] + 4 * t[0].numel(), True), (t[5], t[5] + 4 * t[0].numel(), t[3])] if t[0].numel() else []
                 for t in todo]

        def meet(a, b):
            return any(x < f and e < y and (w or v) for x, y, w in spans[a] for e, f, v in spans[b])

        turns = optim._in_turn(todo)
        of = {id(t[0]): i for i, (turn, _) in enumerate(turns) for t in turn}
        assert all(todo[k] is t for turn, numbers in turns for t, k in zip(turn, numbers))
        assert sorted(k for _, numbers in turns for k in numbers) == list(range(len(todo)))
        for b in range(len(todo)):
            earlier = [of[id(todo[a][0])] for a in range(b) if meet(a, b)]
            assert of[id(todo[b][0])] == 1 + max(earlier, default=-1)
        apart = sorted((x, y) for s in spans for x, y, _ in s)
        starts, ends = [x for s in spans for x, _, _ in s], [y for s in spans for _, y, _ in s]
        assert optim._disjoint(starts, ends) == all(a[1] <= b[0] for a, b in zip(apart, apart[1:]))
