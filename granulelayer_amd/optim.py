"""Fused AdamW for the layer parameters, mirroring sparse_pooling/optim.py (FusedAdamW).

Reads the fp32 ``main_grad`` buffers written by the fused backward (zeroed in the same streaming pass) or, of parameters
without one, ``.grad`` in its own type, and updates the tensors of a parameter group together: a launch of the HIP
kernel takes 38 of them (gl_adam).
Semantics are dense AdamW for every element (optim.py:1-15): m = b1 m + (1-b1) g,
v = b2 v + (1-b2) g^2, p = p (1 - lr wd) - lr (m / bc1) / (sqrt(v / bc2) + eps), bc_i = 1 - b_i^t.

Moments are fp32 (``moments="fp32"``), bf16 (``"bf16"``, the reference default) or 8 bits (``"int8"``, no
counterpart in the reference): blocks of 256 neighbouring elements of a tensor share two fp32 scales,

    m = s c |c|       c from -127 to 127    s = max |m| / 127^2
    v = (r c^2)^2     c from 0 to 255       r = sqrt(max v) / 255^2

with c one of a value's two neighbours, drawn so that it is kept on average, and 1 at least where v > 0: a step takes
1 - b2 off v, less than codes are apart, so the nearest one would stay where it is.  The draw is a hash of the element's place,
parameter, moments and step (and, as the rounding of bf16 parameters, of the seed): equal runs are equal.
``stochastic_rounding=False`` takes the nearest all the same: sqrt(v) is then 1.1 of itself after 2,000 steps of like
gradients and b2 = 0.999, and many times too large a few thousand steps after gradients got small.  A step takes the new
moments before they are put into 8 bits; a block with an infinity or a NaN in its moments is NaN from then on.  The state of
a parameter has codes ``m`` (int8) and ``v`` (uint8) and scales ``m_scale`` and ``v_scale``; ``moment_values`` gives what they
stand for.

Parameters are fp32, or bf16 with the reference's three variants (optim.py:5-9, 52-62): an fp32 master copy
in the optimizer state (``master_weights=True``; the update runs on it and the parameter gets its
nearest-even rounding), stochastic rounding (the default without masters: noise from Triton's
``tl.randint(seed, element)`` below the bf16 cut, the seed counting tensors as the reference's
``_seed`` does), or nearest-even rounding (``stochastic_rounding=False``).

A step captured into a graph replays the learning rate, the bias corrections and the seeds that it was captured with.  A
first step makes the state, so it comes before the capture.
"""
from __future__ import annotations

from operator import le
from typing import Iterable, List, Tuple
from weakref import ref

import torch

from .backend import adam_row as _ROW, backend_for

_MOMENTS = {"bf16": torch.bfloat16, "fp32": torch.float32, "int8": torch.int8}
_TYPES = (torch.float32, torch.bfloat16)
_BLOCK = 256  # elements of a tensor that share the scales of 8-bit moments


_EXTRA = ("master", "m_scale", "v_scale")  # what the state of some kinds has beside m and v


def _as_known(st, refs, at) -> bool:
    """Whether a state's further tensors are those of the references, and where they were."""
    for key, ref, a in zip(_EXTRA, refs, at):
        t = st.get(key)
        if (t is not None) if ref is None else (t is None or t is not ref() or t.data_ptr() != a):
            return False
    return True


def _disjoint(starts, ends) -> bool:
    """Whether of ranges of bytes, given by their starts and their ends in any order, no two meet."""
    starts, ends = sorted(starts), sorted(ends)
    return all(map(le, ends, starts[1:]))


def _in_turn(todo):
    """Of tensors to step of which some meet in memory: lists of those that may step at once, with their numbers in the order
    of all.  A tensor comes after all earlier ones that write what it touches, or touch what it writes."""
    kept, seen = [], set()
    for t in todo:
        if t[3] or id(t[0]) not in seen:  # (there twice: its first step uses up its .grad)
            seen.add(id(t[0]))
            kept.append(t)
    spans = []
    for k, (p, g, _, main, at, g_at, n, *_) in enumerate(kept):
        if n:
            spans.append((at, at + n * p.element_size(), k, True))
            spans.append((g_at, g_at + n * g.element_size(), k, main))
    meets, writers, readers = [[] for _ in kept], [], []
    for start, end, k, written in sorted(spans):
        writers = [s for s in writers if s[0] > start]
        readers = [s for s in readers if s[0] > start] if written else readers
        for _, j in writers + readers if written else writers:
            if j != k:
                meets[max(j, k)].append(min(j, k))
        (writers if written else readers).append((end, k))
    turns, turn = [], []
    for k, (t, earlier) in enumerate(zip(kept, meets)):
        turn.append(1 + max((turn[j] for j in earlier), default=-1))
        if turn[-1] == len(turns):
            turns.append(([], []))
        turns[turn[-1]][0].append(t)
        turns[turn[-1]][1].append(k)
    return turns


class FusedAdamW(torch.optim.Optimizer):
    def __init__(self, params: Iterable[torch.nn.Parameter], lr=1e-3, betas=(0.9, 0.999), eps=1e-8,
                 weight_decay=0.0, moments: str = "bf16", master_weights: bool = False,
                 stochastic_rounding: bool = True):
        if moments not in _MOMENTS:
            raise ValueError("moments must be 'bf16', 'fp32' or 'int8'")
        defaults = dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay)
        super().__init__(params, defaults)
        self.moments = moments
        self.master_weights = master_weights
        self.stochastic_rounding = stochastic_rounding
        self._seed = 0
        self._known, self._kinds = {}, {}

    def state_bytes(self) -> int:
        n = 0
        for st in self.state.values():
            for t in st.values():
                if torch.is_tensor(t):
                    n += t.numel() * t.element_size()
        return n

    def load_state_dict(self, state_dict):
        """As torch's, but every tensor of the state keeps its own type (torch's casts it to the parameter's).  Hooks see
        and change what they do with any optimizer: what the last pre-hook leaves is loaded, and post-hooks come last."""
        seen = []
        hooks = (self.register_load_state_dict_pre_hook(lambda _, given: seen.append(given)),
                 self.register_load_state_dict_post_hook(lambda _: self._take_tensors(seen[-1]), prepend=True))
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

    def _take_tensors(self, state_dict):
        self._known.clear()
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(ids, params):
            for key, value in state_dict["state"].get(i, {}).items():
                if torch.is_tensor(value):
                    self.state[p][key] = value.detach().to(p.device, copy=True)

    def _new_state(self, p):
        st = dict(step=0)
        if self.moments == "int8":
            st["m"] = torch.zeros(p.shape, device=p.device, dtype=torch.int8)
            st["v"] = torch.zeros(p.shape, device=p.device, dtype=torch.uint8)
            for key in ("m_scale", "v_scale"):
                st[key] = torch.zeros(-(-p.numel() // _BLOCK), device=p.device)
        else:
            for key in ("m", "v"):
                st[key] = torch.zeros(p.shape, device=p.device, dtype=_MOMENTS[self.moments])
        if self.master_weights and p.dtype != torch.float32:
            st["master"] = p.detach().float().clone()
        return st

    @staticmethod
    def _check_state(p, st):
        """The moments' type; raises where the state does not fit the parameter."""
        m, v, master = st["m"], st["v"], st.get("master")
        if m.dtype not in _MOMENTS.values() or v.dtype != (torch.uint8 if m.dtype == torch.int8 else m.dtype):
            raise TypeError(f"moments must both be float32, both bfloat16, or codes in int8 and uint8 (got {m.dtype}, {v.dtype})")
        of = [(m, p.numel()), (v, p.numel())]
        if m.dtype == torch.int8:
            for key in ("m_scale", "v_scale"):
                if st[key].dtype != torch.float32:
                    raise TypeError(f"{key} must be float32 (got {st[key].dtype})")
                of.append((st[key], -(-p.numel() // _BLOCK)))
        if master is not None:
            if p.dtype != torch.bfloat16 or master.dtype != torch.float32:
                raise TypeError("master must be a float32 copy of a bfloat16 parameter")
            of.append((master, p.numel()))
        for t, n in of:
            if t.numel() != n or t.get_device() != p.get_device() or not t.is_contiguous():
                raise ValueError("the optimizer state must be contiguous tensors of the parameter's size and device")
        return m.dtype

    def _known_state(self, p, st):
        """What a step needs of a parameter's state, checked: addresses for the next step, which looks whether the tensors
        are still these and where they were (nothing is kept alive for that)."""
        if not st:
            st.update(self._new_state(p))
        mdt = self._check_state(p, st)
        backend = backend_for(p.device)
        extra = [st.get(key) for key in _EXTRA]
        kind = (backend, p.device, p.dtype, mdt, extra[0] is not None)
        kind = self._kinds.setdefault(kind, kind)
        known = (ref(st["m"]), ref(st["v"]), st["m"].data_ptr(), st["v"].data_ptr(),
                 tuple(0 if t is None else t.data_ptr() for t in extra),
                 tuple(None if t is None else ref(t) for t in extra) if any(t is not None for t in extra) else None,
                 p.numel(), p.dtype, p.get_device(), kind)
        self._known[id(p)] = known
        return known

    @staticmethod
    def _gradient(p, g, main):
        """g as the kernel reads it, checked."""
        if p.dtype not in _TYPES:
            raise NotImplementedError(f"FusedAdamW updates fp32 or bf16 parameters (got {p.dtype})")
        if not p.is_contiguous() or (main and not g.is_contiguous()):
            raise ValueError("FusedAdamW needs contiguous parameters and gradients")
        if main:
            if g.dtype != torch.float32:
                raise TypeError("grad must be a contiguous float32 tensor")
        else:
            g = (g if g.dtype in _TYPES else g.float()).resolve_neg().contiguous()
        if g.numel() != p.numel() or g.get_device() != p.get_device():
            raise ValueError("param and grad must have the same number of elements and be on one device")
        return g

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            self._step_group(group)
        return loss

    def _step_group(self, group):
        f32, bf16 = torch.float32, torch.bfloat16
        todo, starts, ends = [], [], []
        for p in group["params"]:  # everything is checked before anything changes
            g = getattr(p, "main_grad", None)
            main = g is not None
            if not main:
                g = p.grad
                if g is None:
                    continue
            pdt, gdt, n, device = p.dtype, g.dtype, p.numel(), p.get_device()
            if (not (gdt is f32 or (gdt is bf16 and not main)) or not g.is_contiguous() or g.is_neg()
                    or not p.is_contiguous() or not (pdt is f32 or pdt is bf16)
                    or g.numel() != n or g.get_device() != device):
                g = self._gradient(p, g, main)
                gdt = g.dtype
            at, g_at = p.data_ptr(), g.data_ptr()
            if n:
                starts += at, g_at
                ends += at + n * (4 if pdt is f32 else 2), g_at + n * (4 if gdt is f32 else 2)
            todo.append((p, g, gdt, main, at, g_at, n, pdt, device))
        turns = [(todo, range(len(todo)))] if _disjoint(starts, ends) else _in_turn(todo)
        if len(turns) > 1:
            for t in todo:
                if self.state.get(t[0]):
                    self._check_state(t[0], self.state[t[0]])
        seed = self._seed + 1
        for turn, numbers in turns:
            self._step_tensors(group, turn, [seed + k for k in numbers])

    def _step_tensors(self, group, todo, seeds):
        """A step of tensors of which none writes what another touches."""
        b1, b2 = group["betas"]
        bf16 = torch.bfloat16
        calls, states, corrections = {}, [], {}
        state, known_of, last = self.state, self._known, (None, None, None)
        for (p, g, gdt, main, at, g_at, n, pdt, device), seed in zip(todo, seeds):
            st = state[p]
            known = known_of.get(id(p)) if st else None
            if known is None:
                known = self._known_state(p, st)
            m_ref, v_ref, m_at, v_at, rest, extra, size, dtype, on, kind = known
            m, v = st["m"], st["v"]
            if (m_ref() is not m or v_ref() is not v or m.data_ptr() != m_at or v.data_ptr() != v_at
                    or n != size or pdt is not dtype or device != on
                    or ("master" in st if extra is None else not _as_known(st, extra, rest))):
                _, _, m_at, v_at, rest, *_, kind = self._known_state(p, st)
            t = st["step"] + 1
            c = corrections.get(t)
            if c is None:  # the last: tells steps apart whose corrections are alike in fp32, for drawn codes
                c = corrections[t] = (1 - b1 ** t, 1 - b2 ** t, 0 if b2 ** t * (1 - b2) >= 2.0 ** -24 else t)
            states.append(st)
            if pdt is not bf16 or kind[4]:  # nothing of the parameter is rounded by noise
                seed = c[2]
            row = _ROW(at, g_at, m_at, v_at, *rest, n, seed & 0xffffffffffffffff, c[0], c[1])
            if kind is not last[0] or gdt is not last[1] or main is not last[2]:
                last = (kind, gdt, main)
                rows = calls.setdefault(last, [])
            rows.append(row)
        self._seed += len(todo)
        for ((backend, dev, pdt, mdt, has_master), gdt, main), rows in calls.items():
            backend.adam_many(dev, rows, pdt, gdt, mdt, group["lr"], b1, b2, group["eps"], group["weight_decay"],
                              stochastic=self.stochastic_rounding and pdt is bf16 and not has_master, clear=main,
                              nearest_codes=not self.stochastic_rounding)
        for st in states:
            st["step"] += 1
        for p, _, _, main, *_ in todo:
            if not main:
                p.grad = None

    @torch.no_grad()
    def moment_values(self) -> List[Tuple[torch.Tensor, torch.Tensor]]:
        """fp32 copies of the moments (m, v), of the parameters' shapes, in the order of the parameters that have
        made a step."""
        out, calls = [], {}
        for group in self.param_groups:
            for p in group["params"]:
                st = self.state.get(p)
                if not st:
                    continue
                if self._check_state(p, st) != torch.int8:
                    out.append((st["m"].to(torch.float32, copy=True), st["v"].to(torch.float32, copy=True)))
                    continue
                m, v = (torch.empty(p.shape, device=p.device) for _ in range(2))
                out.append((m, v))
                calls.setdefault(p.device, []).append(
                    _ROW(v.data_ptr(), m.data_ptr(), st["m"].data_ptr(), st["v"].data_ptr(), 0, st["m_scale"].data_ptr(),
                         st["v_scale"].data_ptr(), p.numel(), 0, 1.0, 1.0))
        for dev, rows in calls.items():
            backend_for(dev).adam_values(dev, rows)
        return out
