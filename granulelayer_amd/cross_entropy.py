"""Softmax cross entropy of a dense head, without a tensor of its logits: the loss of ``softmax(x W^T + b)`` against a class a
row.

The other end of a model around the sparse layer: its last projection goes onto a large number of classes (a
vocabulary), whose logits would be the largest tensor of the step.  The forward is one product whose tiles leave their
softmax statistics instead of logits; the backward makes the logits again, a piece of the classes at a time, and
keeps their gradient only until two more products have taken it.  The forward of a training step fills the first
piece's place already where that saves time, with exponentials (of bf16 operands 2 bytes each, of fp32 ones 4) that the
backward turns into the gradient: one piece's memory in all, held from the forward to the backward, for every loss that
waits for its own.  ``workspace_budget`` bounds it; under activation checkpointing it is held in the backward alone.
Operands are those of ``dense_projection``, fp32 or bf16 with products, sums and statistics in fp32, and gradients go to
``main_grad`` where the parameters have it (no counterpart in the reference).

With bf16 operands the gradient at the logits is rounded to bf16 before the products with the weight and with x, half a
step, 2^-8, of each term at most; the bias' gradient sums it unrounded.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from .backend import backend_for
from .dense import _main_grads, _owner, _through_function

REDUCTIONS = ("none", "mean", "sum")


def _check(x, weight, target, bias, reduction, workspace_budget):
    if reduction not in REDUCTIONS:
        raise ValueError(f"unknown reduction {reduction!r} (one of {REDUCTIONS})")
    if workspace_budget is not None and (isinstance(workspace_budget, bool) or not isinstance(workspace_budget, int)
                                         or workspace_budget < 1):
        raise ValueError(f"workspace_budget must be a positive number of bytes or None (got {workspace_budget!r})")
    if weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"weight must be [classes, input_dim] (got {tuple(weight.shape)})")
    N, K = weight.shape
    if x.dim() < 1 or x.shape[-1] != K:
        raise ValueError(f"x must be [..., {K}] (got {tuple(x.shape)})")
    if x.dtype != weight.dtype or x.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"x and weight must both be float32 or both bfloat16 (got {x.dtype} and {weight.dtype})")
    if target.shape != x.shape[:-1]:
        raise ValueError(f"target must be {list(x.shape[:-1])} (got {tuple(target.shape)})")
    if target.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"target must be int64 or int32 (got {target.dtype})")
    if bias is not None:
        if bias.shape != (N,):
            raise ValueError(f"bias must be [{N}] (got {tuple(bias.shape)})")
        if bias.dtype != weight.dtype:
            raise TypeError(f"bias must be {weight.dtype} as the weight is (got {bias.dtype})")
    for name, t in (("weight", weight), ("target", target), ("bias", bias)):
        if t is not None and t.device != x.device:
            raise ValueError(f"{name} on {t.device} but x on {x.device}")


class DenseCrossEntropyFunction(torch.autograd.Function):
    """x [M, K], target [M] -> the loss; keeps the operands, five words a row, and the first piece's exponentials where
    they are worth it, which the first backward turns into its gradient in place.  All of them are saved tensors: activation
    checkpointing and hooks on saved tensors have them."""

    @staticmethod
    def forward(ctx, x, w, b, target, reduction, ignore_index, budget):
        be = backend_for(x.device)
        loss, kept, exps = be.ce_forward(x, w, b, target, reduction, ignore_index, True, budget)
        ctx.capture = be.capture_id(x.device) if exps is not None else 0
        ctx.place = 0 if exps is None else exps.data_ptr()
        ctx.used_up = False
        ctx.save_for_backward(x, w, b, target, kept, exps)
        ctx.owners = _owner(w), _owner(b)
        ctx.reduction, ctx.ignore_index, ctx.budget = reduction, ignore_index, budget
        return loss

    @staticmethod
    def backward(ctx, dloss):
        # what once_differentiable adds is needed where a graph of the backward is made
        return _graph_gradients(ctx, dloss) if torch.is_grad_enabled() else _gradients(ctx, dloss)


def _gradients(ctx, dloss):
    x, w, b, target, kept, exps = ctx.saved_tensors
    need_x, need_w, need_b = ctx.needs_input_grad[:3]
    dx = torch.empty_like(x, memory_format=torch.contiguous_format) if need_x else None
    mg_w, mg_b, use_main = _main_grads(*ctx.owners, need_w, need_b)
    if use_main:
        dw, db = mg_w, mg_b
    else:
        dw = torch.empty_like(w, memory_format=torch.contiguous_format) if need_w else None
        db = torch.empty_like(b, memory_format=torch.contiguous_format) if need_b else None
    be = backend_for(x.device)
    # Used up: a second backward of a retained graph makes them again, and so does one that a captured graph may replay
    # without its forward.  (A hook may have brought them to any address.)
    used_up, ctx.used_up = ctx.used_up, True
    own = exps if not used_up and exps is not None and exps.data_ptr() == ctx.place else None
    if exps is not None and (used_up or be.capture_id(x.device) != ctx.capture or exps.data_ptr() % 256):
        exps = None
    be.ce_backward(dloss.resolve_neg(), x, w, b, target, ctx.reduction, ctx.ignore_index, kept, dx, dw, db, use_main,
                   ctx.budget, exps)
    if own is not None and own.untyped_storage().nbytes() == own.numel():
        own.untyped_storage().resize_(0)  # a retained graph need not hold what nothing reads again
    return dx, None if use_main else dw, None if use_main else db, None, None, None, None


_graph_gradients = once_differentiable(_gradients)


def dense_cross_entropy(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, bias: Optional[torch.Tensor] = None,
                        reduction: str = "mean", ignore_index: int = -100,
                        workspace_budget: Optional[int] = None) -> torch.Tensor:
    """Cross entropy of ``softmax(x @ weight.T + bias)`` against the classes ``target``, in float32.

    x [..., K] and weight [N, K], both float32 or both bfloat16 (their rows any stride apart); bias [N] of their
    type; target [...] int64 or int32.  ``reduction``: "none" (a loss a row), "sum", or "mean" over the rows that
    count.  Rows with ``ignore_index`` have the loss 0 and no gradient, whatever x holds there; a mean of no rows is 0.
    Any other target that is no class makes the loss NaN.  A class whose bias is -inf takes no part; logits past 2.3e38 in
    size count as infinite.  The backward's
    pieces of gradients at the logits take up to ``workspace_budget`` bytes (4 GiB by default; of 256 classes at
    least), from the forward on where that keeps exponentials for it (from 512 bfloat16 or 64 float32 features on; with 4
    bytes for every 64 of them).  It takes the operands as they were: none of them may change before it.  Tangents of
    forward-mode differentiation are refused."""
    _check(x, weight, target, bias, reduction, workspace_budget)
    N, K = weight.shape
    x2 = x if x.dim() == 2 else x.reshape(-1, K)
    t = target.reshape(-1)
    t = (t if t.dtype == torch.int64 else t.long()).contiguous()
    budget = 0 if workspace_budget is None else workspace_budget
    if _through_function(x, weight, bias):
        loss = DenseCrossEntropyFunction.apply(x2, weight, bias, t, reduction, ignore_index, budget)
    else:
        loss = backend_for(x.device).ce_forward(x2, weight, bias, t, reduction, ignore_index, False)[0]
    return loss.view(target.shape) if reduction == "none" and target.dim() != 1 else loss


class DenseCrossEntropy(nn.Module):
    """``dense_cross_entropy`` with the head's parameters: weight [classes, input_dim] ~ N(0, 1 / input_dim) and, with
    ``bias``, zeros [classes], of ``dtype``.  The input is cast to the weight's type.  A weight shared with another
    module (an embedding's table) is passed as ``weight``; where it has ``main_grad``, the other module's gradient has to
    go there too, as FusedAdamW reads nothing else then."""

    def __init__(self, input_dim: int, classes: int, bias: bool = False, dtype: torch.dtype = torch.bfloat16,
                 reduction: str = "mean", ignore_index: int = -100, workspace_budget: Optional[int] = None, device=None,
                 seed: int = 0, weight: Optional[nn.Parameter] = None):
        super().__init__()
        if input_dim < 1 or classes < 1:
            raise ValueError("input_dim and classes must be at least 1")
        if reduction not in REDUCTIONS:
            raise ValueError(f"unknown reduction {reduction!r} (one of {REDUCTIONS})")
        if weight is not None:
            if tuple(weight.shape) != (classes, input_dim):
                raise ValueError(f"weight must be [{classes}, {input_dim}] (got {tuple(weight.shape)})")
            dtype, device = weight.dtype, weight.device
        if dtype not in (torch.float32, torch.bfloat16):
            raise NotImplementedError(f"dtype {dtype} (the MI355X path computes fp32 or bf16 operands)")
        self.input_dim, self.classes, self.reduction, self.ignore_index = input_dim, classes, reduction, ignore_index
        self.workspace_budget = workspace_budget
        dev = torch.device(device or "cpu")
        if weight is None:
            gen = torch.Generator(device=dev).manual_seed(seed)
            weight = nn.Parameter((torch.randn(classes, input_dim, generator=gen, device=dev) * input_dim ** -0.5).to(dtype))
        self.weight = weight
        if bias:
            self.bias = nn.Parameter(torch.zeros(classes, dtype=dtype, device=dev))
        else:
            self.register_parameter("bias", None)

    def enable_main_grad(self):
        """Accumulate the parameters' gradients into persistent fp32 ``main_grad`` buffers (autograd then
        returns None for them)."""
        for p in self.parameters():
            if getattr(p, "main_grad", None) is None:
                p.main_grad = torch.zeros(p.shape, device=p.device, dtype=torch.float32)

    def zero_main_grad(self):
        for p in self.parameters():
            if getattr(p, "main_grad", None) is not None:
                p.main_grad.zero_()

    def forward(self, x: torch.Tensor, target: torch.Tensor) -> torch.Tensor:
        return dense_cross_entropy(x.to(self.weight.dtype), self.weight, target, self.bias, self.reduction,
                                   self.ignore_index, self.workspace_budget)

    def extra_repr(self) -> str:
        return (f"in={self.input_dim}, classes={self.classes}, bias={self.bias is not None}, dtype={self.weight.dtype}, "
                f"reduction={self.reduction!r}, ignore_index={self.ignore_index}")
