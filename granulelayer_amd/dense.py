"""Dense projection beside the sparse one: y = act(x W^T + b) + residual.

What a model around a sparse layer needs next to it: the map from its width into the layer's inputs,
and from the pooled outputs back onto a residual stream.  Bias, activation and residual are the
product's epilogue on the GPU, activations are the sparse layer's (identity, relu, erf gelu; gelu by a
polynomial, within 2.5e-7 of erf's, and about 0 at -inf where erf's form gives NaN), operands fp32 or bf16 with
products and sums in fp32, and gradients go to ``main_grad`` where the parameters have it, as the sparse layer's do (no
counterpart in the reference).

The backward needs x and, through the activation, z = x W^T + b.  ReLU keeps one bit of z an element.
GELU keeps z in the operands' type, or in 8 bits (``activation_checkpoint="int8"``, activations8.py),
which also keeps x in 8 bits; the gradients are then those at the values that were kept.

With bf16 operands the gradient at z, dz = dy act'(z), is rounded to bf16 before dX and dW (the matrix
instructions take two operands of one type), also where dy is fp32 because the residual is: half a step, 2^-8, of each
term at most, so 2.3e-3 of dX and dW in all where the rounding of the result alone gives 1.7e-3.  db sums dz unrounded.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import nn
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from .activations8 import check_activation_checkpoint
from .backend import backend_for
from .config import ACTIVATIONS

_KEEP = {"identity": "none", "relu": "sign", "gelu": "z"}


def _check(x, weight, bias, residual, activation, activation_checkpoint):
    if activation not in ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r} (one of {ACTIVATIONS})")
    check_activation_checkpoint(activation_checkpoint)
    if weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"weight must be [output_dim, input_dim] (got {tuple(weight.shape)})")
    N, K = weight.shape
    if x.dim() < 1 or x.shape[-1] != K:
        raise ValueError(f"x must be [..., {K}] (got {tuple(x.shape)})")
    if x.dtype != weight.dtype or x.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"x and weight must both be float32 or both bfloat16 (got {x.dtype} and {weight.dtype})")
    if bias is not None:
        if tuple(bias.shape) != (N,):
            raise ValueError(f"bias must be [{N}] (got {tuple(bias.shape)})")
        if bias.dtype != weight.dtype:
            raise TypeError(f"bias must be {weight.dtype} as the weight is (got {bias.dtype})")
    if residual is not None:
        if residual.shape[:-1] != x.shape[:-1] or residual.shape[-1:] != weight.shape[:1]:
            raise ValueError(f"residual must be {[*x.shape[:-1], N]} as the result is (got {tuple(residual.shape)}; "
                             "expand a broadcast one)")
        if residual.dtype not in (torch.float32, torch.bfloat16):
            raise TypeError(f"residual must be float32 or bfloat16 (got {residual.dtype})")
    for name, t in (("weight", weight), ("bias", bias), ("residual", residual)):
        if t is not None and t.device != x.device:
            raise ValueError(f"{name} on {t.device} but x on {x.device}")


def _through_function(*operands) -> bool:
    """Whether a call goes through its autograd function: an operand needs its gradient, or may have a tangent of forward-mode
    differentiation, which the function refuses."""
    if forward_ad._current_level >= 0:
        return True
    if torch.is_grad_enabled():
        for t in operands:
            if t is not None and t.requires_grad:
                return True
    return False


def _owner(t):
    """The tensor whose ``main_grad`` a backward looks for, or None.  (What is saved may come back as another tensor, without
    its attributes: activation checkpointing and hooks on saved tensors do that.)"""
    return t if t is not None and t.requires_grad and (t.is_leaf or hasattr(t, "main_grad")) else None


def _main_grads(w, b, need_w, need_b):
    """The fp32 ``main_grad`` buffers when every parameter that needs a gradient has one."""
    bufs = []
    for name, p, need in (("weight", w, need_w), ("bias", b, need_b)):
        mg = getattr(p, "main_grad", None) if need else None
        if need and mg is None:
            return None, None, False
        if mg is not None and (mg.dtype != torch.float32 or mg.shape != p.shape or mg.device != p.device
                               or not mg.is_contiguous()):
            raise ValueError(f"{name}.main_grad must be a contiguous float32 tensor of the {name}'s shape and device")
        bufs.append(mg)
    return bufs[0], bufs[1], need_w or need_b


class DenseProjectionFunction(torch.autograd.Function):
    """x [M, K], residual [M, N] or None -> y [M, N]; keeps x (or its 8-bit form), W and what the activation's
    derivative needs of z.  The bias may change before the backward, which reads only its shape and main_grad."""

    @staticmethod
    def forward(ctx, x, w, b, res, activation, activation_checkpoint):
        be = backend_for(x.device)
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        packed = activation_checkpoint == "int8"
        keep = _KEEP[activation] if need_x or need_w or need_b else "none"
        if keep == "z" and packed:
            keep = "z8"
        y, z, z_exp = be.dense_forward(x, w, b, res, activation, keep)
        xs = (None, None, None)  # x, or its codes and exponents
        if need_w:
            xs = (None, *be.pack8(x)) if packed else (x, None, None)
        ctx.save_for_backward(*xs, w, None, z, z_exp)
        ctx.weight = _owner(w)
        # a computed bias stands there by its shape and type alone
        ctx.bias = b if b is None or b.is_leaf or hasattr(b, "main_grad") else torch.empty_like(b, device="meta")
        ctx.activation, ctx.keep, ctx.x_shape, ctx.x_dtype = activation, keep, x.shape, x.dtype
        ctx.res_dtype = None if res is None else res.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, xq, xe, w, _, z, z_exp = ctx.saved_tensors
        b = ctx.bias
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dy = dy.resolve_neg()
        dres = dy.to(ctx.res_dtype) if need_r else None
        if not (need_x or need_w or need_b):
            return None, None, None, dres, None, None
        mg_w, mg_b, use_main = _main_grads(ctx.weight, b, need_w, need_b)
        gtype = torch.float32 if use_main else w.dtype
        dx = torch.empty(ctx.x_shape, device=w.device, dtype=ctx.x_dtype) if need_x else None
        dw = mg_w if use_main else (torch.empty(w.shape, device=w.device, dtype=gtype) if need_w else None)
        db = mg_b if use_main else (torch.empty(b.shape, device=w.device, dtype=gtype) if need_b else None)
        backend_for(dy.device).dense_backward(dy, ctx.activation, ctx.keep, z, z_exp, x, xq, xe, w, dx, dw, db, use_main)
        return dx, None if use_main else dw, None if use_main else db, dres, None, None


def dense_projection(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                     residual: Optional[torch.Tensor] = None, activation: str = "identity",
                     activation_checkpoint: str = "exact") -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual``.

    x [..., K] and weight [N, K], both float32 or both bfloat16 (products and sums in fp32); bias [N] of
    their type; residual [..., N] float32 or bfloat16.  The result has x's type, or float32 with a
    float32 residual, and is rounded once.  Rows may be any stride apart.  The backward of bfloat16
    operands rounds the gradient at the product to bfloat16 before the products for x and the weight.  Tangents of
    forward-mode differentiation are refused."""
    _check(x, weight, bias, residual, activation, activation_checkpoint)
    N, K = weight.shape
    x2 = x if x.dim() == 2 else x.reshape(-1, K)
    r2 = residual if residual is None or residual.dim() == 2 else residual.reshape(-1, N)
    if _through_function(x, weight, bias, residual):
        y = DenseProjectionFunction.apply(x2, weight, bias, r2, activation, activation_checkpoint)
    else:
        y = backend_for(x.device).dense_forward(x2, weight, bias, r2, activation, "none")[0]
    return y if x.dim() == 2 else y.view(*x.shape[:-1], N)


class DenseProjection(nn.Module):
    """``dense_projection`` with its parameters: weight [output_dim, input_dim] ~ N(0, 1 / input_dim) and
    bias [output_dim] ~ N(0, bias_std^2) of ``dtype``.  The input is cast to the weight's type."""

    def __init__(self, input_dim: int, output_dim: int, activation: str = "identity", bias: bool = True,
                 dtype: torch.dtype = torch.bfloat16, activation_checkpoint: str = "exact", device=None, seed: int = 0,
                 bias_std: float = 0.0):
        super().__init__()
        if input_dim < 1 or output_dim < 1:
            raise ValueError("input_dim and output_dim must be at least 1")
        if activation not in ACTIVATIONS:
            raise ValueError(f"unknown activation {activation!r} (one of {ACTIVATIONS})")
        if dtype not in (torch.float32, torch.bfloat16):
            raise NotImplementedError(f"dtype {dtype} (the MI355X path computes fp32 or bf16 operands)")
        self.input_dim, self.output_dim, self.activation = input_dim, output_dim, activation
        self.activation_checkpoint = check_activation_checkpoint(activation_checkpoint)
        dev = torch.device(device or "cpu")
        gen = torch.Generator(device=dev).manual_seed(seed)
        w = torch.randn(output_dim, input_dim, generator=gen, device=dev) * input_dim ** -0.5
        self.weight = nn.Parameter(w.to(dtype))
        if bias:
            b = torch.randn(output_dim, generator=gen, device=dev) * bias_std
            self.bias = nn.Parameter(b.to(dtype))
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

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        return dense_projection(x.to(self.weight.dtype), self.weight, self.bias, residual, self.activation,
                                self.activation_checkpoint)

    def extra_repr(self) -> str:
        return (f"in={self.input_dim}, out={self.output_dim}, activation={self.activation}, "
                f"bias={self.bias is not None}, dtype={self.weight.dtype}, "
                f"activation_checkpoint={self.activation_checkpoint}")
