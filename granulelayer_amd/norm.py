"""Layer norm in front of a sparse layer or a projection: y = (x - mean) / sqrt(variance + eps) * weight + bias.

What a model's residual stream goes through before each of them, and the other end of ``dense_projection``'s residual:
x may be the float32 stream and the result the bfloat16 operand (``out_dtype``), rounded once.  Means, variances and
the gradients' sums are float32; gradients of weight and bias go to ``main_grad`` where the parameters have it, as
the other layers' do, and are added in a fixed order (no counterpart in the reference).
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import nn
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from .backend import backend_for
from .dense import _main_grads, _owner

_DTYPES = (torch.float32, torch.bfloat16)


def _check(x, weight, bias, eps, out_dtype):
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must be [..., features] (got {tuple(x.shape)})")
    if x.dtype not in _DTYPES or out_dtype not in _DTYPES:
        raise TypeError(f"x and the result must be float32 or bfloat16 (got {x.dtype} and {out_dtype})")
    if not eps >= 0:
        raise ValueError(f"eps must be at least 0 (got {eps})")
    D = x.shape[-1]
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if t.shape != (D,):
            raise ValueError(f"{name} must be [{D}] (got {tuple(t.shape)})")
        if t.dtype not in _DTYPES:
            raise TypeError(f"{name} must be float32 or bfloat16 (got {t.dtype})")
        if t.device != x.device:
            raise ValueError(f"{name} on {t.device} but x on {x.device}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"weight and bias must be of one dtype (got {weight.dtype} and {bias.dtype})")


class LayerNormFunction(torch.autograd.Function):
    """x [M, D] -> y [M, D]; keeps x, the weight, and each row's mean and factor.  The bias may change before the
    backward, which reads only its shape and main_grad."""

    @staticmethod
    def forward(ctx, x, w, b, eps, out_dtype):
        y, stats = backend_for(x.device).norm_forward(x, w, b, eps, out_dtype, True)
        ctx.save_for_backward(x, w, stats)
        ctx.weight = _owner(w)
        # a computed bias stands there by its shape and type alone
        ctx.bias = b if b is None or b.is_leaf or hasattr(b, "main_grad") else torch.empty_like(b, device="meta")
        return y

    @staticmethod
    def backward(ctx, dy):
        # what once_differentiable adds is needed where a graph of the backward is made
        return _graph_gradients(ctx, dy) if torch.is_grad_enabled() else _gradients(ctx, dy)


def _gradients(ctx, dy):
    x, w, stats = ctx.saved_tensors
    b = ctx.bias
    need_x, need_w, need_b = ctx.needs_input_grad[:3]
    dx = torch.empty_like(x, memory_format=torch.contiguous_format) if need_x else None
    mg_w, mg_b, use_main = _main_grads(ctx.weight, b, need_w, need_b)
    if use_main:
        dw, db = mg_w, mg_b
    else:
        dw = torch.empty_like(w, memory_format=torch.contiguous_format) if need_w else None
        db = torch.empty_like(b, device=x.device, memory_format=torch.contiguous_format) if need_b else None
    backend_for(x.device).norm_backward(dy, x, w, stats, dx, dw, db, use_main)
    return dx, None if use_main else dw, None if use_main else db, None, None


_graph_gradients = once_differentiable(_gradients)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``(x - mean) / sqrt(variance + eps) * weight + bias`` over the last dimension.

    x [..., D] float32 or bfloat16, its rows any stride apart; weight and bias [D] of one of these types, or None.
    The result is of ``out_dtype`` (x's type by default).  A row with an infinity or a NaN is NaN, the others are
    not touched by it; so are the gradients but for those of weight and bias, which sum over all rows.  Tangents of
    forward-mode differentiation are refused."""
    out_dtype = x.dtype if out_dtype is None else out_dtype
    _check(x, weight, bias, eps, out_dtype)
    D = x.shape[-1]
    x2 = x if x.dim() == 2 else x.reshape(-1, D)
    if (forward_ad._current_level >= 0  # an operand may have a tangent, which the function refuses
            or torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                            or (bias is not None and bias.requires_grad))):
        y = LayerNormFunction.apply(x2, weight, bias, eps, out_dtype)
    else:
        y = backend_for(x.device).norm_forward(x2, weight, bias, eps, out_dtype, False)[0]
    return y if x.dim() == 2 else y.view(x.shape)


class LayerNorm(nn.Module):
    """``layer_norm`` with its parameters: weight [dim] ones and bias [dim] zeros of ``dtype``."""

    def __init__(self, dim: int, eps: float = 1e-5, bias: bool = True, dtype: torch.dtype = torch.float32,
                 out_dtype: Optional[torch.dtype] = None, device=None):
        super().__init__()
        if dim < 1:
            raise ValueError("dim must be at least 1")
        if not eps >= 0:
            raise ValueError(f"eps must be at least 0 (got {eps})")
        if dtype not in _DTYPES or out_dtype not in (None, *_DTYPES):
            raise NotImplementedError("dtype and out_dtype must be float32 or bfloat16")
        self.dim, self.eps, self.out_dtype = dim, eps, out_dtype
        self.weight = nn.Parameter(torch.ones(dim, dtype=dtype, device=device))
        if bias:
            self.bias = nn.Parameter(torch.zeros(dim, dtype=dtype, device=device))
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

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return layer_norm(x, self.weight, self.bias, self.eps, self.out_dtype)

    def extra_repr(self) -> str:
        return f"{self.dim}, eps={self.eps}, bias={self.bias is not None}, dtype={self.weight.dtype}, out_dtype={self.out_dtype}"
